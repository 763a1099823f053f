"""Plain 64-bit forms of the decode-step operators and the inputs their tests share."""
import math

import numpy as np
import torch

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def make_pools(gen, pages, page, heads, dim, dtype, layout="nhd", fill=1.0):
    """K and V pools [pages, page, heads, dim] on the CPU, as views of the layout asked for."""
    shape = (pages, page, heads, dim) if layout == "nhd" else (pages, heads, page, dim)
    out = []
    for _ in range(2):
        t = (torch.randn(shape, generator=gen, dtype=torch.float32) * fill).to(DTYPES[dtype])
        out.append(t if layout == "nhd" else t.transpose(1, 2))
    return out


def on_device(pool, dev):
    """The same tensor on the device with the same layout."""
    if pool.is_contiguous():
        return pool.to(dev)
    return pool.transpose(1, 2).contiguous().to(dev).transpose(1, 2)


def rotate(x, positions, inv_freq, interleaved, factor):
    x = x.double()
    half = inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq.double()[None, :]
    c, s = (factor * angle.cos())[:, None, :], (factor * angle.sin())[:, None, :]
    y = x.clone()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y


def attend(q, k_pool, v_pool, table, lens, scale, window=0):
    """out [b, hq, d], lse [b, hq], p: list of [hq, attended] and the first attended token of each sequence."""
    pages, page, hkv, d = k_pool.shape
    b, hq = q.shape[0], q.shape[1]
    out = torch.zeros(b, hq, d, dtype=torch.float64)
    spread = torch.zeros(b, hq, d, dtype=torch.float64)  # sum of p |v|: what a relative error of p is relative to
    lse = torch.full((b, hq), -math.inf, dtype=torch.float64)
    probs, firsts = [], []
    size = torch.zeros(b, hq, dtype=torch.float64)  # largest sum of |q||k| of a score, scaled
    for i in range(b):
        n = max(0, min(int(lens[i]), table.shape[1] * page))
        first = max(0, n - window) if window else 0
        t = torch.arange(first, n)
        pg = table[i].long()[t // page]
        ok = (pg >= 0) & (pg < pages)
        pg = torch.where(ok, pg, torch.zeros_like(pg))
        k, v = k_pool[pg, t % page].double(), v_pool[pg, t % page].double()
        p_all = torch.zeros(hq, n - first, dtype=torch.float64)
        for h in range(hq):
            kv = h // (hq // hkv)
            if ok.any():
                s = scale * (k[ok, kv] @ q[i, h].double())
                m = s.max()
                if m != -math.inf:
                    e = torch.exp(s - m)
                    p = e / e.sum()
                    out[i, h] = p @ v[ok, kv]
                    spread[i, h] = p @ v[ok, kv].abs()
                    lse[i, h] = m + torch.log(e.sum())
                    p_all[h, ok] = p
                    size[i, h] = abs(scale) * (k[ok, kv].abs() @ q[i, h].double().abs()).max()
        probs.append(p_all)
        firsts.append(first)
    return out, lse, probs, firsts, spread, size


def evict(k_pool, v_pool, table, lens, weights, positions, budget, recent):
    """New pools, weights, positions (numpy) and lengths; inputs are left alone."""
    page = k_pool.shape[1]
    k_new, v_new = k_pool.clone(), v_pool.clone()
    w_new, p_new = weights.copy(), positions.copy()
    cap = table.shape[1] * page
    new_lens = []
    for i in range(weights.shape[0]):
        n = max(0, min(int(lens[i]), cap))
        k = min(n, budget)
        new_lens.append(k)
        if n <= budget:
            continue
        for h in range(weights.shape[1]):
            w, pos = weights[i, h, :n].astype(np.float64), positions[i, h, :n].astype(np.int64)
            safe = pos > pos.max() - recent
            nan = np.isnan(w)
            w = np.where(nan, 0.0, w) + 0.0
            rank = np.lexsort((np.arange(n), -w, ~nan, ~safe))
            kept = np.zeros(n, dtype=bool)
            kept[rank[:k]] = True
            holes, movers = np.flatnonzero(~kept[:k]), k + np.flatnonzero(kept[k:])
            w_new[i, h, holes], p_new[i, h, holes] = weights[i, h, movers], positions[i, h, movers]
            w_new[i, h, k:n], p_new[i, h, k:n] = 0.0, -1
            heads = slice(None) if weights.shape[1] == 1 else slice(h, h + 1)
            for s, d in zip(movers, holes):
                sp, dp = int(table[i, s // page]), int(table[i, d // page])
                if 0 <= sp < k_pool.shape[0] and 0 <= dp < k_pool.shape[0]:
                    k_new[dp, d % page, heads] = k_pool[sp, s % page, heads]
                    v_new[dp, d % page, heads] = v_pool[sp, s % page, heads]
    return k_new, v_new, w_new, p_new, np.array(new_lens, dtype=np.int32)
