"""What the decode-step operators over paged KV pools are measured on.

Three operators of tair_kvcache_b200.kernel that a serving engine calls around the pools the connector moves:

  append  batch_append_kv_pages   rotary positions on new queries and keys, keys and values into their pool slots
  attend  batch_attend_kv_pages   attention of one new token per sequence over its pages, attention weights accumulated
  evict   batch_evict_kv_pages    the heaviest and the newest tokens kept, packed into the first slots of the pages

`run` does one pass in plain torch, or with `own` set through the package's kernels.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_kernel = None


def _ops():
    global _kernel
    if _kernel is None:
        from tair_kvcache_b200 import kernel
        _kernel = kernel
    return _kernel


# ----------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one sequence in interactive use: the new token's queries and keys of an 8-KV-head model, latency counts
        dict(name="append_one_token", op="append", tokens=1, q_heads=32, kv_heads=8, head_dim=128, rotary=128,
             interleaved=False, page=16, layout="nhd", dtype="bf16", far=8192, scaling="none"),
        # one decode step of a batch, half of each head rotated in interleaved pairs
        dict(name="append_decode_batch", op="append", tokens=193, q_heads=16, kv_heads=4, head_dim=64, rotary=32,
             interleaved=True, page=64, layout="hnd", dtype="fp16", far=131072, scaling="linear"),
        # the prompt of a long-context model written in one go, positions beyond the trained range
        dict(name="append_prompt", op="append", tokens=16384, q_heads=32, kv_heads=8, head_dim=128, rotary=128,
             interleaved=False, page=16, layout="nhd", dtype="bf16", far=1048576, scaling="yarn"),
        # first tokens of a chat: one short sequence, 32 query heads on 8 KV heads
        dict(name="attend_one_short", op="attend", batch=1, low=100, high=100, q_heads=32, kv_heads=8, head_dim=128,
             page=16, layout="nhd", dtype="bf16", window=0, weights="none"),
        # a serving batch of ragged lengths between 512 and 8192 tokens
        dict(name="attend_batch_ragged", op="attend", batch=64, low=512, high=8192, q_heads=32, kv_heads=8,
             head_dim=128, page=16, layout="nhd", dtype="bf16", window=0, weights="none"),
        # one very long document on one of eight tensor-parallel ranks: a single KV head, the length split over the GPU
        dict(name="attend_one_long", op="attend", batch=1, low=131072, high=131072, q_heads=8, kv_heads=1,
             head_dim=128, page=32, layout="nhd", dtype="fp16", window=0, weights="none"),
        # a batch whose cache will be evicted from: every head's weights are accumulated
        dict(name="attend_weights", op="attend", batch=16, low=2000, high=6001, q_heads=32, kv_heads=8, head_dim=128,
             page=16, layout="nhd", dtype="bf16", window=0, weights="heads"),
        # a small model with an odd number of heads, a sliding window and pages laid out head by head
        dict(name="attend_window_odd", op="attend", batch=37, low=1, high=5000, q_heads=15, kv_heads=3, head_dim=80,
             page=48, layout="hnd", dtype="fp16", window=4096, weights="shared"),
        # steady state of a bounded cache: every sequence is one token over its budget
        dict(name="evict_one_step", op="evict", batch=32, low=2049, high=2049, budget=2048, recent=256, kv_heads=8,
             head_dim=128, page=16, layout="nhd", dtype="bf16", weights="heads", mixed=True),
        # after the prompt: the cache is cut to its budget, each head for itself
        dict(name="evict_after_prompt", op="evict", batch=16, low=6001, high=8192, budget=4096, recent=512, kv_heads=8,
             head_dim=128, page=16, layout="nhd", dtype="bf16", weights="heads", mixed=False),
        # one long document cut to a quarter, all heads together
        dict(name="evict_long_shared", op="evict", batch=1, low=131072, high=131072, budget=32768, recent=4096,
             kv_heads=8, head_dim=128, page=32, layout="nhd", dtype="fp16", weights="shared", mixed=False),
        # a few short ragged sequences, some of them under the budget
        dict(name="evict_short_odd", op="evict", batch=7, low=65, high=700, budget=301, recent=33, kv_heads=3,
             head_dim=80, page=48, layout="hnd", dtype="fp16", weights="heads", mixed=True),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "evict"])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    case = dict(op=op, kv_heads=kv_heads, head_dim=rng.choice([64, 80, 96, 128, 128, 256]),
                page=rng.choice([8, 16, 32, 48, 64]), layout=rng.choice(["nhd", "hnd"]),
                dtype=rng.choice(["bf16", "fp16"]))
    row = kv_heads * case["head_dim"]
    if op == "append":
        case["q_heads"] = kv_heads * group
        most = min(16384, int(16384 * 6144 / (row * (group + 2))))
        case["tokens"] = _log_int(rng, 1, max(1, most))
        case["rotary"] = 2 * rng.randint(1, case["head_dim"] // 2) if rng.random() < 0.5 else case["head_dim"]
        case["interleaved"] = rng.random() < 0.5
        case["far"] = _log_int(rng, 4096, 1048576)
        case["scaling"] = rng.choice(["none", "linear", "ntk", "yarn", "llama3"])
        return case
    case["batch"] = _log_int(rng, 1, 64)
    most = min(131072, int(64 * 4352 * 1024 / (row * case["batch"])))
    case["high"] = _log_int(rng, 1 if op == "attend" else 16, max(16, most // (1 if op == "attend" else 2)))
    case["low"] = rng.randint(1, case["high"])
    if op == "attend":
        case["q_heads"] = kv_heads * group
        case["window"] = rng.randint(1, case["high"]) if rng.random() < 0.25 else 0
        case["weights"] = rng.choice(["none", "none", "heads", "shared"])
    else:
        case["budget"] = rng.randint(1, case["high"])
        case["recent"] = rng.randint(0, case["budget"] // 2)
        case["weights"] = rng.choice(["heads", "shared"])
        case["mixed"] = rng.random() < 0.5
    return case


def _lengths(case):
    """Evenly spaced between low and high: their sum, and so the work, does not depend on the seed."""
    b = case["batch"]
    if b == 1:
        return [case["high"]]
    return [case["low"] + (case["high"] - case["low"]) * i // (b - 1) for i in range(b)]


# ----------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------
def _pools(case, pages, gen, fill):
    """K and V pools as [pages, page, kv_heads, head_dim] views; "hnd" keeps a head's tokens of a page together."""
    p, h, d = case["page"], case["kv_heads"], case["head_dim"]
    shape = (pages, p, h, d) if case["layout"] == "nhd" else (pages, h, p, d)
    pools = []
    for _ in range(2):
        if fill:
            t = torch.randn(shape, generator=gen, device="cuda", dtype=_DTYPES[case["dtype"]])
        else:
            t = torch.zeros(shape, device="cuda", dtype=_DTYPES[case["dtype"]])
        pools.append(t if case["layout"] == "nhd" else t.transpose(1, 2))
    return pools


def _tables(case, lens, gen):
    """A block table whose pages lie scattered over the pool; the pool holds a few pages of no one."""
    page = case["page"]
    width = max(1, -(-max(lens) // page))
    need = case["batch"] * width
    pages = need + 3
    order = torch.randperm(pages, generator=gen, device="cuda")[:need]
    return order.to(torch.int32).view(case["batch"], width), pages


def _frequencies(case):
    """One angle per position and pair of elements; a long-context scaling stretches the slow ones."""
    half = case["rotary"] // 2
    j = np.arange(half, dtype=np.float64)
    base, scale = 10000.0, 8.0
    kind = case["scaling"]
    if kind == "ntk":
        base *= scale ** (case["rotary"] / max(1, case["rotary"] - 2))
    freq = base ** (-2.0 * j / case["rotary"])
    factor = 1.0
    if kind == "linear":
        freq = freq / scale
    elif kind in ("yarn", "llama3"):
        turns = 8192.0 * freq / (2.0 * math.pi)  # turns within the trained length
        low, high = (1.0, 32.0) if kind == "yarn" else (1.0, 4.0)
        keep = np.clip((turns - low) / (high - low), 0.0, 1.0)
        freq = freq * keep + freq / scale * (1.0 - keep)
        if kind == "yarn":
            factor = 0.1 * math.log(scale) + 1.0
    return torch.tensor(freq, dtype=torch.float32, device="cuda"), factor


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    hkv, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        t, hq = case["tokens"], case["q_heads"]
        pages = -(-t // case["page"]) + 4
        k_pool, v_pool = _pools(case, pages, gen, fill=False)
        # query, key and value are slices of one fused projection, as a model hands them over
        qkv = torch.randn(t, (hq + 2 * hkv) * d, generator=gen, device="cuda", dtype=dtype)
        q, k, v = qkv.split([hq * d, hkv * d, hkv * d], dim=1)
        if t < 1024:  # a decode step: the sequences of a batch stand at positions far apart
            positions = torch.randint(0, case["far"], (t,), generator=gen, device="cuda")
        else:  # a prompt, or its next piece
            first = torch.randint(0, max(1, case["far"] - t), (1,), generator=gen, device="cuda")
            positions = first + torch.arange(t, device="cuda")
        order = torch.randperm(pages, generator=gen, device="cuda")
        token = torch.arange(t, device="cuda")
        slots = (order[token // case["page"]] * case["page"] + token % case["page"]).to(torch.int32)
        inv_freq, factor = _frequencies(case)
        return dict(case=case, q=q.view(t, hq, d), k=k.view(t, hkv, d), v=v.view(t, hkv, d), positions=positions,
                    slots=slots, k_pool=k_pool, v_pool=v_pool, inv_freq=inv_freq, factor=factor)
    lens = _lengths(case)
    table, pages = _tables(case, lens, gen)
    shuffled = torch.tensor(lens, dtype=torch.int32, device="cuda")
    shuffled = shuffled[torch.randperm(len(lens), generator=gen, device="cuda")]
    k_pool, v_pool = _pools(case, pages, gen, fill=True)
    cap = table.shape[1] * case["page"]
    state = dict(case=case, table=table, lens=shuffled, k_pool=k_pool, v_pool=v_pool, weights=None)
    heads = hkv if case["weights"] == "heads" else 1
    slot = torch.arange(cap, device="cuda", dtype=torch.int32)
    inside = (slot[None, :] < shuffled[:, None])[:, None, :]
    if case["op"] == "attend":
        # queries that look at some keys much harder than at others
        state["q"] = 2.0 * torch.randn(case["batch"], case["q_heads"], d, generator=gen, device="cuda", dtype=dtype)
        if case["weights"] != "none":
            w = torch.exp(2.0 * torch.randn(case["batch"], heads, cap, generator=gen, device="cuda"))
            state["weights"] = w * inside
            state["weights_out"] = torch.zeros_like(w)
        return state
    # accumulated weights are spread over orders of magnitude; some tokens were never looked at
    w = torch.exp(2.0 * torch.randn(case["batch"], heads, cap, generator=gen, device="cuda"))
    w = w * (torch.rand(w.shape, generator=gen, device="cuda") > 0.05)
    state["weights"] = w * inside
    positions = slot.expand(case["batch"], heads, cap)
    if case["mixed"]:
        # earlier evictions have moved tokens about: any slot but the newest token's may hold any position
        key = torch.rand(case["batch"], heads, cap, generator=gen, device="cuda") + 2.0 * (slot[None, None, :] >=
                                                                                             shuffled[:, None, None] - 1)
        positions = torch.argsort(key, dim=2).to(torch.int32)
    state["positions"] = torch.where(inside, positions, torch.full_like(positions, -1)).contiguous()
    state["weights_out"] = torch.zeros_like(state["weights"])
    state["positions_out"] = torch.full_like(state["positions"], -1)
    return state


# ----------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------
def run(state):
    return {"append": _append, "attend": _attend, "evict": _evict}[state["case"]["op"]](state)


def _append(s):
    case = s["case"]
    if own:
        q_out = _ops().batch_append_kv_pages(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["k_pool"],
                                             s["v_pool"], s["inv_freq"], interleaved=case["interleaved"],
                                             attention_factor=s["factor"])
        return q_out, s["k_pool"], s["v_pool"]
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()[None, :]
    cos = (angle.cos() * s["factor"]).float()[:, None, :]
    sin = (angle.sin() * s["factor"]).float()[:, None, :]
    rd = case["rotary"]

    def rotate(x):
        x = x.float()
        y = x.clone()
        if case["interleaved"]:
            a, b = x[..., 0:rd:2], x[..., 1:rd:2]
            y[..., 0:rd:2], y[..., 1:rd:2] = a * cos - b * sin, b * cos + a * sin
        else:
            a, b = x[..., :rd // 2], x[..., rd // 2:rd]
            y[..., :rd // 2], y[..., rd // 2:rd] = a * cos - b * sin, b * cos + a * sin
        return y.to(s["q"].dtype)

    slots = s["slots"].long()
    where = (slots // case["page"], slots % case["page"])
    s["k_pool"][where] = rotate(s["k"])
    s["v_pool"][where] = s["v"]
    return rotate(s["q"]), s["k_pool"], s["v_pool"]


def _attend(s):
    case = s["case"]
    if own:
        out = _ops().batch_attend_kv_pages(s["q"], s["k_pool"], s["v_pool"], s["table"], s["lens"],
                                           window=case["window"], weights=s["weights"],
                                           weights_out=s.get("weights_out"))
        return out if s["weights"] is None else (out, s["weights_out"])
    b, hkv, d, page = case["batch"], case["kv_heads"], case["head_dim"], case["page"]
    cap = s["table"].shape[1] * page
    pages = s["table"].long()
    q = s["q"].float().reshape(b, hkv, -1, d)
    k = s["k_pool"][pages].float().reshape(b, cap, hkv, d)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)) / math.sqrt(d)
    del k
    t = torch.arange(cap, device=q.device)[None, :]
    lens = s["lens"].long()[:, None]
    seen = t < lens
    if case["window"] > 0:
        seen = seen & (t >= lens - case["window"])
    scores = scores.masked_fill(~seen[:, None, None, :], -math.inf)
    top = scores.amax(dim=3, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    p = p / p.sum(dim=3, keepdim=True).clamp_min(1e-30)
    v = s["v_pool"][pages].float().reshape(b, cap, hkv, d)
    out = torch.matmul(p, v.permute(0, 2, 1, 3)).reshape(b, case["q_heads"], d).to(s["q"].dtype)
    if s["weights"] is None:
        return out
    mass = p.sum(dim=2) if case["weights"] == "heads" else p.sum(dim=(1, 2))[:, None, :]
    s["weights_out"].copy_(torch.where(seen[:, None, :], s["weights"] + mass, s["weights_out"]))
    return out, s["weights_out"]


def _evict(s):
    case = s["case"]
    if own:
        lens = _ops().batch_evict_kv_pages(s["k_pool"], s["v_pool"], s["table"], s["lens"], s["weights"],
                                           s["positions"], case["budget"], case["recent"],
                                           weights_out=s["weights_out"], positions_out=s["positions_out"])
        return s["k_pool"], s["v_pool"], s["weights_out"], s["positions_out"], lens
    w, pos, page = s["weights"], s["positions"], case["page"]
    b, heads, cap = w.shape
    slot = torch.arange(cap, device=w.device)[None, None, :]
    n = s["lens"].long()[:, None, None]
    keep_n = n.clamp_max(case["budget"])
    inside = slot < n
    newest = torch.where(inside, pos, torch.full_like(pos, -1)).amax(dim=2, keepdim=True)
    key = torch.where(inside & (pos > newest - case["recent"]), torch.full_like(w, math.inf), w)
    key = torch.where(inside, key, torch.full_like(w, -math.inf))
    order = torch.sort(key, dim=2, descending=True, stable=True).indices
    kept = torch.zeros_like(inside.expand(b, heads, cap)).scatter(2, order, (slot < keep_n).expand(b, heads, cap))
    hole = (slot < keep_n) & ~kept
    mover = (slot >= keep_n) & kept
    hb, hh, dst = hole.nonzero(as_tuple=True)  # both lists in the order (row, head, slot): they pair off
    _, _, src = mover.nonzero(as_tuple=True)
    w_new = torch.where(slot < keep_n, w, torch.where(inside, torch.zeros_like(w), s["weights_out"]))
    p_new = torch.where(slot < keep_n, pos, torch.where(inside, torch.full_like(pos, -1), s["positions_out"]))
    w_new[hb, hh, dst] = w[hb, hh, src]
    p_new[hb, hh, dst] = pos[hb, hh, src]
    s["weights_out"].copy_(w_new)
    s["positions_out"].copy_(p_new)
    table = s["table"].long()
    to, fro = (table[hb, dst // page], dst % page), (table[hb, src // page], src % page)
    for pool in (s["k_pool"], s["v_pool"]):
        if heads == 1:
            pool[to[0], to[1]] = pool[fro[0], fro[1]]
        else:
            pool[to[0], to[1], hh] = pool[fro[0], fro[1], hh]
    return s["k_pool"], s["v_pool"], s["weights_out"], s["positions_out"], s["lens"].clamp_max(case["budget"])


# ----------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------
def work(case):
    d, hkv = case["head_dim"], case["kv_heads"]
    row = hkv * d * 2  # K or V bytes of one token
    if case["op"] == "append":
        t, hq = case["tokens"], case["q_heads"]
        pairs = t * (hq + hkv) * case["rotary"] // 2
        return {"bytes": t * (2 * hq * d * 2 + 4 * row + 8 + 4) + 2 * case["rotary"], "flops": 6 * pairs}
    lens = _lengths(case)
    heads = hkv if case["weights"] == "heads" else 1
    entries = sum(-(-n // case["page"]) for n in lens)
    if case["op"] == "attend":
        seen = sum(min(n, case["window"]) if case["window"] else n for n in lens)
        moved = 2 * row * seen + 2 * case["batch"] * case["q_heads"] * d * 2 + 4 * entries + 4 * case["batch"]
        if case["weights"] != "none":
            moved += 8 * heads * seen
        return {"bytes": moved, "flops": 4 * case["q_heads"] * d * seen}
    moved = flops = 0
    for n in lens:
        k, r = min(n, case["budget"]), min(n, case["recent"])
        # tokens kept from behind the budget: the newest lie at the end, or anywhere; the heavy ones anywhere
        if case["mixed"] or k == n:
            moves = k * (n - k) / n
        else:
            moves = min(r, n - k) + (k - r) * max(0, n - r - k) / max(1, n - r)
        moved += heads * (8 * n + 8 * n) + moves * 4 * row  # a shared row moves whole, a head's row by itself
        flops += heads * n
    return {"bytes": int(moved + 4 * entries + 8 * case["batch"]), "flops": int(flops)}


# ----------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ----------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](case, s)


def _exact_append(case, s):
    rd = case["rotary"]
    turn = torch.polar(torch.full((case["tokens"], rd // 2), float(s["factor"]), dtype=torch.float64, device="cuda"),
                       torch.outer(s["positions"].double(), s["inv_freq"].double()))

    def rotated(x):
        x = x.double()
        head = x[..., :rd]
        # each pair as one complex number, multiplied by factor * exp(i angle)
        pairs = head.unflatten(-1, (rd // 2, 2)) if case["interleaved"] else head.unflatten(-1, (2, rd // 2)).mT
        z = torch.view_as_complex(pairs.contiguous()) * turn[:, None, :]
        back = torch.view_as_real(z)
        back = back.flatten(-2) if case["interleaved"] else back.mT.flatten(-2)
        return torch.cat([back, x[..., rd:]], dim=-1)

    k_pool, v_pool = s["k_pool"].double(), s["v_pool"].double()
    page = case["page"]
    for pool, rows in ((k_pool, rotated(s["k"])), (v_pool, s["v"].double())):
        flat = pool.reshape(-1, case["kv_heads"], case["head_dim"])
        flat.index_copy_(0, s["slots"].long(), rows)
        pool.copy_(flat.view(-1, page, case["kv_heads"], case["head_dim"]))
    return rotated(s["q"]), k_pool, v_pool


def _exact_attend(case, s):
    b, hq, hkv, d, page = case["batch"], case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros(b, hq, d, dtype=torch.float64, device="cuda")
    grown = None if s["weights"] is None else s["weights_out"].double()
    for i, n in enumerate(s["lens"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        at = torch.arange(first, n, device="cuda")
        rows = s["table"][i].long()[at // page], at % page
        k, v = s["k_pool"][rows].double(), s["v_pool"][rows].double()
        for h in range(hkv):
            mine = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            p = torch.softmax((k[:, h] @ s["q"][i, mine].double().T) * d ** -0.5, dim=0)
            out[i, mine] = p.T @ v[:, h]
            if grown is not None:
                if case["weights"] == "heads":
                    grown[i, h, first:n] = s["weights"][i, h, first:n].double() + p.sum(dim=1)
                else:
                    if h == 0:
                        grown[i, 0, first:n] = s["weights"][i, 0, first:n].double()
                    grown[i, 0, first:n] += p.sum(dim=1)
    return out if grown is None else (out, grown)


def _exact_evict(case, s):
    w, pos, lens = s["weights"].cpu().numpy(), s["positions"].cpu().numpy(), s["lens"].cpu().numpy()
    table, page = s["table"].cpu().numpy(), case["page"]
    w_out, p_out = s["weights_out"].cpu().numpy(), s["positions_out"].cpu().numpy()
    k_pool, v_pool = s["k_pool"].clone(), s["v_pool"].clone()
    for i in range(w.shape[0]):
        n, k = int(lens[i]), min(int(lens[i]), case["budget"])
        for h in range(w.shape[1]):
            wi, pi = w[i, h, :n].astype(np.float64), pos[i, h, :n]
            safe = pi > pi.max() - case["recent"]
            rank = np.lexsort((np.arange(n), -wi, ~safe))
            kept = np.sort(rank[:k])
            movers = kept[kept >= k]
            holes = np.setdiff1d(np.arange(k), kept)
            w_out[i, h, :n], p_out[i, h, :n] = 0.0, -1
            w_out[i, h, :k], p_out[i, h, :k] = wi[:k], pi[:k]
            w_out[i, h, holes], p_out[i, h, holes] = wi[movers], pi[movers]
            src = torch.from_numpy(table[i, movers // page].astype(np.int64) * page + movers % page).cuda()
            dst = torch.from_numpy(table[i, holes // page].astype(np.int64) * page + holes % page).cuda()
            heads = slice(h, h + 1) if w.shape[1] > 1 else slice(None)
            for pool, old in ((k_pool, s["k_pool"]), (v_pool, s["v_pool"])):
                pool[dst // page, dst % page, heads] = old[src // page, src % page, heads]
    return (k_pool, v_pool, torch.from_numpy(w_out).cuda(), torch.from_numpy(p_out).cuda(),
            torch.from_numpy(np.minimum(lens, case["budget"])).cuda())
