"""The decode-step operators where numbers, shapes and callers are at their limits, against the 64-bit forms."""
import math
import subprocess
import sys

import pytest
import torch

import paged_decode_oracle as oracle
from conftest import ROOT
from test_gpu_paged_decode import DEV, _attend_case, _attend_tolerance

from tair_kvcache_b200 import _cabi
from tair_kvcache_b200.kernel import (batch_append_kv_pages, batch_attend_kv_pages, batch_evict_kv_pages,
                                      rotary_frequencies)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("nats", [12, 16, 18, 24])
@pytest.mark.parametrize("hq,hkv,window", [(4, 1, 0), (12, 1, 0), (8, 2, 5000)])  # eight rows, sixteen, a late sink
def test_attend_with_a_sink_whose_value_is_zero(dtype, nats, hq, hkv, window):
    """One key wins by `nats` and has the value zero: the output is made of the small probabilities alone.  Tolerance: the
    one of ordinary cases, whose spread is here that of the small ones, and in fp16 the 2^-40 of the largest probability that
    the two halves resolve, for each token."""
    n, dim = 8193, 64
    q, k_pool, v_pool, table, lens = _attend_case(nats, [n], hq, hkv, dim, dtype, poison=False)
    q = torch.ones_like(q)
    k_pool = (k_pool * 0.05).clone()
    sink = (table[0, n // 2 // 16].long(), n // 2 % 16)
    k_pool[sink] = nats / 8.0  # 64 elements of it times 1 / 8
    v_pool = (v_pool.abs() * 64).clone()
    v_pool[sink] = 0.0
    want, _, _, _, spread, size = oracle.attend(q, k_pool, v_pool, table, lens, 0.125, window)
    got = batch_attend_kv_pages(q.to(DEV), k_pool.to(DEV), v_pool.to(DEV), table.to(DEV), lens.to(DEV), window=window)
    tol = _attend_tolerance(want, spread, size, n, dtype)
    if dtype == "fp16":
        t = torch.arange(max(0, n - window) if window else 0, n)
        total = v_pool[table[0, t // 16].long(), t % 16].double().abs().sum(dim=0)  # [hkv, dim]
        tol = tol + 2.0 ** -40 * total.repeat_interleave(hq // hkv, dim=0)
    off = (got.cpu().double() - want).abs()
    assert (off <= tol).all(), ((off / tol).max(), (off / want.abs()).max())
    assert (want.abs() > 0).all() and math.isfinite(tol.max())


@pytest.mark.parametrize("shim", [True, False])
def test_attend_with_a_window_beyond_32_bits(shim, monkeypatch):
    if not shim:
        monkeypatch.setattr(_cabi, "shim", lambda: None)
    q, k_pool, v_pool, table, lens = (t.to(DEV) for t in _attend_case(31, [700, 30], 8, 2, 64, "bf16"))
    want = batch_attend_kv_pages(q, k_pool, v_pool, table, lens)
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 63):
        assert torch.equal(batch_attend_kv_pages(q, k_pool, v_pool, table, lens, window=window), want), window


def test_one_token_views_with_odd_strides():
    """The stride of an axis of length one may be anything; these are no multiple of the four bytes a query is read by."""
    dim, hq, hkv = 64, 4, 2
    q, k_pool, v_pool, table, lens = (t.to(DEV) for t in _attend_case(5, [90], hq, hkv, dim, "bf16"))
    want = batch_attend_kv_pages(q, k_pool, v_pool, table, lens)
    odd = torch.empty(hq * dim + 1, dtype=torch.bfloat16, device=DEV)[:hq * dim].as_strided((1, hq, dim), (hq * dim + 1, dim, 1))
    odd.copy_(q)
    assert torch.equal(batch_attend_kv_pages(odd, k_pool, v_pool, table, lens), want)
    kv = torch.randn(1, hkv, dim, device=DEV).to(torch.bfloat16)
    odd_kv = torch.empty(hkv * dim, dtype=torch.bfloat16, device=DEV).as_strided((1, hkv, dim), (7, dim, 1))
    odd_kv.copy_(kv)
    slot, position = torch.tensor([20], device=DEV), torch.tensor([89], device=DEV)
    inv_freq, _ = rotary_frequencies(dim, device=DEV)
    results = []
    for query, key in ((q, kv), (odd, odd_kv)):
        pools = torch.zeros_like(k_pool), torch.zeros_like(v_pool)
        results.append((batch_append_kv_pages(query, key, key, position, slot, *pools, inv_freq), *pools))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def _decode_loop(steps, batch, hq, hkv, dim, width, page, seed):
    """Pools with room for two caches of the same sequences, and for each step the new tokens' queries, keys and values."""
    gen = torch.Generator().manual_seed(seed)
    pages = 2 * batch * width
    pools = [torch.zeros(pages, page, hkv, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    tables = torch.randperm(pages, generator=gen).to(torch.int32).view(2, batch, width)
    qkv = torch.randn(steps, batch, hq + 2 * hkv, dim, generator=gen).to(torch.bfloat16)
    return pools, tables, qkv


@pytest.mark.parametrize("hw", [1, 2])
def test_a_cache_bounded_to_a_window_attends_what_the_window_does(hw):
    """budget = recent = W and no window, against an unbounded cache in order and window W: the same tokens, so the same
    attention - the tokens come in another order, so each within its own tolerance of the 64-bit form."""
    steps, batch, hq, hkv, dim, width, page, w = 70, 2, 8, 2, 64, 10, 8, 21
    (k_pool, v_pool), tables, qkv = _decode_loop(steps, batch, hq, hkv, dim, width, page, 3)
    whole, bounded = tables.to(DEV)
    inv_freq, _ = rotary_frequencies(dim, device=DEV)
    lens = torch.zeros(batch, dtype=torch.int32, device=DEV)
    weights = torch.zeros(batch, hw, width * page, device=DEV)
    positions = torch.full((batch, hw, width * page), -1, dtype=torch.int32, device=DEV)
    row = torch.arange(batch, device=DEV)
    moved = False
    for step in range(steps):
        q, k, v = qkv[step].to(DEV).split([hq, hkv, hkv], dim=1)
        at = torch.full((batch,), step, device=DEV)
        batch_append_kv_pages(None, k, v, at, whole[row, at // page].long() * page + at % page, k_pool, v_pool, inv_freq)
        to = lens.long()
        q = batch_append_kv_pages(q, k, v, at, bounded[row, to // page].long() * page + to % page, k_pool, v_pool, inv_freq)
        positions[row, :, to] = step
        lens = batch_evict_kv_pages(k_pool, v_pool, bounded, lens + 1, weights, positions, w, recent=w)
        got = batch_attend_kv_pages(q, k_pool, v_pool, bounded, lens, weights=weights)
        windowed = batch_attend_kv_pages(q, k_pool, v_pool, whole, torch.full_like(lens, step + 1), window=w)
        n = min(step + 1, w)
        assert lens.tolist() == [n] * batch
        assert (positions[..., :n].sort(dim=2).values == torch.arange(step + 1 - n, step + 1, device=DEV)).all()
        moved = moved or not (positions[..., :n].diff(dim=2) == 1).all()
        want, _, _, _, spread, size = oracle.attend(q.cpu(), k_pool.cpu(), v_pool.cpu(), tables[0],
                                                    torch.full((batch,), step + 1), dim ** -0.5, w)
        tol = _attend_tolerance(want, spread, size, w, "bf16")
        for out in (got, windowed):
            assert ((out.cpu().double() - want).abs() <= tol).all()
    assert moved  # or there was nothing to tell apart


def test_a_window_goes_by_slots_after_an_eviction():
    """What the documentation says of a window over a cache that was evicted from: the last slots, whatever they hold."""
    q, k_pool, v_pool, table, lens = _attend_case(9, [150, 90], 8, 2, 64, "bf16", poison=False)
    dk, dv, dt = k_pool.to(DEV), v_pool.to(DEV), table.to(DEV)
    weights = torch.rand(2, 2, table.shape[1] * 16, generator=torch.Generator().manual_seed(2)).to(DEV)
    positions = torch.arange(weights.shape[2], dtype=torch.int32, device=DEV).expand_as(weights).contiguous()
    new = batch_evict_kv_pages(dk, dv, dt, lens.to(DEV), weights, positions, 60, 10)
    assert not (positions[0, 0, :60].diff() > 0).all()
    for window in (0, 25):
        want, _, _, _, spread, size = oracle.attend(q, dk.cpu(), dv.cpu(), table, new.cpu(), 0.125, window)
        got = batch_attend_kv_pages(q.to(DEV), dk, dv, dt, new, window=window)
        assert ((got.cpu().double() - want).abs() <= _attend_tolerance(want, spread, size, 60, "bf16")).all()


@pytest.mark.parametrize("heads", ["kv", "one"])
@pytest.mark.parametrize("window", [0, 100])
def test_weights_of_bad_pages_are_carried_over(heads, window):
    """With separate arrays: attended slots get old + received, slots of pages outside the pool their old weight, slots out of
    the range nothing.  The bound is that of the accumulation's own test."""
    lens = [170, 300, 64]
    q, k_pool, v_pool, table, n = _attend_case(15, lens, 8, 2, 64, "bf16", poison=False)
    table[0, 9], table[1, 4], table[1, 17], table[2, :4] = -1, k_pool.shape[0], 2 ** 31 - 1, -7
    hw = 2 if heads == "kv" else 1
    before = torch.rand(3, hw, table.shape[1] * 16, generator=torch.Generator().manual_seed(1))
    out = torch.full_like(before, -3.0).to(DEV)
    dk, dv = k_pool.to(DEV), v_pool.to(DEV)
    batch_attend_kv_pages(q.to(DEV), dk, dv, table.to(DEV), n.to(DEV), window=window, weights=before.to(DEV), weights_out=out)
    _, _, probs, firsts, _, size = oracle.attend(q, k_pool, v_pool, table, n, 0.125, window)
    want, slack = torch.full(before.shape, -3.0, dtype=torch.float64), torch.zeros(before.shape, dtype=torch.float64)
    for i, p in enumerate(probs):
        t = slice(firsts[i], firsts[i] + p.shape[1])
        mass = p.view(hw, 8 // hw, -1).sum(dim=1)
        want[i, :, t] = before[i, :, t].double() + mass
        slack[i, :, t] = mass * (2 * (2.0 ** -21 * size[i].max() + 2.0 ** -17) + 2.0 ** -18) + 2.0 ** -23 * want[i, :, t]
    assert ((out.cpu().double() - want).abs() <= slack).all()
    bad = (table < 0) | (table >= k_pool.shape[0])
    for i, page in bad.nonzero().tolist():
        t = [t for t in range(page * 16, page * 16 + 16) if firsts[i] <= t < lens[i]]
        assert torch.equal(out[i, :, t].cpu(), before[i, :, t])


@pytest.mark.parametrize("tokens,budget,page", [(64, 10, 16), (5000, 700, 16), (400000, 20000, 64)])  # one CTA, a cluster, uncached
def test_more_protected_slots_than_the_budget(tokens, budget, page):
    """Positions that occur four times: more slots are protected than fit.  All of them rank equal, whatever their weights, so
    the lowest stay; unprotected ones go, infinite and NaN weights among them."""
    recent = budget // 2  # protects 4 * recent slots
    gen = torch.Generator().manual_seed(tokens)
    width = -(-tokens // page)
    k_pool = torch.randn(width, page, 1, 8, generator=gen).to(torch.bfloat16)
    v_pool = torch.randn(width, page, 1, 8, generator=gen).to(torch.bfloat16)
    table = torch.arange(width, dtype=torch.int32)[None]
    positions = torch.zeros(1, 1, width * page, dtype=torch.int32)
    positions[0, 0, :tokens] = (torch.arange(tokens) // 4)[torch.randperm(tokens, generator=gen)].int()
    weights = torch.rand(1, 1, width * page, generator=gen)
    weights[0, 0, ::7], weights[0, 0, 3::11] = math.inf, math.nan
    safe = positions[0, 0, :tokens] > positions[0, 0, :tokens].max() - recent
    kept = safe.nonzero()[:budget, 0]
    assert safe.sum() > budget
    low = set(range(budget))
    holes, movers = sorted(low - set(kept.tolist())), [t for t in kept.tolist() if t >= budget]
    source = torch.arange(budget)
    source[holes] = torch.tensor(movers)
    dk, dv, dw, dp = k_pool.to(DEV), v_pool.to(DEV), weights.to(DEV), positions.to(DEV)
    lens = batch_evict_kv_pages(dk, dv, table.to(DEV), torch.tensor([tokens], dtype=torch.int32, device=DEV), dw, dp, budget, recent)
    assert lens.tolist() == [budget]
    assert torch.equal(dp[0, 0, :budget].cpu(), positions[0, 0, source])
    assert torch.equal(dw[0, 0, :budget].cpu().view(torch.int32), weights[0, 0, source].view(torch.int32))
    for got, old in ((dk, k_pool), (dv, v_pool)):
        assert torch.equal(got.cpu().view(-1, 8)[:budget].view(torch.int16), old.view(-1, 8)[source].view(torch.int16))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (24, 2)])  # eight rows, sixteen
@pytest.mark.parametrize("n", [50, 3000])              # whole, and cut and joined
def test_attend_values_that_are_not_finite(n, hq, hkv, dtype):
    """An element of an attended value that is infinite or NaN stays in its element and its KV head; one that is not
    attended - before the window - is not seen at all."""
    q, k_pool, v_pool, table, lens = _attend_case(n, [n], hq, hkv, 64, dtype, q_scale=0.5)
    for t, head, element, value in ((n - 3, 0, 5, math.inf), (n - 20, 0, 6, -math.inf), (n - 7, 1, 7, math.nan), (n - 49, 0, 9, math.nan)):
        v_pool[table[0, t // 16].long(), t % 16, head, element] = value
    window = 40
    got = batch_attend_kv_pages(q.to(DEV), k_pool.to(DEV), v_pool.to(DEV), table.to(DEV), lens.to(DEV), window=window).cpu()
    finite = torch.ones(1, hq, 64, dtype=torch.bool)
    finite[:, :hq // 2, 5:7] = False
    finite[:, hq // 2:, 7] = False
    assert torch.equal(got.isfinite(), finite)
    want, _, _, _, spread, size = oracle.attend(q, k_pool, v_pool.nan_to_num(0.0, posinf=0.0, neginf=0.0), table, lens, 0.125, window)
    assert ((got.double() - want).abs() <= _attend_tolerance(want, spread, size, window, dtype))[finite].all()
    whole = batch_attend_kv_pages(q.to(DEV), k_pool.to(DEV), v_pool.to(DEV), table.to(DEV), lens.to(DEV)).cpu()
    finite[:, :hq // 2, 9] = False  # the last one is attended now
    assert torch.equal(whole.isfinite(), finite)


_FIRST_CALL = """
import sys
sys.path.insert(0, %(root)r)
import torch
import tair_kvcache_b200
from tair_kvcache_b200.kernel import batch_append_kv_pages, batch_attend_kv_pages, batch_evict_kv_pages, rotary_frequencies
dev = torch.device("cuda:0")
gen = torch.Generator().manual_seed(0)
k, v = (torch.randn(%(pages)d, 16, 2, 64, generator=gen).to(torch.bfloat16).to(dev) for _ in range(2))
qkv = torch.randn(1, 8, 64, generator=gen).to(torch.bfloat16).to(dev)
table = torch.arange(%(pages)d, dtype=torch.int32, device=dev)[None]
n = %(pages)d * 16
lens = torch.tensor([n], dtype=torch.int32, device=dev)
weights = torch.rand(1, 2, n, generator=gen).to(dev)
positions = torch.arange(n, dtype=torch.int32).expand(1, 2, n).contiguous().to(dev)
at = torch.tensor([n - 1], device=dev)
inv_freq, _ = rotary_frequencies(64, device=dev)
start = [t.clone() for t in (k, v, weights, positions)]

def step():
    q = batch_append_kv_pages(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], at, at, k, v, inv_freq)
    out = batch_attend_kv_pages(q, k, v, table, lens, weights=weights)
    return q, out, batch_evict_kv_pages(k, v, table, lens, weights, positions, n // 3, 5)

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = step()
graph.replay()
first = [t.clone() for t in (*captured, k, v, weights, positions)]
for t, old in zip((k, v, weights, positions), start):
    t.copy_(old)
assert all(torch.equal(a, b) for a, b in zip(first, (*step(), k, v, weights, positions)))
print("captured first")
"""


@pytest.mark.parametrize("pages", [4, 2000])  # units whole, one CTA a head; cut and joined, a cluster of sixteen
def test_the_first_call_of_a_process_may_be_captured(pages):
    """Kernels, attributes and the device's answers are all met for the first time while a stream captures."""
    proc = subprocess.run([sys.executable, "-c", _FIRST_CALL % dict(root=ROOT, pages=pages)], stdout=subprocess.PIPE,
                          stderr=subprocess.STDOUT, text=True, timeout=300)
    assert proc.returncode == 0 and "captured first" in proc.stdout, proc.stdout[-2000:]
