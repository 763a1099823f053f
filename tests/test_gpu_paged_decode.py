"""The decode-step operators against their 64-bit forms: rotary append, paged attention, eviction by attention weight."""
import math

import numpy as np
import pytest
import torch

import paged_decode_oracle as oracle

import tair_kvcache_b200  # noqa: F401
from tair_kvcache_b200 import _cabi
from tair_kvcache_b200.kernel import (batch_append_kv_pages, batch_attend_kv_pages, batch_evict_kv_pages,
                                      batch_gather_kv_pages, batch_scatter_kv_pages, rotary_frequencies)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _bits(t):
    return t.contiguous().view(torch.int16)


def _status():
    return torch.zeros(4, dtype=torch.int32, device=DEV)


# ----------------------------------------------------------------------------------------------------------------
# append
# ----------------------------------------------------------------------------------------------------------------
def _append_case(seed, tokens, hq, hkv, dim, dtype, page=16, layout="nhd", far=100000):
    gen = torch.Generator().manual_seed(seed)
    pages = -(-tokens // page) + 3
    k_pool, v_pool = oracle.make_pools(gen, pages, page, hkv, dim, dtype, layout)
    qkv = torch.randn(tokens, hq + 2 * hkv, dim, generator=gen).to(oracle.DTYPES[dtype])
    positions = torch.randint(0, far, (tokens,), generator=gen)
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    return qkv, positions, slots, k_pool, v_pool


def _append_tolerance(exact, x, half, interleaved, factor, dtype):
    """Half a step of the type's rounding (half the smallest subnormal where fp16 runs out), and for the rotated pair
    the error of cosine and sine - 2 pi 2^-25 from the angle in turns, 2^-22 from sincospi - and of three roundings in
    32 bits, together below 2^-20 of |x| + |y|."""
    t = oracle.DTYPES[dtype]
    tol = exact.abs() * (torch.finfo(t).eps / 2) + (2.0 ** -25 if dtype == "fp16" else 0.0)
    x = x.double().abs()
    pair = torch.zeros_like(x)
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    pair[..., first] = pair[..., second] = x[..., first] + x[..., second]
    return tol + 2.0 ** -20 * factor * pair


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rd,page,layout", [
    (1, 32, 8, 128, 128, 16, "nhd"),      # one token: its heads are shared by two CTAs
    (1, 1, 1, 8, 2, 1, "nhd"),            # the smallest of everything
    (7, 4, 2, 64, 32, 16, "hnd"),         # half of the head rotated
    (33, 15, 3, 80, 80, 48, "nhd"),       # odd head counts, 40 pairs
    (150, 5, 5, 96, 66, 8, "nhd"),        # 33 pairs: no piece wider than one element
    (150, 8, 2, 100, 20, 8, "hnd"),       # pieces of two elements
    (5, 2, 1, 72, 24, 16, "nhd"),         # pieces of four
    (3, 2, 2, 7, 6, 5, "nhd"),            # an odd head dimension
    (9, 3, 1, 256, 0, 64, "nhd"),         # nothing is rotated
    (2, 130, 2, 128, 64, 16, "nhd"),      # many heads: several rounds of a CTA
    (300, 4, 1, 1024, 1024, 16, "nhd"),   # the largest head
])
def test_append_rotates_and_writes(tokens, hq, hkv, dim, rd, page, layout, interleaved, dtype):
    qkv, positions, slots, k_pool, v_pool = _append_case(tokens + dim, tokens, hq, hkv, dim, dtype, page, layout)
    inv_freq = (10000.0 ** (-torch.arange(rd // 2, dtype=torch.float64) * 2 / max(rd, 1))).float()
    factor = 1.0 if rd % 4 else 1.2079441541679836
    dk, dv = oracle.on_device(k_pool, DEV), oracle.on_device(v_pool, DEV)
    d = qkv.to(DEV)
    q, k, v = d[:, :hq], d[:, hq:hq + hkv], d[:, hq + hkv:]  # strided slices of one tensor
    got = batch_append_kv_pages(q, k, v, positions.to(DEV), slots.to(DEV), dk, dv, inv_freq.to(DEV),
                                interleaved=interleaved, attention_factor=factor)
    want_q = oracle.rotate(qkv[:, :hq], positions, inv_freq, interleaved, factor)
    tol = _append_tolerance(want_q, qkv[:, :hq], rd // 2, interleaved, factor, dtype)
    assert ((got.cpu().double() - want_q).abs() <= tol).all()
    want_k = oracle.rotate(qkv[:, hq:hq + hkv], positions, inv_freq, interleaved, factor)
    tol = _append_tolerance(want_k, qkv[:, hq:hq + hkv], rd // 2, interleaved, factor, dtype)
    at = (slots // page, slots % page)
    assert ((dk.cpu()[at].double() - want_k).abs() <= tol).all()
    # elements that are not rotated, the values, and every other row of the pools: bit by bit
    assert torch.equal(_bits(got.cpu()[..., rd:]), _bits(qkv[:, :hq, rd:]))
    assert torch.equal(_bits(dv.cpu()[at]), _bits(qkv[:, hq + hkv:]))
    others = torch.ones(k_pool.shape[:2], dtype=torch.bool)
    others[at] = False
    assert torch.equal(_bits(dk.cpu()[others]), _bits(k_pool[others]))
    assert torch.equal(_bits(dv.cpu()[others]), _bits(v_pool[others]))


def test_append_far_positions_keep_their_angle():
    """Positions near 2^31: the angle in 64 bits, reduced before it is rounded (2^31 * 2^-53 turns are lost at most)."""
    qkv, _, slots, k_pool, v_pool = _append_case(3, 64, 2, 1, 64, "fp16")
    positions = torch.tensor([2 ** 31 - 1 - 7 * i for i in range(64)])
    inv_freq, factor = rotary_frequencies(64, scaling="yarn", factor=32.0, device=DEV)
    dk, dv = k_pool.to(DEV), v_pool.to(DEV)
    d = qkv.to(DEV)
    got = batch_append_kv_pages(d[:, :2], d[:, 2:3], d[:, 3:], positions.to(torch.int32).to(DEV),
                                slots.to(torch.int32).to(DEV), dk, dv, inv_freq, attention_factor=factor)
    want = oracle.rotate(qkv[:, :2], positions, inv_freq.cpu(), False, factor)
    tol = _append_tolerance(want, qkv[:, :2], 32, False, factor, "fp16")
    tol = tol + 2.0 ** -21 * factor * qkv.double().abs().max() * 2  # 2 pi * 2^-22 turns of the product's rounding
    assert ((got.cpu().double() - want).abs() <= tol).all()


def test_append_padding_and_bad_slots():
    qkv, positions, slots, k_pool, v_pool = _append_case(5, 6, 2, 2, 64, "bf16", page=16)
    slots[1], slots[3], slots[4] = -1, -2, k_pool.shape[0] * 16  # padding, below and just behind the pool
    inv_freq, _ = rotary_frequencies(64, device=DEV)
    d = qkv.to(DEV)
    for slot_type in (torch.int64, torch.int32):
        dk, dv = k_pool.to(DEV), v_pool.to(DEV)
        status = _status()
        got = batch_append_kv_pages(d[:, :2], d[:, 2:4], d[:, 4:], positions.to(DEV), slots.to(slot_type).to(DEV), dk, dv,
                                    inv_freq, status=status)
        assert status.tolist()[:2] == [2, 5]
        keep = torch.tensor([0, 2, 5])
        others = torch.ones(k_pool.shape[:2], dtype=torch.bool)
        others[slots[keep] // 16, slots[keep] % 16] = False
        assert torch.equal(_bits(dk.cpu()[others]), _bits(k_pool[others]))
        assert torch.equal(_bits(dv.cpu()[slots[keep] // 16, slots[keep] % 16]), _bits(qkv[keep, 4:]))
        want = oracle.rotate(qkv[:, :2], positions, inv_freq.cpu(), False, 1.0)  # padded queries too
        assert ((got.cpu().double() - want).abs() <= _append_tolerance(want, qkv[:, :2], 32, False, 1.0, "bf16")).all()
    # a slot beyond 32 bits is not taken for a small one
    status = _status()
    dk, dv = k_pool.to(DEV), v_pool.to(DEV)
    far = torch.full((6,), (1 << 32) + 5, dtype=torch.int64, device=DEV)
    batch_append_kv_pages(None, d[:, 2:4], d[:, 4:], positions.to(DEV), far, dk, dv, inv_freq, status=status)
    assert status.tolist()[:2] == [6, 6] and torch.equal(_bits(dk.cpu()), _bits(k_pool))


def test_append_in_place_without_queries_and_from_a_list():
    qkv, positions, slots, k_pool, v_pool = _append_case(9, 40, 4, 2, 128, "bf16")
    inv_freq, _ = rotary_frequencies(128, device=DEV)
    d = qkv.to(DEV)
    dk, dv = k_pool.to(DEV), v_pool.to(DEV)
    apart = batch_append_kv_pages(d[:, :4], d[:, 4:6], d[:, 6:], positions.to(DEV), slots.to(DEV), dk, dv, inv_freq)
    dk2, dv2, d2 = k_pool.to(DEV), v_pool.to(DEV), qkv.to(DEV)
    same = batch_append_kv_pages(d2[:, :4], d2[:, 4:6], d2[:, 6:], positions.to(DEV), slots.tolist(), dk2, dv2, inv_freq,
                                 query_out=d2[:, :4])
    assert same.data_ptr() == d2.data_ptr()
    assert torch.equal(_bits(same), _bits(apart)) and torch.equal(dk, dk2) and torch.equal(dv, dv2)
    dk3, dv3 = k_pool.to(DEV), v_pool.to(DEV)
    assert batch_append_kv_pages(None, d[:, 4:6], d[:, 6:], positions.to(DEV), slots.to(DEV), dk3, dv3, inv_freq) is None
    assert torch.equal(dk, dk3) and torch.equal(dv, dv3)
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    assert batch_append_kv_pages(d[:0, :4], d[:0, 4:6], d[:0, 6:], none, none, dk3, dv3, inv_freq).shape == (0, 4, 128)


# ----------------------------------------------------------------------------------------------------------------
# attend
# ----------------------------------------------------------------------------------------------------------------
def _attend_case(seed, lens, hq, hkv, dim, dtype, page=16, layout="nhd", poison=True, q_scale=2.0):
    gen = torch.Generator().manual_seed(seed)
    width = max(1, -(-max(max(lens), 1) // page))
    pages = len(lens) * width + 2
    k_pool, v_pool = oracle.make_pools(gen, pages, page, hkv, dim, dtype, layout)
    table = torch.randperm(pages, generator=gen)[:len(lens) * width].to(torch.int32).view(len(lens), width)
    if poison:  # everything that no sequence holds is NaN or infinity
        used = torch.zeros(pages, page, dtype=torch.bool)
        for i, n in enumerate(lens):
            t = torch.arange(n)
            used[table[i].long()[t // page], t % page] = True
        k_pool[~used] = math.nan
        v_pool[~used] = math.inf
    q = (torch.randn(len(lens), hq, dim, generator=gen) * q_scale).to(oracle.DTYPES[dtype])
    return q, k_pool, v_pool, table, torch.tensor(lens, dtype=torch.int32)


def _attend_tolerance(out, spread, size, longest, dtype):
    """Output rounding of half a step; and, relative to sum p |v|: scores in 32 bits, off by 2^-21 of sum |q||k| for a
    product of at most 256 terms added by the matrix instruction, twice for numerator and denominator; the exponent's
    argument, below 64 in magnitude, rounded to 2^-18; p in two halves, 2^-16; 16 tokens a step added up in 32 bits,
    2^-24 for each step of a share and join, at most longest / 16."""
    t = oracle.DTYPES[dtype]
    rel = 2 * (2.0 ** -21 * size + 2.0 ** -18) + 2.0 ** -16 + 2.0 ** -24 * (longest / 16 + 64)
    return out.abs() * (torch.finfo(t).eps / 2) + rel[..., None] * spread + (2.0 ** -25 if dtype == "fp16" else 0.0)


def _check_attend(q, k_pool, v_pool, table, lens, dtype, window=0, scale=None, **more):
    dim = q.shape[2]
    scale_ = dim ** -0.5 if scale is None else scale
    want, lse, probs, firsts, spread, size = oracle.attend(q, k_pool, v_pool, table, lens, scale_, window)
    dk, dv = oracle.on_device(k_pool, DEV), oracle.on_device(v_pool, DEV)
    got_lse = torch.full(q.shape[:2], 7.0, device=DEV)
    got = batch_attend_kv_pages(q.to(DEV), dk, dv, table.to(DEV), lens.to(DEV), scale=scale, window=window, lse=got_lse,
                                **more)
    tol = _attend_tolerance(want, spread, size, int(lens.max()), dtype)
    bad = (got.cpu().double() - want).abs() > tol
    assert not bad.any() and not got.isnan().any(), (bad.nonzero()[:5], got.isnan().sum())
    empty = lse == -math.inf
    assert (got_lse.cpu()[empty] == -math.inf).all() and (got.cpu()[empty] == 0).all()
    # lse in 32 bits: score error as above, relative rounding of a number below 256
    assert ((got_lse.cpu().double() - lse)[~empty].abs() <= (2.0 ** -20 * size + 2.0 ** -15)[~empty]).all()
    return got, probs, firsts, size, (dk, dv)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lens,hq,hkv,dim,page,layout,window", [
    ([1], 1, 1, 8, 1, "nhd", 0),
    ([0], 4, 2, 64, 16, "nhd", 0),
    ([0, 1, 0, 17, 64, 65, 0], 8, 8, 128, 16, "nhd", 0),        # one query head per KV head, empty rows
    ([100], 32, 8, 128, 16, "nhd", 0),
    ([1000, 3, 511, 2049], 32, 4, 128, 16, "hnd", 0),           # a group of eight
    ([300, 777], 36, 4, 128, 32, "nhd", 0),                     # nine: the sixteen-row form
    ([300, 777, 1], 16, 1, 64, 64, "nhd", 0),                   # sixteen
    ([130, 257], 71, 1, 64, 16, "nhd", 0),                      # more heads than a row tile holds
    ([640, 33], 34, 2, 128, 16, "hnd", 0),                      # seventeen: a row tile of one
    ([500, 1500], 6, 2, 256, 16, "nhd", 0),
    ([500, 150], 24, 2, 256, 8, "hnd", 0),
    ([400, 90, 31], 15, 3, 80, 48, "hnd", 0),                   # padded head dimension, odd page size
    ([400, 90, 31], 10, 2, 72, 7, "nhd", 0),
    ([400, 90, 31, 0], 10, 2, 96, 16, "nhd", 50),               # windows that begin inside a page and a step
    ([5000], 8, 1, 128, 16, "nhd", 4096),
    ([9000], 8, 1, 128, 32, "nhd", 0),                          # one sequence over many CTAs
    ([40] * 70 + [700] * 3, 8, 4, 64, 16, "nhd", 0),            # many sequences per CTA
    ([5] * 300, 2, 1, 32, 16, "nhd", 0),                        # more sequences than a CTA has threads
    ([77, 150], 4, 2, 64, 4, "nhd", 0),                         # four, two and one tokens to a TMA box
    ([77, 150], 4, 2, 128, 2, "hnd", 20),
    ([333], 4, 2, 136, 1, "nhd", 0),
    ([333, 70], 4, 2, 200, 12, "nhd", 69),
    ([700, 13, 0, 260], 32, 8, 64, 16, "nhd", 0),               # steps of two heads
    ([700, 13, 0, 260], 48, 4, 80, 16, "nhd", 0),               # of four, sixteen-row tiles
    ([700, 13, 0, 260], 12, 12, 96, 64, "nhd", 100),
    ([9000], 68, 4, 80, 5, "nhd", 0),                           # seventeen heads to a group: two row tiles
])
def test_attend_matches_the_definition(lens, hq, hkv, dim, page, layout, window, dtype):
    case = _attend_case(sum(lens) + dim, lens, hq, hkv, dim, dtype, page, layout)
    _check_attend(*case, dtype, window=window)


@pytest.mark.parametrize("heads", ["kv", "one"])
@pytest.mark.parametrize("lens,hq,hkv,dim,window", [
    ([0, 1, 63, 64, 65], 4, 2, 64, 0),
    ([3000, 10], 32, 8, 128, 0),
    ([3000, 10], 18, 1, 128, 100),
    ([1200, 513, 100], 20, 2, 80, 700),
    ([20000], 8, 1, 64, 0),
    ([5000, 77, 3], 24, 8, 64, 0),
    ([5000, 77, 3], 40, 4, 80, 333),
])
def test_attend_accumulates_weights(lens, hq, hkv, dim, window, heads):
    q, k_pool, v_pool, table, n = _attend_case(sum(lens), lens, hq, hkv, dim, "bf16")
    cap = table.shape[1] * 16
    hw = hkv if heads == "kv" else 1
    before = torch.rand(len(lens), hw, cap + 5, generator=torch.Generator().manual_seed(1))
    untouched = torch.full_like(before, -3.0)
    out = untouched.to(DEV)
    _, probs, firsts, size, _ = _check_attend(q, k_pool, v_pool, table, n, "bf16", window=window, weights=before.to(DEV),
                                              weights_out=out)
    want, slack = untouched.double(), torch.zeros(before.shape, dtype=torch.float64)
    for i, p in enumerate(probs):
        t = slice(firsts[i], firsts[i] + p.shape[1])
        mass = p.view(hw, hq // hw, -1).sum(dim=1)
        want[i, :, t] = before[i, :, t].double() + mass
        # p off by its score's and the sum's error and the exponent's argument, then sums in 32 bits
        slack[i, :, t] = mass * (2 * (2.0 ** -21 * size[i].max() + 2.0 ** -17) + 2.0 ** -18) + 2.0 ** -23 * want[i, :, t]
    assert ((out.cpu().double() - want).abs() <= slack).all()
    same = before.to(DEV)  # in place: the same numbers where attended, the old ones elsewhere
    batch_attend_kv_pages(q.to(DEV), oracle.on_device(k_pool, DEV), oracle.on_device(v_pool, DEV), table.to(DEV),
                          n.to(DEV), window=window, weights=same)
    assert torch.equal(same.cpu(), torch.where(untouched == out.cpu(), before, out.cpu()))


def test_attend_bad_pages_and_lengths_take_no_part():
    lens = [70, 200, 48]
    q, k_pool, v_pool, table, n = _attend_case(8, lens, 8, 2, 64, "bf16")
    table[1, 3], table[1, 7], table[2, 0] = -1, k_pool.shape[0], 2 ** 31 - 1
    table[2, 1], table[2, 2] = -5, -6           # nothing of sequence 2 is left
    n[0] = 100000                                # cut to the table's 13 pages
    k_pool, v_pool = k_pool.nan_to_num(0.5), v_pool.nan_to_num(0.5, posinf=0.25)
    status = _status()
    w = torch.zeros(3, 2, table.shape[1] * 16, device=DEV)
    _, probs, firsts, _, _ = _check_attend(q, k_pool, v_pool, table, n, "bf16", status=status, weights=w)
    assert status.tolist()[:2] == [2 + 3 + 1, 3]
    got = w.cpu().double()
    for i, p in enumerate(probs):
        assert torch.allclose(got[i, :, :p.shape[1]], p.view(2, 4, -1).sum(dim=1), rtol=1e-3, atol=1e-6)
    assert (got[1, :, 48:64] == 0).all() and (got[2] == 0).all()


def test_attend_infinite_and_nan_scores():
    q, k_pool, v_pool, table, n = _attend_case(2, [40, 40, 40], 2, 1, 16, "bf16", poison=False)
    k_pool, v_pool = k_pool.abs(), v_pool
    q = q.abs()
    k_pool[table[0, 0].long(), 3] = -math.inf                          # one token of -inf: as if it were not there
    for pg in table[1].long():
        k_pool[pg] = -math.inf                                         # all of them: zeros
    k_pool[table[2, 1].long(), 2, 0, 0] = math.nan                     # one NaN: NaN
    got = batch_attend_kv_pages(q.to(DEV), k_pool.to(DEV), v_pool.to(DEV), table.to(DEV), n.to(DEV))
    want, _, _, _, spread, size = oracle.attend(q[:1], k_pool.nan_to_num(0, neginf=-3e38), v_pool, table[:1], n[:1], 0.25)
    assert ((got[:1].cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -12 * spread).all()
    assert (got[1] == 0).all() and got[2].isnan().all()


def test_attend_large_scores_and_a_late_maximum():
    """The running maximum moves at every step and the largest score comes last; scores in the thousands."""
    q, k_pool, v_pool, table, n = _attend_case(4, [2000], 4, 1, 64, "bf16", poison=False)
    q = torch.ones_like(q)
    for t in range(2000):
        k_pool[table[0, t // 16].long(), t % 16] = float(t // 8)
    got = batch_attend_kv_pages(q.to(DEV), k_pool.to(DEV), v_pool.to(DEV), table.to(DEV), n.to(DEV), scale=0.125)
    want, _, _, _, spread, _ = oracle.attend(q, k_pool, v_pool, table, n, 0.125)
    # every score is a whole number of eighths below 2^24: exact; the maximum's distance from the others is exact too
    assert ((got.cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -15 * spread).all()


def test_attend_strided_queries_graph_and_streams():
    lens = [900, 30, 2500, 0, 64]
    q, k_pool, v_pool, table, n = _attend_case(6, lens, 16, 4, 128, "bf16")
    dk, dv, dt, dn = k_pool.to(DEV), v_pool.to(DEV), table.to(DEV), n.to(DEV)
    first = batch_attend_kv_pages(q.to(DEV), dk, dv, dt, dn)
    wide = torch.randn(5, 40, 128).to(torch.bfloat16).to(DEV)
    wide[:, 8:24] = q.to(DEV)
    wide_table = torch.full((5, dt.shape[1] + 9), -1, dtype=torch.int32, device=DEV)
    wide_table[:, :dt.shape[1]] = dt
    again = batch_attend_kv_pages(wide[:, 8:24], dk, dv, wide_table[:, :dt.shape[1]], dn)
    assert torch.equal(_bits(first), _bits(again))
    # two streams at once, several times: each call has its own workspace
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                o.append(batch_attend_kv_pages(wide[:, 8:24], dk, dv, dt, dn))
    torch.cuda.synchronize()
    assert all(torch.equal(_bits(first), _bits(o)) for os in outs for o in os)
    # captured, then replayed over other lengths and queries
    sq, sn = wide[:, 8:24].clone(), dn.clone()
    w = torch.zeros(5, 4, dt.shape[1] * 16, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = batch_attend_kv_pages(sq, dk, dv, dt, sn, weights=w)
    new_n = torch.tensor([1, 30, 2000, 0, 63], dtype=torch.int32)
    sq.copy_(q.flip(0).to(DEV))
    sn.copy_(new_n.to(DEV))
    graph.replay()
    graph.replay()
    want = batch_attend_kv_pages(q.flip(0).to(DEV), dk, dv, dt, new_n.to(DEV), weights=None)
    assert torch.equal(_bits(held), _bits(want))
    mass = w.sum(dim=(1, 2)).cpu()
    assert torch.allclose(mass, torch.tensor([32.0, 32.0, 32.0, 0.0, 32.0]), rtol=1e-4)


# ----------------------------------------------------------------------------------------------------------------
# evict
# ----------------------------------------------------------------------------------------------------------------
def _evict_case(seed, lens, hkv, hw, dim, dtype="bf16", page=16, layout="nhd", ties=False, mixed=True):
    gen = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    width = max(1, -(-max(lens) // page))
    pages = len(lens) * width + 2
    k_pool, v_pool = oracle.make_pools(gen, pages, page, hkv, dim, dtype, layout)
    table = torch.randperm(pages, generator=gen)[:len(lens) * width].to(torch.int32).view(len(lens), width)
    cap = width * page
    w = np.exp(2 * rng.standard_normal((len(lens), hw, cap))).astype(np.float32)
    if ties:
        w = rng.integers(0, 4, size=w.shape).astype(np.float32)
    pos = np.broadcast_to(np.arange(cap, dtype=np.int32), w.shape).copy()
    if mixed:
        for i, n in enumerate(lens):
            for h in range(hw):
                pos[i, h, :n] = rng.permutation(n)
    return k_pool, v_pool, table, torch.tensor(lens, dtype=torch.int32), w, pos


def _check_evict(k_pool, v_pool, table, n, w, pos, budget, recent, in_place=True):
    want = oracle.evict(k_pool, v_pool, table, n, w, pos, budget, recent)
    dk, dv = oracle.on_device(k_pool, DEV), oracle.on_device(v_pool, DEV)
    dw, dp = torch.from_numpy(w).to(DEV), torch.from_numpy(pos).to(DEV)
    more = {}
    if not in_place:
        more = dict(weights_out=torch.full_like(dw, -9.0), positions_out=torch.full_like(dp, -9))
    lens = batch_evict_kv_pages(dk, dv, table.to(DEV), n.to(DEV), dw, dp, budget, recent, **more)
    got_w, got_p = (dw, dp) if in_place else (more["weights_out"], more["positions_out"])
    assert np.array_equal(lens.cpu().numpy(), want[4])
    cap = table.shape[1] * k_pool.shape[1]
    for i in range(w.shape[0]):
        m = max(0, min(int(n[i]), cap))
        assert np.array_equal(got_p[i].cpu().numpy()[:, :m], want[3][i, :, :m]), i
        assert np.array_equal(got_w[i].cpu().numpy()[:, :m], want[2][i, :, :m], equal_nan=True), i
        rest_w, rest_p = (w, pos) if in_place else (np.full_like(w, -9.0), np.full_like(pos, -9))
        assert np.array_equal(got_w[i].cpu().numpy()[:, m:], rest_w[i, :, m:], equal_nan=True)
        assert np.array_equal(got_p[i].cpu().numpy()[:, m:], rest_p[i, :, m:])
    if not in_place:
        assert np.array_equal(dw.cpu().numpy(), w, equal_nan=True) and np.array_equal(dp.cpu().numpy(), pos)
    assert torch.equal(_bits(dk.cpu()), _bits(want[0])) and torch.equal(_bits(dv.cpu()), _bits(want[1]))


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lens,budget,recent,hkv,hw,dim,page,layout,ties", [
    ([2], 1, 0, 1, 1, 8, 1, "nhd", False),
    ([2], 1, 1, 1, 1, 8, 16, "nhd", True),
    ([0, 5, 10, 11, 40], 10, 3, 2, 2, 64, 16, "nhd", False),       # empty, under, at and over the budget
    ([257, 513, 100, 512], 256, 32, 3, 3, 80, 48, "hnd", True),    # ties across the threads of a CTA
    ([257, 513, 100, 512], 256, 32, 3, 1, 80, 48, "hnd", False),   # all heads together
    ([3001], 3000, 100, 8, 8, 128, 16, "nhd", False),              # one token over
    ([5000, 4096], 1024, 1024, 4, 4, 128, 16, "nhd", False),       # only the newest are kept
    ([7000], 6999, 0, 2, 1, 64, 64, "nhd", True),
    ([9000, 100], 77, 5, 1, 1, 256, 16, "nhd", True),              # over several CTAs, threshold among ties
])
def test_evict_matches_the_definition(lens, budget, recent, hkv, hw, dim, page, layout, ties, in_place):
    case = _evict_case(sum(lens), lens, hkv, hw, dim, page=page, layout=layout, ties=ties)
    _check_evict(*case, budget, recent, in_place)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("tokens", [131072, 360000, 500009])
def test_evict_one_long_sequence(tokens, in_place):
    """Over a whole cluster; the second fills its shared memory, the third does not fit."""
    case = _evict_case(tokens, [tokens], 1, 1, 8, page=64, ties=tokens % 2 == 1, mixed=False)
    _check_evict(*case, tokens // 3, 1000, in_place)


def test_evict_special_weights():
    """NaN ranks above all but the protected, zeros of both signs are equal, infinities and negative numbers in order."""
    k_pool, v_pool, table, n, w, pos = _evict_case(1, [64, 64, 64, 64], 1, 1, 8, mixed=False)
    w[0, 0, 40:50], w[0, 0, 3] = np.nan, -np.nan
    w[1, 0] = np.where(np.arange(w.shape[2]) % 2 == 0, 0.0, -0.0)
    w[2, 0] = -w[2, 0]
    w[2, 0, 5], w[2, 0, 60], w[2, 0, 61] = -np.inf, np.inf, -0.0
    w[3, 0] = 1.0                                       # all equal: the lowest slots stay, nothing moves
    for recent in (0, 4):
        _check_evict(k_pool, v_pool, table, n, w, pos, 16, recent)


def test_evict_bad_pages_and_lengths():
    k_pool, v_pool, table, n, w, pos = _evict_case(12, [200, 130], 2, 2, 64)
    table[0, 0], table[0, 9] = -1, k_pool.shape[0]
    n[1] = 100000                                        # cut to the table
    want = oracle.evict(k_pool, v_pool, table, n, w, pos, 64, 8)
    dk, dv, dw, dp, status = k_pool.to(DEV), v_pool.to(DEV), torch.from_numpy(w).to(DEV), torch.from_numpy(pos).to(DEV), _status()
    lens = batch_evict_kv_pages(dk, dv, table.to(DEV), n.to(DEV), dw, dp, 64, 8, status=status)
    assert lens.tolist() == [64, 64]
    assert torch.equal(_bits(dk.cpu()), _bits(want[0])) and torch.equal(_bits(dv.cpu()), _bits(want[1]))
    assert np.array_equal(dw.cpu().numpy(), want[2]) and np.array_equal(dp.cpu().numpy(), want[3])
    assert status[0].item() > 1 and status[1].item() == 2


def test_evict_captured_and_replayed():
    k_pool, v_pool, table, n, w, pos = _evict_case(21, [300, 500], 2, 2, 64)
    dk, dv, dt, dn = k_pool.to(DEV), v_pool.to(DEV), table.to(DEV), n.to(DEV)
    dw, dp = torch.from_numpy(w).to(DEV), torch.from_numpy(pos).to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens = batch_evict_kv_pages(dk, dv, dt, dn, dw, dp, 128, 16)
    graph.replay()
    want = oracle.evict(k_pool, v_pool, table, n, w, pos, 128, 16)
    assert lens.tolist() == [128, 128] and np.array_equal(dw.cpu().numpy(), want[2])
    assert torch.equal(_bits(dk.cpu()), _bits(want[0]))


# ----------------------------------------------------------------------------------------------------------------
# together
# ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shared", [False, True])
def test_decode_steps_with_a_bounded_cache(shared):
    """A prompt and forty decode steps of two sequences with a budget: append, attend with weights, evict; between two of
    them the blocks leave for a staging buffer and come back to other pages.  Each step's attention is checked against
    the tokens that the operators say are in the cache, kept here by position in plain tensors."""
    hq, hkv, dim, page, budget, recent, batch = 8, 2, 64, 16, 96, 16, 2
    gen = torch.Generator().manual_seed(17)
    width = 8
    pages = 40
    k_pool = torch.zeros(pages, page, hkv, dim, dtype=torch.bfloat16, device=DEV)
    v_pool = torch.zeros_like(k_pool)
    order = torch.randperm(pages, generator=gen)
    table = order[:batch * width].to(torch.int32).view(batch, width).to(DEV)
    spare = order[batch * width:2 * batch * width].to(torch.int32).view(batch, width).to(DEV)
    hw = 1 if shared else hkv
    weights = torch.zeros(batch, hw, width * page, device=DEV)
    positions = torch.full((batch, hw, width * page), -1, dtype=torch.int32, device=DEV)
    lens = torch.zeros(batch, dtype=torch.int32, device=DEV)
    inv_freq, factor = rotary_frequencies(dim, scaling="llama3", factor=8.0, device=DEV)
    keys, values = {}, {}  # (sequence, position) -> what was written

    def append(new, qkv):
        """new: per sequence the positions its next tokens have."""
        rows, pos, slots = [], [], []
        for b in range(batch):
            base = int(lens[b])
            for j, p in enumerate(new[b]):
                rows.append(len(rows))
                pos.append(p)
                t = base + j
                slots.append(int(table[b, t // page]) * page + t % page)
                positions[b, :, t] = p
            lens[b] += len(new[b])
        d = qkv.to(DEV)
        q = batch_append_kv_pages(d[:, :hq], d[:, hq:hq + hkv], d[:, hq + hkv:], torch.tensor(pos, device=DEV),
                                  torch.tensor(slots, dtype=torch.int32, device=DEV), k_pool, v_pool, inv_freq,
                                  attention_factor=factor)
        i = 0
        flat_k, flat_v = k_pool.view(-1, hkv, dim), v_pool.view(-1, hkv, dim)
        for b in range(batch):
            for p in new[b]:
                keys[b, p], values[b, p] = flat_k[slots[i]].cpu(), flat_v[slots[i]].cpu()
                want = oracle.rotate(qkv[i:i + 1, hq:hq + hkv], torch.tensor([p]), inv_freq.cpu(), False, factor)[0]
                tol = _append_tolerance(want, qkv[i, hq:hq + hkv], dim // 2, False, factor, "bf16")
                assert ((keys[b, p].double() - want).abs() <= tol).all()
                i += 1
        return q

    prompt = [list(range(90)), list(range(95))]
    qkv = torch.randn(185, hq + 2 * hkv, dim, generator=gen).to(torch.bfloat16)
    append(prompt, qkv)
    total = [90, 95]
    for step in range(40):
        qkv = torch.randn(batch, hq + 2 * hkv, dim, generator=gen).to(torch.bfloat16)
        q = append([[total[0]], [total[1]]], qkv)
        total = [t + 1 for t in total]
        old = weights.clone()
        out = batch_attend_kv_pages(q, k_pool, v_pool, table, lens, weights=weights)
        for b in range(batch):
            n = int(lens[b])
            for h in range(hq):
                kv = h // (hq // hkv)
                cached = positions[b, 0 if shared else kv, :n].tolist()
                assert len(set(cached)) == n and max(cached) == total[b] - 1
                k = torch.stack([keys[b, p][kv] for p in cached]).double()
                v = torch.stack([values[b, p][kv] for p in cached]).double()
                p = torch.softmax(k @ q[b, h].cpu().double() * dim ** -0.5, dim=0)
                want = p @ v
                assert ((out[b, h].cpu().double() - want).abs() <= want.abs() * 2.0 ** -9 * 2 + 2.0 ** -12 * (p @ v.abs())).all()
            grown = (weights[b] - old[b]).double().sum().item()
            assert abs(grown - hq) < 1e-3
        lens = batch_evict_kv_pages(k_pool, v_pool, table, lens, weights, positions, budget, recent)
        assert int(lens.max()) <= budget
        for b in range(batch):
            n = int(lens[b])
            newest = set(range(total[b] - min(recent, n), total[b]))
            for h in range(hw):
                assert newest <= set(positions[b, h, :n].tolist())
        if step == 20:  # out to staging and back into other pages
            ptrs = torch.tensor([k_pool.data_ptr(), v_pool.data_ptr()], dtype=torch.int64, device=DEV)
            staging = torch.empty(batch * width * 2 * page * hkv * dim, dtype=torch.bfloat16, device=DEV)
            batch_gather_kv_pages(ptrs, staging, table.reshape(-1), None, 1, page * hkv * dim * 2, pages)
            k_pool[table.long().view(-1)] = math.nan
            v_pool[table.long().view(-1)] = math.nan
            batch_scatter_kv_pages(ptrs, staging, spare.reshape(-1), None, 1, page * hkv * dim * 2, pages)
            table, spare = spare, table


def test_pools_in_one_tensor_and_behind_four_gigabytes():
    """K and V as halves of one tensor, [2, pages, ...]; rows more than 2^32 bytes apart."""
    page, hkv, dim, hq = 64, 1, 64, 4
    pages = (5 << 30) // (2 * page * hkv * dim * 2)  # 5 GiB for both
    both = torch.empty(2, pages, page, hkv, dim, dtype=torch.bfloat16, device=DEV)
    k_pool, v_pool = both[0], both[1]
    gen = torch.Generator().manual_seed(3)
    lens = [100, 130]
    table = torch.tensor([[0, pages - 1, 5], [pages // 2, pages - 2, 7]], dtype=torch.int32)
    small_k, small_v = oracle.make_pools(gen, 6, page, hkv, dim, "bf16")
    for i, pg in enumerate(table.view(-1).tolist()):
        k_pool[pg], v_pool[pg] = small_k[i].to(DEV), small_v[i].to(DEV)
    small_table = torch.arange(6, dtype=torch.int32).view(2, 3)
    q = torch.randn(2, hq, dim, generator=gen).to(torch.bfloat16)
    n = torch.tensor(lens, dtype=torch.int32)
    want, _, _, _, spread, size = oracle.attend(q, small_k, small_v, small_table, n, dim ** -0.5)
    got = batch_attend_kv_pages(q.to(DEV), k_pool, v_pool, table.to(DEV), n.to(DEV))
    assert ((got.cpu().double() - want).abs() <= _attend_tolerance(want, spread, size, 130, "bf16")).all()
    rng = np.random.default_rng(3)
    w = rng.random((2, 1, 192), dtype=np.float32)
    pos = np.broadcast_to(np.arange(192, dtype=np.int32), w.shape).copy()
    ref = oracle.evict(small_k, small_v, small_table, n, w, pos, 70, 10)
    batch_evict_kv_pages(k_pool, v_pool, table.to(DEV), n.to(DEV), torch.from_numpy(w).to(DEV),
                         torch.from_numpy(pos).to(DEV), 70, 10)
    for i, pg in enumerate(table.view(-1).tolist()):
        assert torch.equal(_bits(k_pool[pg].cpu()), _bits(ref[0][i])) and torch.equal(_bits(v_pool[pg].cpu()), _bits(ref[1][i]))
    key = torch.randn(2, hkv, dim, generator=gen).to(torch.bfloat16).to(DEV)
    slots = torch.tensor([pages * page - 1, 3], device=DEV)
    batch_append_kv_pages(None, key, key, torch.tensor([0, 0], device=DEV), slots, k_pool, v_pool,
                          rotary_frequencies(dim, device=DEV)[0])
    assert torch.equal(_bits(k_pool[pages - 1, page - 1]), _bits(key[0])) and torch.equal(_bits(v_pool[0, 3]), _bits(key[1]))


def test_nothing_to_do():
    """Empty batches, block tables without pages, sequences without tokens: results are written all the same."""
    k_pool = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device=DEV)
    v_pool = torch.zeros_like(k_pool)

    def i32(*shape):
        return torch.zeros(shape, dtype=torch.int32, device=DEV)

    for b, width in ((0, 3), (0, 0), (3, 0), (3, 2), (3, 9)):  # of the last two one is cut into runs, one is not
        q = torch.ones(b, 4, 64, dtype=torch.bfloat16, device=DEV)
        out, lse = torch.full_like(q, 7.0), torch.full((b, 4), 7.0, device=DEV)
        w = torch.full((b, 2, width * 16), 3.0, device=DEV)
        batch_attend_kv_pages(q, k_pool, v_pool, i32(b, width), i32(b), out=out, lse=lse, weights=w)
        assert (out == 0).all() and (lse == -math.inf).all() and (w == 3.0).all()
        pos = i32(b, 2, width * 16)
        lens = batch_evict_kv_pages(k_pool, v_pool, i32(b, width), i32(b), w, pos, 5, 2)
        assert lens.shape == (b,) and (lens == 0).all() and (w == 3.0).all() and (pos == 0).all()
        # lengths beyond an empty table are cut to nothing
        if b and not width:
            status = _status()
            lens = batch_evict_kv_pages(k_pool, v_pool, i32(b, 0), i32(b) + 9, w, pos, 5, 2, status=status)
            assert (lens == 0).all() and status.tolist()[:2] == [b, b]


def test_many_calls_in_a_row_read_what_the_one_before_wrote():
    """Kernels of one call start before the one in front has ended: the chain append, attend, evict without any
    synchronisation gives what it gives with one after every call."""
    gen = torch.Generator().manual_seed(4)
    hq, hkv, dim, width = 8, 2, 64, 24
    results = []
    for sync in (True, False):
        gen.manual_seed(4)
        k_pool, v_pool = (t.to(DEV) for t in oracle.make_pools(gen, 4 * width + 1, 16, hkv, dim, "bf16"))
        table = torch.randperm(4 * width, generator=gen).to(torch.int32).view(4, width).to(DEV)
        lens = torch.tensor([384, 200, 383, 10], dtype=torch.int32, device=DEV) - 30
        weights = torch.rand(4, hkv, width * 16, generator=gen).to(DEV)
        positions = torch.arange(width * 16, dtype=torch.int32).expand(4, hkv, -1).contiguous().to(DEV)
        inv_freq, _ = rotary_frequencies(dim, device=DEV)
        row = torch.arange(4, device=DEV)
        outs = []
        for step in range(30):
            qkv = torch.randn(4, hq + 2 * hkv, dim, generator=gen).to(torch.bfloat16).to(DEV)
            at = lens.long().clamp_max(width * 16 - 1)
            slots = table[row, at // 16].long() * 16 + at % 16
            positions[row, :, at] = 1000 + step
            q = batch_append_kv_pages(qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], at, slots, k_pool, v_pool, inv_freq)
            if sync:
                torch.cuda.synchronize()
            lens = (lens + 1).clamp_max(width * 16)
            outs.append(batch_attend_kv_pages(q, k_pool, v_pool, table, lens, weights=weights))
            if sync:
                torch.cuda.synchronize()
            lens = batch_evict_kv_pages(k_pool, v_pool, table, lens, weights, positions, 190, 20)
            if sync:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        results.append([_bits(torch.stack(outs)), weights, positions, _bits(k_pool), _bits(v_pool), lens])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_refusals_on_the_device():
    k_pool, v_pool, table, n, w, pos = _evict_case(2, [64], 2, 2, 64)
    dk, dv, dt, dn = k_pool.to(DEV), v_pool.to(DEV), table.to(DEV), n.to(DEV)
    dw, dp = torch.from_numpy(w).to(DEV), torch.from_numpy(pos).to(DEV)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=DEV)
    inv = rotary_frequencies(64, device=DEV)[0]
    one = torch.zeros(1, dtype=torch.int64, device=DEV)
    kv = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    bad = [
        lambda: batch_attend_kv_pages(q[:, :3], dk, dv, dt, dn),                      # heads do not divide
        lambda: batch_attend_kv_pages(q.half(), dk, dv, dt, dn),                      # another type
        lambda: batch_attend_kv_pages(q, dk, dv[:-1], dt, dn),                        # pools differ
        lambda: batch_attend_kv_pages(q, dk.float(), dv.float(), dt, dn),             # 32-bit pools
        lambda: batch_attend_kv_pages(q, dk, dv, dt.long(), dn),
        lambda: batch_attend_kv_pages(q, dk, dv, dt, dn.long()),
        lambda: batch_attend_kv_pages(q, dk, dv, dt, dn, window=-1),
        lambda: batch_attend_kv_pages(q, dk, dv, dt, dn, weights=dw[:, :, :63]),      # shorter than the table
        lambda: batch_attend_kv_pages(q, dk, dv, dt, dn, weights_out=dw),
        lambda: batch_attend_kv_pages(q, dk, dv, dt, dn, weights=dw, weights_out=dw[:, :1]),
        lambda: batch_attend_kv_pages(q, dk, dv, dt, dn, weights=dw[:, :1].expand(1, 2, 64)),  # written rows shared
        lambda: batch_attend_kv_pages(q.requires_grad_(), dk, dv, dt, dn),
        lambda: batch_evict_kv_pages(dk, dv, dt, dn, dw, dp, 0),
        lambda: batch_evict_kv_pages(dk, dv, dt, dn, dw, dp, 8, 9),
        lambda: batch_evict_kv_pages(dk, dv, dt, dn, dw, dp.long(), 8, 2),
        lambda: batch_evict_kv_pages(dk, dv, dt, dn, dw, dp[:, :1], 8, 2),
        lambda: batch_append_kv_pages(None, kv, kv, one, one.float(), dk, dv, inv),
        lambda: batch_append_kv_pages(None, kv, kv, one[:0], one, dk, dv, inv),
        lambda: batch_append_kv_pages(None, kv, kv, one, one, dk, dv, torch.zeros(33, device=DEV)),  # more than the head
        lambda: batch_append_kv_pages(None, kv[:, :1], kv[:, :1], one, one, dk, dv, inv),
        lambda: batch_append_kv_pages(None, kv, kv, one, one, dk, dv, inv, query_out=q),
        lambda: batch_append_kv_pages(None, kv, kv, one, one, dk, dk, inv),
        lambda: batch_append_kv_pages(None, kv, kv, one, one, dk[:, :, :1].expand(-1, -1, 2, -1),
                                      dv[:, :, :1].expand(-1, -1, 2, -1), inv),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    q = q.detach()
    odd = torch.zeros(4 * 16 * 2 * 64 + 4, dtype=torch.bfloat16, device=DEV)[4:].view(4, 16, 2, 64)  # 8 bytes off
    for call in (lambda: batch_attend_kv_pages(q, odd, odd.clone(), dt, dn),
                 lambda: batch_evict_kv_pages(odd, odd.clone(), dt, dn, dw, dp, 8, 2),
                 lambda: batch_attend_kv_pages(torch.zeros(1, 4, 65, dtype=torch.bfloat16, device=DEV)[:, :, 1:], dk, dv, dt, dn)):
        with pytest.raises(_cabi.KvcmError) as e:
            call()
        assert e.value.code == _cabi.KVCM_ER_INVALID_ADDRESS
    torch.cuda.synchronize()
