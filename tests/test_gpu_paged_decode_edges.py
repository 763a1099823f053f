"""The decode-step operators where numbers, shapes and callers are at their limits, against the 64-bit forms."""
import math

import pytest
import torch

import paged_decode_oracle as oracle
from test_gpu_paged_decode import DEV, _attend_case, _attend_tolerance

from tair_kvcache_b200 import _cabi
from tair_kvcache_b200.kernel import batch_append_kv_pages, batch_attend_kv_pages, rotary_frequencies

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
