"""The decode-step entry points where no GPU is needed: refusals before anything is launched, workspace sizes, frequencies."""
import ctypes
import math

import pytest
import torch

import tair_kvcache_b200  # noqa: F401
from tair_kvcache_b200 import _cabi
from tair_kvcache_b200.kernel import rotary_frequencies
from tair_kvcache_b200.kernel import paged_decode

PARAMS, ADDRESS, LIMIT = _cabi.KVCM_ER_INVALID_PARAMS, _cabi.KVCM_ER_INVALID_ADDRESS, _cabi.KVCM_EC_OUT_OF_LIMIT
NO_DEVICE = _cabi.KVCM_ER_NO_DEVICE
A = 1 << 20  # an address nobody looks behind


def _pools(**changes):
    fields = dict(k_pool=A, v_pool=2 * A, pool_pages=10, page_stride=16 * 2 * 64, token_stride=2 * 64, head_stride=64,
                  page_tokens=16, n_kv_heads=2, head_dim=64, dtype=_cabi.DTYPE_BF16)
    fields.update(changes)
    return _cabi.KvPools(**fields)


def _append(pools=None, q=A, qs=(256, 64), hq=4, qo=A, qos=(256, 64), k=A, ks=(128, 64), v=A, vs=(128, 64), pos=A, pos_b=8,
            slots=A, slot_b=4, tokens=3, inv=A, rd=64):
    pools = _pools() if pools is None else pools
    return _cabi.lib().kvcm_b200_append_pages(ctypes.addressof(pools), q, *qs, hq, qo, *qos, k, *ks, v, *vs, pos, pos_b,
                                              slots, slot_b, tokens, inv, rd, 0, 1.0, None, None)


def _attend(pools=None, q=A, qs=(256, 64), batch=2, hq=4, table=A, width=8, lens=A, window=0, out=A, w=None, ws=(0, 0),
            wo=None, wos=(0, 0), hw=0, space=A, size=None):
    pools = _pools() if pools is None else pools
    if size is None:
        size = max(0, _cabi.lib().kvcm_b200_attend_workspace_bytes(min(max(batch, 0), 70000), hq, 2, 64,
                                                                   min(128, max(0, width * 16)), 1))
    return _cabi.lib().kvcm_b200_attend_pages(ctypes.addressof(pools), q, *qs, batch, hq, table, 8, width, lens, 0.125,
                                              window, out, None, w, *ws, wo, *wos, hw, space, size, None, None)


def _evict(pools=None, batch=2, table=A, width=8, lens=A, budget=32, recent=4, hw=2, w=A, ws=(256, 128), p=2 * A,
           ps=(256, 128), wo=A, wos=(256, 128), po=2 * A, pos=(256, 128), new=3 * A, space=A, size=1 << 20):
    pools = _pools() if pools is None else pools
    return _cabi.lib().kvcm_b200_evict_pages(ctypes.addressof(pools), batch, table, 8, width, lens, budget, recent, hw, w,
                                             *ws, p, *ps, wo, *wos, po, *pos, new, space, size, None, None)


def test_well_formed_calls_get_as_far_as_the_device():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: these addresses are not real")
    for call in (_append, _attend, _evict):
        assert call() == NO_DEVICE
    assert _append(q=None, qo=None, hq=0) == NO_DEVICE and _append(rd=0, inv=None) == NO_DEVICE
    assert _append(tokens=0, k=None) == NO_DEVICE and _attend(batch=0, q=None) == NO_DEVICE
    assert _attend(w=A, ws=(256, 128), wo=A, wos=(256, 128), hw=2) == NO_DEVICE
    assert _attend(width=0, table=None) == NO_DEVICE
    assert _evict(width=0, table=None, w=None, p=None, wo=None, po=None) == NO_DEVICE


@pytest.mark.parametrize("changes,code", [
    (dict(k_pool=None), ADDRESS), (dict(v_pool=None), ADDRESS), (dict(page_tokens=0), PARAMS), (dict(n_kv_heads=0), PARAMS),
    (dict(head_dim=0), PARAMS), (dict(pool_pages=-1), PARAMS), (dict(pool_pages=1 << 31), PARAMS), (dict(dtype=2), PARAMS),
    (dict(page_stride=-8), PARAMS), (dict(n_kv_heads=1 << 20), PARAMS),
])
def test_pools_that_are_refused_by_all(changes, code):
    for call in (_append, _attend, _evict):
        assert call(pools=_pools(**changes)) == code, call


def test_refusals_of_append():
    for kw in (dict(tokens=-1), dict(rd=65), dict(rd=66), dict(rd=-2), dict(pos_b=2), dict(slot_b=1), dict(hq=-1)):
        assert _append(**kw) == PARAMS, kw
    for kw in (dict(k=None), dict(v=None), dict(pos=None), dict(slots=None), dict(inv=None), dict(q=None), dict(qo=None),
               dict(k=A + 1), dict(q=A + 3)):
        assert _append(**kw) == ADDRESS, kw
    assert _append(pools=_pools(head_dim=1026)) == PARAMS


def test_refusals_of_attend():
    for kw in (dict(batch=-1), dict(hq=0), dict(hq=3), dict(width=-1), dict(window=-1), dict(w=A, hw=2), dict(wo=A),
               dict(w=A, wo=A, hw=3), dict(w=A, wo=A, hw=0), dict(size=100),
               dict(w=A, ws=(256, 128), wo=A, wos=(512, 128), hw=2)):
        assert _attend(**kw) == PARAMS, kw
    for kw in (dict(q=None), dict(table=None), dict(lens=None), dict(out=None), dict(space=None), dict(space=A + 8),
               dict(q=A + 2), dict(out=A + 2), dict(qs=(256, 65)), dict(pools=_pools(k_pool=A + 8)),
               dict(pools=_pools(token_stride=132)), dict(pools=_pools(head_dim=60))):
        assert _attend(**kw) == ADDRESS, kw
    assert _attend(pools=_pools(head_dim=264)) == PARAMS
    for kw in (dict(batch=65537), dict(hq=4098), dict(width=(1 << 26) + 1), dict(batch=65536, hq=64, width=1 << 20, size=1 << 62)):
        assert _attend(**kw) == LIMIT, kw


def test_refusals_of_evict():
    for kw in (dict(batch=-1), dict(width=-1), dict(budget=0), dict(recent=-1), dict(recent=33), dict(hw=3), dict(size=16),
               dict(new=A, lens=A), dict(new=A + 4, lens=A), dict(wos=(256, 64)), dict(pos=(512, 128))):
        assert _evict(**kw) == PARAMS, kw
    for kw in (dict(table=None), dict(lens=None), dict(w=None), dict(p=None), dict(wo=None), dict(po=None), dict(new=None),
               dict(space=None), dict(space=A + 4), dict(pools=_pools(v_pool=A + 2)), dict(pools=_pools(head_stride=68))):
        assert _evict(**kw) == ADDRESS, kw
    assert _evict(width=(1 << 26) + 1) == LIMIT


def test_workspace_sizes():
    attend, evict = _cabi.lib().kvcm_b200_attend_workspace_bytes, _cabi.lib().kvcm_b200_evict_workspace_bytes
    plain, with_weights = attend(4, 32, 8, 128, 4096, 0), attend(4, 32, 8, 128, 4096, 1)
    assert 0 < plain < with_weights and with_weights - plain >= 4 * 32 * 4096 * 4
    assert attend(0, 1, 1, 8, 0, 0) > 0
    for bad in ((-1, 1, 1, 8, 1, 0), (1, 3, 2, 8, 1, 0), (1, 1, 1, 257, 1, 0), (1, 1, 1, 8, -1, 0), (1, 1, 1, 8, 1 << 31, 0)):
        assert attend(*bad) == -1, bad
    assert evict(2, 8, 1000, 400) >= 2 * 8 * (400 * 8 + 4) and evict(2, 8, 1000, 900) >= 2 * 8 * (100 * 8 + 4)
    assert evict(0, 1, 0, 1) > 0 and evict(3, 1, 10, 100) >= 3 * 4 and evict(2, 8, 1000, 400) % 256 == 0
    for bad in ((-1, 1, 1, 1), (1, 0, 1, 1), (1, 1, -1, 1), (1, 1, 1, 0)):
        assert evict(*bad) == -1, bad


def test_python_refuses_cpu_tensors_and_gradients():
    layout = paged_decode._layout
    pool = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        paged_decode._pools(layout(pool), layout(pool.clone()))
    with pytest.raises(ValueError, match="one shape"):
        paged_decode._pools(layout(pool), layout(pool[:3]))
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        paged_decode._pools(layout(pool.float()), layout(pool.float()))
    with pytest.raises(ValueError, match="no gradient"):
        paged_decode._no_grad(torch.zeros(1, requires_grad=True))
    with torch.no_grad():
        paged_decode._no_grad(torch.zeros(1, requires_grad=True))
    with pytest.raises(ValueError, match="share memory"):
        paged_decode._own_rows(layout(torch.zeros(1, 1, 8).expand(2, 1, 8)), "x")


def test_contiguity_of_a_layout_is_torchs():
    layout = paged_decode._layout
    base = torch.zeros(4, 6, 8)
    for t in (base, base[:, :1], base[:1], base[:, ::2], base.transpose(0, 1), base[:, :, :1], base[0], base[0, :, 0], base[:0],
              torch.zeros(1, 1).expand(3, 1), torch.zeros(3, 1).expand(3, 5)):
        if t.numel():
            assert paged_decode._contiguous(layout(t)) == t.is_contiguous(), (t.shape, t.stride())


def test_rotary_frequencies():
    plain, factor = rotary_frequencies(128, base=500000.0, device="cpu")
    j = torch.arange(64, dtype=torch.float64)
    want = 500000.0 ** (-2 * j / 128)
    assert factor == 1.0 and ((plain.double() - want).abs() <= want * 2.0 ** -24 * 1.01).all()
    assert torch.equal(rotary_frequencies(128, base=500000.0, scaling="linear", factor=4.0, device="cpu")[0], plain / 4)
    ntk, _ = rotary_frequencies(128, scaling="ntk", factor=8.0, device="cpu")
    first, _ = rotary_frequencies(128, device="cpu")
    assert ntk[0] == 1.0 and abs(ntk[-1] * 8 / first[-1] - 1) < 1e-6  # the slowest pair is interpolated
    for kind in ("yarn", "llama3"):
        scaled, factor = rotary_frequencies(128, scaling=kind, factor=8.0, original_length=8192, device="cpu")
        ratio = first / scaled
        assert ratio[0] == 1.0 and abs(ratio[-1] - 8.0) < 1e-5 and (ratio[1:] >= ratio[:-1] * (1 - 1e-6)).all()
        turns = 8192 * first / (2 * math.pi)
        fast = turns > (33.0 if kind == "yarn" else 4.0)
        if kind == "llama3":
            assert (ratio[fast] == 1.0).all() and ((ratio[turns < 1.0] - 8.0).abs() < 1e-5).all()
        assert factor == (0.1 * math.log(8.0) + 1.0 if kind == "yarn" else 1.0)
    same, _ = rotary_frequencies(64, scaling="yarn", factor=1.0, device="cpu")
    assert torch.allclose(same, rotary_frequencies(64, device="cpu")[0], rtol=1e-6)
    assert rotary_frequencies(0, device="cpu")[0].numel() == 0
    assert rotary_frequencies(2, scaling="ntk", factor=4.0, device="cpu")[0].tolist() == [1.0]
    for bad in (dict(rotary_dim=3), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, factor=0.5),
                dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, scaling="llama3", high_freq_factor=1.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(device="cpu", **bad)


def test_pools_live_until_the_call_without_the_shim(monkeypatch):
    """Without the shim the entry points get the address of a struct: it has to hold its fields while they run."""
    fields = (4096, 8192, 10, 20, 30, 40, 16, 2, 64, _cabi.DTYPE_FP16)
    seen = []

    def fake(name, pools, *args):
        others = [_cabi.KvPools(*[7] * 10) for _ in range(64)]  # would take the place of one that was freed
        held = pools if isinstance(pools, _cabi.KvPools) else _cabi.KvPools.from_address(
            pools if isinstance(pools, int) else ctypes.addressof(pools._obj))
        seen.append((tuple(getattr(held, f[0]) for f in _cabi.KvPools._fields_), args, len(others)))

    monkeypatch.setattr(_cabi, "shim", lambda: None)
    monkeypatch.setattr(_cabi, "call", fake)
    _cabi.call_pages("kvcm_b200_evict_pages", fields, 1, 2)
    assert seen == [(fields, (1, 2), 64)]
