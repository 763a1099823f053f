"""What the Python operators hand to the entry points, from layouts alone: no GPU is needed to describe a tensor on one."""
import math

import pytest
import torch

import tair_kvcache_b200  # noqa: F401
from tair_kvcache_b200 import _cabi
from tair_kvcache_b200.kernel import paged_decode

GPU = torch.device("cuda", 0)


def contiguous(shape):
    return tuple(math.prod(shape[i + 1:]) for i in range(len(shape)))


def layout(shape, dtype, stride=None):
    return torch.Size(shape), contiguous(shape) if stride is None else stride, dtype, GPU


def flat(*layouts):
    return [field for one in layouts for field in one]


POOL = layout((10, 16, 2, 64), torch.bfloat16)
QUERY = layout((3, 4, 64), torch.bfloat16)
TABLE = layout((3, 5), torch.int32)
LENS = layout((3,), torch.int32)


def attend_plan(window=0, out=None, lse=None, weights=None, weights_out=None, query=QUERY, k=POOL, v=POOL, table=TABLE, lens=LENS):
    return paged_decode._attend_plan(window, out, lse, weights, weights_out, *flat(query, k, v, table, lens))


def test_a_window_beyond_the_table_is_the_table():
    for window, handed in ((0, 0), (1, 1), (79, 79), (80, 80), (81, 80), (2 ** 31, 80), (2 ** 32, 80), (2 ** 32 + 5, 80), (2 ** 70, 80)):
        assert attend_plan(window)[3] == handed, window
    assert attend_plan(7, table=layout((3, 0), torch.int32))[3] == 1  # no window would be another call
    with pytest.raises(ValueError):
        attend_plan(-1)


def test_integers_are_not_cut_without_the_shim(monkeypatch):
    """ctypes would pass 2^32 + 5 on as 5; the shim refuses it, and so does the route without it."""
    monkeypatch.setattr(_cabi, "shim", lambda: None)
    called = []
    monkeypatch.setattr(_cabi, "call", lambda name, *args: called.append(args))
    pools = (4096, 8192, 10, 2048, 128, 64, 16, 2, 64, 0)
    args = [0, 0, 0, 0, 0, 0, 0, 4096, 128, 64, 4096, 128, 64, 4096, 8, 4096, 4, 3, 4096, 64, 0, 1.0, 0, 0]
    _cabi.call_pages("kvcm_b200_append_pages", pools, *args)
    assert len(called) == 1 and called[0][1:] == tuple(args)
    tokens = 17
    assert _cabi.SIGNATURES["kvcm_b200_append_pages"][1:][tokens] is _cabi._i32 and args[tokens] == 3
    for value in (2 ** 31, 2 ** 32 + 5, -2 ** 31 - 1):
        with pytest.raises(TypeError):
            _cabi.call_pages("kvcm_b200_append_pages", pools, *args[:tokens], value, *args[tokens + 1:])
    with pytest.raises(TypeError):  # page_tokens
        _cabi.call_pages("kvcm_b200_append_pages", (*pools[:6], 2 ** 32 + 16, *pools[7:]), *args)
    with pytest.raises(TypeError):  # a stride
        _cabi.call_pages("kvcm_b200_append_pages", (*pools[:3], 2 ** 63, *pools[4:]), *args)
    assert len(called) == 1


def test_no_tensor_that_requires_gradients_is_read_or_written():
    def x(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype)

    pools = dict(k_pool=x(4, 16, 2, 64), v_pool=x(4, 16, 2, 64))
    sequences = dict(block_table=x(1, 2, dtype=torch.int32), context_lens=x(1, dtype=torch.int32))
    append = dict(query=x(1, 4, 64), key=x(1, 2, 64), value=x(1, 2, 64), positions=x(1, dtype=torch.int64),
                  slot_indices=x(1, dtype=torch.int64), inv_freq=x(32, dtype=torch.float32), query_out=x(1, 4, 64), **pools)
    attend = dict(query=x(1, 4, 64), out=x(1, 4, 64), lse=x(1, 4, dtype=torch.float32), weights=x(1, 2, 32, dtype=torch.float32),
                  weights_out=x(1, 2, 32, dtype=torch.float32), **pools, **sequences)
    evict = dict(weights=x(1, 2, 32, dtype=torch.float32), positions=x(1, 2, 32, dtype=torch.int32), budget=4,
                 weights_out=x(1, 2, 32, dtype=torch.float32), **pools, **sequences)
    for op, kwargs in ((paged_decode.batch_append_kv_pages, append), (paged_decode.batch_attend_kv_pages, attend),
                       (paged_decode.batch_evict_kv_pages, evict)):
        for name, t in kwargs.items():
            if not isinstance(t, torch.Tensor) or not t.is_floating_point():
                continue
            t.requires_grad_()
            with pytest.raises(ValueError, match="no gradient"):
                op(**kwargs)
            with torch.no_grad(), pytest.raises(ValueError, match="one GPU"):  # these tensors are on none
                op(**kwargs)
            t.requires_grad_(False)


def append_plan(query=layout((1, 4, 64), torch.bfloat16), query_out=None, key=layout((1, 2, 64), torch.bfloat16),
                value=layout((1, 2, 64), torch.bfloat16), k=POOL, v=POOL):
    index = layout((key[0][0],), torch.int64)
    return paged_decode._append_plan(query, query_out, *flat(key, value, index, index, k, v, layout((32,), torch.float32)))


def test_strides_of_axes_of_length_one_say_nothing():
    # a view of one token, or of one head, may have any stride there: neither its value nor its alignment counts
    odd = layout((1, 4, 64), torch.bfloat16, (257, 64, 1))
    assert attend_plan(query=odd, table=layout((1, 5), torch.int32), lens=layout((1,), torch.int32))[1][:2] == (0, 64)
    head = layout((3, 2, 64), torch.bfloat16, (128, 64, 1))
    assert attend_plan(query=head)[1][:2] == (128, 64)
    one_head = layout((3, 1, 64), torch.bfloat16, (256, 13, 1))
    pool = layout((10, 16, 1, 64), torch.bfloat16)
    assert attend_plan(query=one_head, k=pool, v=pool)[1][:2] == (256, 0)
    plan = append_plan(odd, odd, layout((1, 2, 64), torch.bfloat16, (3, 64, 1)), layout((1, 2, 64), torch.bfloat16, (5, 64, 1)))
    assert plan[2][:2] == plan[3] == (0, 64) and plan[4] == plan[5] == (0, 64)
    # pools that differ in such a stride alone have one layout
    k, v = layout((1, 16, 2, 64), torch.bfloat16, (4096, 128, 64, 1)), layout((1, 16, 2, 64), torch.bfloat16, (9999, 128, 64, 1))
    assert attend_plan(k=k, v=v)[0][:4] == (1, 0, 128, 64)
    with pytest.raises(ValueError, match="one shape"):
        attend_plan(k=POOL, v=layout((10, 16, 2, 64), torch.bfloat16, (4096, 128, 64, 1)))


def test_a_call_on_another_device_leaves_torchs_current_one(monkeypatch):
    """The two runtimes share the driver's current context: whichever binds last is what both may report."""
    current, events = [0], []

    class Device:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.previous, current[0] = current[0], self.index
            events.append(("torch", self.index))

        def __exit__(self, *_):
            current[0] = self.previous
            events.append(("torch", self.previous))

    def bind(index):
        current[0] = index
        events.append(("library", index))

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(paged_decode, "_raw_stream", lambda index: 1000 + index)
    monkeypatch.setattr(_cabi, "bind_device", bind)
    monkeypatch.setattr(_cabi, "call_pages", lambda name, pools, *args: events.append((name, current[0], args)))
    paged_decode._launch("op", torch.device("cuda", 1), (), 7)
    assert events == [("torch", 1), ("library", 1), ("op", 1, (7, 1001)), ("torch", 0)] and current == [0]
    events.clear()
    paged_decode._launch("op", torch.device("cuda", 0), (), 7)
    assert events == [("library", 0), ("op", 0, (7, 1000))] and current == [0]


def test_same_memory_means_same_strides():
    """In place is one layout twice.  A query and its result at one address with strides that differ where they count are
    refused; where an axis has length one they do not count, for weights and positions neither."""
    import ctypes
    address = 1 << 20
    pools = _cabi.KvPools(address, 2 * address, 10, 16 * 2 * 64, 2 * 64, 64, 16, 2, 64, _cabi.DTYPE_BF16)

    def append(tokens, heads, strides, out_strides, out=address):
        return _cabi.lib().kvcm_b200_append_pages(
            ctypes.addressof(pools), address, *strides, heads, out, *out_strides, address, 128, 64, address, 128, 64, address, 8,
            address, 4, tokens, address, 64, 0, 1.0, None, None)

    if not torch.cuda.is_available():  # what passes the checks ends at the missing device
        assert append(3, 4, (256, 64), (256, 64)) == _cabi.KVCM_ER_NO_DEVICE
        assert append(1, 4, (256, 64), (512, 64)) == append(3, 1, (256, 64), (256, 128)) == _cabi.KVCM_ER_NO_DEVICE
        assert append(3, 4, (256, 64), (512, 64), out=9 * address) == _cabi.KVCM_ER_NO_DEVICE
    assert append(3, 4, (256, 64), (512, 64)) == append(3, 4, (256, 64), (64, 192)) == _cabi.KVCM_ER_INVALID_PARAMS
    weights = layout((1, 1, 80), torch.float32, (80, 80, 1))
    other = layout((1, 1, 80), torch.float32, (999, 77, 1))
    plan = attend_plan(weights=weights, weights_out=other, query=layout((1, 4, 64), torch.bfloat16),
                       table=layout((1, 5), torch.int32), lens=layout((1,), torch.int32))
    assert plan[4] == plan[5] == (0, 0, 1)


@pytest.mark.parametrize("dim,base,factor,length", [(128, 10000.0, 8.0, 8192), (64, 500000.0, 32.0, 4096), (80, 10000.0, 3.5, 1000)])
def test_the_inside_of_the_frequency_ramps(dim, base, factor, length):
    """yarn and llama3 pair by pair from their definitions, in 64-bit numbers; float32 is off by half a step."""
    def close(got, want):
        return all(abs(g - w) <= w * (2.0 ** -24 + 1e-12) for g, w in zip(got.double().tolist(), want))

    plain = [base ** (-2.0 * j / dim) for j in range(dim // 2)]
    scaled, _ = paged_decode.rotary_frequencies(dim, base, "llama3", factor, length, device="cpu")
    want, inside = [], 0
    for f in plain:
        wavelength = 2 * math.pi / f
        if wavelength < length / 4.0:
            want.append(f)
        elif wavelength > length / 1.0:
            want.append(f / factor)
        else:
            smooth = (length / wavelength - 1.0) / (4.0 - 1.0)
            want.append((1 - smooth) * f / factor + smooth * f)
            inside += 1
    assert inside > 0 and close(scaled, want)
    scaled, attention = paged_decode.rotary_frequencies(dim, base, "yarn", factor, length, device="cpu")

    def pair(turns):  # the (real) pair whose angle makes that many turns over `length` tokens: base^(-2 j / dim) = 2 pi turns / length
        return -dim / 2.0 * math.log(2 * math.pi * turns / length, base)

    low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), dim - 1)
    want = []
    for j, f in enumerate(plain):
        share = min(max((j - low) / (high - low), 0.0), 1.0)  # of the interpolated frequency
        want.append(f / factor * share + f * (1 - share))
    assert high - low > 2 and close(scaled, want) and attention == 0.1 * math.log(factor) + 1.0
