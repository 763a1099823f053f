"""What the decode-step entry points ask of the CUDA runtime, on a stand-in for it: the library's own objects linked with
tests/cpp/fake_cuda_runtime.cc, whose requests can be refused.  A kernel that takes its work from another's results must
not be launched once that one was refused."""
import ctypes
import os
import re
import subprocess

import pytest

from conftest import ROOT

import tair_kvcache_b200  # noqa: F401
from tair_kvcache_b200 import _cabi

A = 1 << 20  # an address nobody looks behind
REFUSED = _cabi.KVCM_ER_CUDAMEMCPY_ERROR
SOURCES = ["append_pages", "attend_pages", "evict_pages", "runtime"]


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    import __graft_entry__ as entry
    builder = entry._load_build_module()
    out = tmp_path_factory.mktemp("fake")
    objects = []
    for name in SOURCES:  # the build keeps its objects; compiled here where they are missing or older than the source
        src, obj = os.path.join(builder.CSRC, name + ".cu"), os.path.join(builder.OBJ_DIR, name + ".o")
        if any(builder._newer(f, obj) for f in [src] + builder.HEADERS):
            obj = str(out / (name + ".o"))
            flags = [f for f in builder.NVCC_FLAGS if f != "-shared"]
            subprocess.run([builder.nvcc()] + flags + ["-I", os.path.join(ROOT, "include"), "-I", builder.CSRC, "-c", "-o", obj, src],
                           check=True)
        objects.append(obj)
    lib = str(out / "libfake.so")
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(builder.nvcc()))), "include")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I", cuda, "-o", lib,
                    os.path.join(ROOT, "tests", "cpp", "fake_cuda_runtime.cc")] + objects, check=True)
    L = ctypes.CDLL(lib)
    for name in ("append_pages", "attend_pages", "evict_pages", "attend_workspace_bytes", "evict_workspace_bytes"):
        fn = getattr(L, "kvcm_b200_" + name)
        fn.argtypes = _cabi.SIGNATURES["kvcm_b200_" + name]
        fn.restype = ctypes.c_int64 if name.endswith("bytes") else ctypes.c_int32
    L.fake_asked.restype = ctypes.c_char_p
    return L


_device = iter(range(1, 64))


def _run(fake, call, cluster=16, launch=-1, attribute=-1):
    """(code, requests) of a call on a device that the library has not met."""
    fake.fake_begin(next(_device), cluster, launch, attribute)
    code = call(fake)
    return code, fake.fake_asked().decode().splitlines()


def _kernels(asked):
    return [re.search(r"(AppendPages|AttendPages|JoinShares|AddWeights|EvictPages|MoveSlots)Kernel", line).group(1)
            for line in asked if line.startswith("launch")]


def _pools():
    return _cabi.KvPools(A, 2 * A, 10, 16 * 2 * 64, 2 * 64, 64, 16, 2, 64, _cabi.DTYPE_BF16)


def _append(L):
    pools = _pools()
    return L.kvcm_b200_append_pages(ctypes.addressof(pools), A, 256, 64, 4, A, 256, 64, A, 128, 64, A, 128, 64, A, 8, A, 4, 3, A, 64,
                                    0, 1.0, None, None)


def _attend(width, weights):
    def call(L):
        pools = _pools()
        size = L.kvcm_b200_attend_workspace_bytes(2, 4, 2, 64, width * 16, int(weights))
        w = (A, 2 * width * 16, width * 16) if weights else (None, 0, 0)
        return L.kvcm_b200_attend_pages(ctypes.addressof(pools), A, 256, 64, 2, 4, A, width, width, A, 0.125, 0, A, None, *w, *w,
                                        2 if weights else 0, A, size, None, None)
    return call


def _evict(tokens, budget=32, batch=1):
    def call(L):
        pools = _cabi.KvPools(A, 2 * A, 10, 16 * 64, 64, 64, 16, 1, 64, _cabi.DTYPE_BF16)
        size = L.kvcm_b200_evict_workspace_bytes(batch, 1, tokens, budget)
        return L.kvcm_b200_evict_pages(ctypes.addressof(pools), batch, A, tokens // 16, tokens // 16, A, budget, 0, 1,
                                       *(A, tokens, tokens) * 4, 2 * A, A, size, None, None)
    return call


@pytest.mark.parametrize("call,kernels", [
    (_append, ["AppendPages"]),
    (_attend(8, False), ["AttendPages"]),
    (_attend(8, True), ["AttendPages", "AddWeights"]),
    (_attend(64, False), ["AttendPages", "JoinShares"]),
    (_attend(64, True), ["AttendPages", "JoinShares", "AddWeights"]),
    (_evict(128), ["EvictPages", "MoveSlots"]),
    (_evict(32), ["EvictPages"]),           # the budget holds the whole table
    (_evict(1 << 20), ["EvictPages", "MoveSlots"]),
])
def test_nothing_is_launched_after_a_refusal(fake, call, kernels):
    code, asked = _run(fake, call)
    assert code == _cabi.KVCM_OK and _kernels(asked) == kernels
    for i in range(len(kernels)):
        code, asked = _run(fake, call, launch=i)
        assert code == REFUSED and _kernels(asked) == kernels[:i + 1]


@pytest.mark.parametrize("call", [_attend(8, True), _attend(64, False), _evict(128)])
def test_nothing_is_launched_without_its_shared_memory(fake, call):
    code, asked = _run(fake, call, attribute=0 if call.__qualname__.startswith("_attend") else 2)
    assert code == REFUSED and _kernels(asked) == [] and asked[-1] == "attribute smem"


def test_a_refusal_is_not_remembered(fake):
    """An attribute that was refused is asked for again, and an error that was returned does not reach the next call."""
    fake.fake_begin(next(_device), 16, -1, 0)
    call = _attend(64, False)
    assert call(fake) == REFUSED
    assert call(fake) == _cabi.KVCM_OK and _kernels(fake.fake_asked().decode().splitlines()) == ["AttendPages", "JoinShares"]
    assert fake.fake_asked().decode().count("attribute smem") == 2


@pytest.mark.parametrize("largest", [16, 8])
@pytest.mark.parametrize("tokens,batch", [(1024, 1), (16384, 1), (131072, 1), (131072, 100), (16 * 22528, 1), (1 << 20, 1)])
def test_clusters_are_no_larger_than_the_device_places(fake, tokens, batch, largest):
    code, asked = _run(fake, _evict(tokens, batch=batch), cluster=largest)
    line = next(x for x in asked if x.startswith("launch"))
    grid, smem, cluster = (int(re.search(k + r"=(\d+)", line).group(1)) for k in ("grid", "smem", "cluster"))
    assert code == _cabi.KVCM_OK and cluster <= largest and grid == batch * cluster
    slots = -(-tokens // cluster)
    assert smem == (slots * 8 if slots <= 22528 else 0)  # a slice that does not fit is read from global memory
    want = {(1024, 1): 1, (16384, 1): 16, (131072, 1): 16, (131072, 100): 8, (16 * 22528, 1): 16, (1 << 20, 1): 16}[tokens, batch]
    assert cluster == min(want, largest)
    if cluster <= 8:  # a launch that needs no opt-in makes none of its own: only the question may
        assert asked[asked.index("attribute cluster") + 1:].count("attribute cluster") == 0
