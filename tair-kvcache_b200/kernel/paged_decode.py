"""A decode step over paged KV pools: what an engine computes on the pools the connector moves.

  batch_append_kv_pages   rotary positions on the new tokens' queries and keys; keys and values into their pool slots
  batch_attend_kv_pages   attention of one new token per sequence over its pages, attention weights accumulated
  batch_evict_kv_pages    the newest and the most attended tokens kept, packed into the first slots of their pages
  rotary_frequencies      the frequencies the first one takes, plain or scaled for long contexts

The reference moves these pools (kv_cache_manager/py_connector/vllm/data_transfer.py:119-217) and leaves the computation
on them to the engine; slot and page numbers mean here what they mean there.  A pool is one layer's K or V, a tensor
indexed [page, token, head, element] - any strides of the first three, so both [pages, page_tokens, heads, dim] tensors
and .transpose(1, 2) views of [pages, heads, page_tokens, dim] ones.  The calls return as soon as the kernels are
enqueued on the current stream of the pools' device and allocate nothing but their results and workspaces, from torch's
allocator, so they can be captured into a CUDA graph.  None of them is differentiable; tensors that require
gradients, read or written, are refused while gradients are recorded.
"""
import functools
import math
from typing import Optional, Tuple

import torch

from .. import _cabi
from .batch_gather_scatter_helper import IndexArg, _index_tensor

_DTYPES = {torch.bfloat16: _cabi.DTYPE_BF16, torch.float16: _cabi.DTYPE_FP16}
_INDEX_BYTES = {torch.int32: 4, torch.int64: 8}


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_length: int = 8192, beta_fast: float = 32.0, beta_slow: float = 1.0,
                       low_freq_factor: float = 1.0, high_freq_factor: float = 4.0,
                       device="cuda") -> Tuple[torch.Tensor, float]:
    """(inv_freq, attention_factor) for batch_append_kv_pages: float32 [rotary_dim / 2] and a number.

    scaling   "none"     base^(-2j / rotary_dim)
              "linear"   the same divided by `factor` (positions interpolated)
              "ntk"      base stretched by factor^(rotary_dim / (rotary_dim - 2)): the slowest pair is interpolated,
                         the fastest kept
              "yarn"     pairs that turn more than beta_fast times within original_length are kept, those that turn less
                         than beta_slow times interpolated, a linear ramp over the pairs between them; cosine and sine
                         are multiplied by 0.1 ln(factor) + 1
              "llama3"   the same two regions by high_freq_factor and low_freq_factor, the ramp linear in the turns
    """
    if rotary_dim < 0 or rotary_dim % 2 or base <= 1.0 or factor < 1.0 or original_length < 1:
        raise ValueError("rotary_dim must be even, base > 1, factor >= 1 and original_length >= 1")
    half = rotary_dim // 2
    j = torch.arange(half, dtype=torch.float64)
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-2.0 * j / max(rotary_dim, 1))
    attention_factor = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        def pair_that_turns(times):  # index of the pair that turns `times` times within original_length
            return rotary_dim * math.log(original_length / (times * 2.0 * math.pi)) / (2.0 * math.log(base))
        low = max(math.floor(pair_that_turns(beta_fast)), 0)
        high = min(math.ceil(pair_that_turns(beta_slow)), rotary_dim - 1)
        stretched = ((j - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        freq = freq / factor * stretched + freq * (1.0 - stretched)
        attention_factor = 0.1 * math.log(factor) + 1.0
    elif scaling == "llama3":
        if high_freq_factor <= low_freq_factor:
            raise ValueError("high_freq_factor must be greater than low_freq_factor")
        turns = original_length * freq / (2.0 * math.pi)
        kept = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0.0, 1.0)
        freq = freq * kept + freq / factor * (1.0 - kept)
    elif scaling not in ("none", "ntk"):
        raise ValueError("unknown scaling %r" % (scaling,))
    return freq.to(torch.float32).to(device), attention_factor


# Layouts are checked once and remembered by what they are - shapes, strides, types, devices, never addresses - so that a
# decode loop, which calls with the same ones over and over, pays for a dictionary lookup.
_REMEMBERED = 1024


def _layout(t: Optional[torch.Tensor]):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _layouts(flat):
    """Layouts whose four fields stand one after the other (a lookup key is made faster that way)."""
    return [flat[i:i + 4] for i in range(0, len(flat), 4)]


def _strides(t):
    """A layout's strides; that of an axis of length one says nothing and counts as zero."""
    return tuple(stride if size > 1 else 0 for size, stride in zip(t[0], t[1]))


def _pools(k, v):
    """The fields of kvcm_b200_kv_pools_t behind the two addresses, from the pools' layouts."""
    (shape, _, dtype, device) = k
    strides = _strides(k)
    if len(shape) != 4 or v[0] != shape or _strides(v) != strides:
        raise ValueError("the K and V pools must be [pages, page_tokens, heads, dim] tensors of one shape and layout")
    if dtype not in _DTYPES or v[2] != dtype:
        raise ValueError("the pools must hold bfloat16 or float16, got %s and %s" % (dtype, v[2]))
    if device.type != "cuda" or v[3] != device:
        raise ValueError("the pools must live on one GPU")
    pages, page_tokens, heads, dim = shape
    sp, st, sh, se = strides
    if page_tokens == 0 or heads == 0 or dim == 0:
        raise ValueError("the pools' pages are empty")
    if se != 1 and dim > 1:
        raise ValueError("the elements of a head must be contiguous in the pools")
    if (pages > 1 and sp == 0) or (page_tokens > 1 and st == 0) or (heads > 1 and sh == 0):
        raise ValueError("rows of the pools share memory")
    return (pages, sp, st, sh, page_tokens, heads, dim, _DTYPES[dtype])


def _no_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError("the paged decode operators have no gradient: call them under torch.no_grad()")


def _heads(t, name: str, pool, count: int):
    """A layout of [count, heads, dim] beside a pool's; the strides between tokens and heads, and the number of heads."""
    shape, strides, dtype, device = t[0], _strides(t), t[2], t[3]
    if len(shape) != 3 or shape[0] != count or shape[2] != pool[0][3]:
        raise ValueError("%s must be [%d, heads, %d], got %s" % (name, count, pool[0][3], list(shape)))
    if dtype != pool[2] or device != pool[3]:
        raise ValueError("%s must have the pools' type and device" % name)
    if strides[2] != 1 and shape[2] > 1:
        raise ValueError("the elements of a head must be contiguous in %s" % name)
    return strides[0], strides[1], shape[1]


def _own_rows(t, name: str):
    """A tensor that is written: no two of its rows may be the same memory."""
    for size, stride in zip(t[0], t[1]):
        if size > 1 and stride == 0:
            raise ValueError("rows of %s share memory" % name)


def _contiguous(t) -> bool:
    expected = 1
    for size, stride in zip(reversed(t[0]), reversed(t[1])):
        if size != 1 and stride != expected:
            return False
        expected *= size
    return True


def _sequences(table, lens, pool):
    """Number of sequences, pages per sequence and the stride between sequences of the table."""
    if len(table[0]) != 2 or table[2] != torch.int32 or table[3] != pool[3]:
        raise ValueError("block_table must be an int32 [sequences, pages] tensor on the pools' device")
    if table[1][1] != 1 and table[0][1] > 1:
        raise ValueError("the pages of a sequence must be contiguous in block_table")
    if len(lens[0]) != 1 or lens[2] != torch.int32 or lens[3] != pool[3] or lens[0][0] != table[0][0] or not _contiguous(lens):
        raise ValueError("context_lens must be a contiguous int32 [sequences] tensor on the pools' device")
    return table[0][0], table[0][1], table[1][0]


def _per_slot(t, name: str, dtype: torch.dtype, pool, batch: int, tokens: int, heads=None):
    """Strides between sequences and heads, and the number of heads, of an array with an entry per slot."""
    shape, strides = t[0], _strides(t)
    if (len(shape) != 3 or t[2] != dtype or t[3] != pool[3] or shape[0] != batch or shape[2] < tokens or
            shape[1] not in ((1, pool[0][2]) if heads is None else (heads,)) or (strides[2] != 1 and shape[2] > 1)):
        raise ValueError("%s must be a %s [%d, %s, >= %d] tensor on the pools' device, contiguous along the last axis, "
                         "with an entry for every token of the block table"
                         % (name, dtype, batch, "1 or %d" % pool[0][2] if heads is None else heads, tokens))
    return strides[0], strides[1], shape[1]


def _status_ptr(status: Optional[torch.Tensor], device: torch.device) -> int:
    if status is None:
        return 0
    if status.numel() < 4 or status.element_size() != 4 or status.device != device or not status.is_contiguous():
        raise ValueError("status must be four 32-bit words on the pools' device")
    return status.data_ptr()


# The current stream's address without building a Stream object around it (2 us of a 14 us call), where torch has that.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _launch(name: str, device: torch.device, pools, *args) -> None:
    """Both runtimes, torch's and the library's, have the pools' device current for the call, and torch's has its own back
    afterwards: it is asked before the library's is changed, as the two share the driver's current context."""
    index = device.index
    stream = _raw_stream(index)
    if torch.cuda.current_device() == index:
        _cabi.bind_device(index)
        _cabi.call_pages(name, pools, *args, stream)
    else:
        with torch.cuda.device(device):
            _cabi.bind_device(index)
            _cabi.call_pages(name, pools, *args, stream)


def _workspace_bytes(name: str, size: int) -> int:
    if size < 0:
        raise _cabi.KvcmError(_cabi.KVCM_EC_OUT_OF_LIMIT, name)
    return size


@functools.lru_cache(maxsize=_REMEMBERED)
def _append_plan(query, query_out, *flat):
    key, value, positions, slots, k, v, inv_freq = _layouts(flat)
    pools = _pools(k, v)
    tokens = key[0][0] if len(key[0]) else 0
    k_args, v_args = _heads(key, "key", k, tokens), _heads(value, "value", k, tokens)
    if k_args[2] != pools[5] or v_args[2] != pools[5]:
        raise ValueError("key and value must have the pools' %d heads" % pools[5])
    for t, name in ((positions, "positions"), (slots, "slot_indices")):
        if len(t[0]) != 1 or t[2] not in _INDEX_BYTES or t[0][0] != tokens or t[3] != k[3] or not _contiguous(t):
            raise ValueError("%s must be a contiguous int32 or int64 [%d] tensor on the pools' device" % (name, tokens))
    if len(inv_freq[0]) != 1 or inv_freq[2] != torch.float32 or inv_freq[3] != k[3] or not _contiguous(inv_freq) or (
            2 * inv_freq[0][0] > pools[6]):
        raise ValueError("inv_freq must be a contiguous float32 tensor of at most dim / 2 frequencies on the pools' device")
    q_args = q_out_args = None
    if query is not None:
        q_args = _heads(query, "query", k, tokens)
        if query_out is None:
            q_out_args = (q_args[2] * pools[6], pools[6])
        else:
            if query_out[0] != query[0]:
                raise ValueError("query_out must have query's shape")
            q_out_args = _heads(query_out, "query_out", k, tokens)[:2]
            _own_rows(query_out, "query_out")
    elif query_out is not None:
        raise ValueError("query_out without query")
    return (pools, tokens, q_args, q_out_args, k_args[:2], v_args[:2], _INDEX_BYTES[positions[2]], _INDEX_BYTES[slots[2]],
            2 * inv_freq[0][0], k[3])


def batch_append_kv_pages(query: Optional[torch.Tensor], key: torch.Tensor, value: torch.Tensor,
                          positions: torch.Tensor, slot_indices: IndexArg, k_pool: torch.Tensor, v_pool: torch.Tensor,
                          inv_freq: torch.Tensor, interleaved: bool = False, attention_factor: float = 1.0,
                          query_out: Optional[torch.Tensor] = None,
                          status: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Rotates queries and keys by their positions and writes keys and values into the pools; returns the queries.

    query [tokens, q_heads, dim] (None: only keys and values), key and value [tokens, kv_heads, dim], strided as they come
    out of a fused projection.  The first 2 * len(inv_freq) elements of each head are rotated by
    positions[t] * inv_freq[j], in pairs (j, j + len(inv_freq)) or, interleaved, (2j, 2j + 1), cosine and sine times
    `attention_factor`; the others pass through.  Token t's key and value go to pool token slot_indices[t] =
    page * page_tokens + offset, the numbers batch_scatter_kv_caches takes; -1 marks a padding token, which writes
    nothing; any other slot outside the pool is skipped and counted in `status` (four zeroed 32-bit words on the GPU).
    The same slot twice in one call is a data race.  `query_out` may be `query`, or memory of its own."""
    _no_grad(query, key, value, inv_freq, k_pool, v_pool, query_out)
    if not isinstance(slot_indices, torch.Tensor):
        slot_indices = _index_tensor(slot_indices, k_pool.device)
    pools, tokens, q_args, q_out_args, k_args, v_args, position_bytes, slot_bytes, rotary_dim, device = _append_plan(
        _layout(query), _layout(query_out), key.shape, key.stride(), key.dtype, key.device, value.shape, value.stride(),
        value.dtype, value.device, positions.shape, positions.stride(), positions.dtype, positions.device, slot_indices.shape,
        slot_indices.stride(), slot_indices.dtype, slot_indices.device, k_pool.shape, k_pool.stride(), k_pool.dtype,
        k_pool.device, v_pool.shape, v_pool.stride(), v_pool.dtype, v_pool.device, inv_freq.shape, inv_freq.stride(),
        inv_freq.dtype, inv_freq.device)
    k_at, v_at = k_pool.data_ptr(), v_pool.data_ptr()
    if k_at == v_at and tokens:
        raise ValueError("keys and values cannot be written to one pool")
    if q_args is None:
        q_all = (0, 0, 0, 0, 0, 0, 0)
    else:
        if query_out is None:
            query_out = torch.empty_like(query, memory_format=torch.contiguous_format)
        q_all = (query.data_ptr(), *q_args, query_out.data_ptr(), *q_out_args)
    _launch("kvcm_b200_append_pages", device, (k_at, v_at, *pools), *q_all, key.data_ptr(), *k_args,
            value.data_ptr(), *v_args, positions.data_ptr(), position_bytes, slot_indices.data_ptr(), slot_bytes, tokens,
            inv_freq.data_ptr(), rotary_dim, int(interleaved), float(attention_factor), _status_ptr(status, device))
    return query_out


@functools.lru_cache(maxsize=_REMEMBERED)
def _attend_plan(window, out, lse, weights, weights_out, *flat):
    query, k, v, table, lens = _layouts(flat)
    pools = _pools(k, v)
    batch, width, table_stride = _sequences(table, lens, k)
    q_args = _heads(query, "query", k, batch)
    n_q_heads, n_kv_heads, dim = q_args[2], pools[5], pools[6]
    if n_q_heads == 0 or n_q_heads % n_kv_heads:
        raise ValueError("%d query heads are not a multiple of %d KV heads" % (n_q_heads, n_kv_heads))
    if window < 0:
        raise ValueError("window must not be negative")
    if out is not None and (out[0] != query[0] or out[2:] != query[2:] or not _contiguous(out)):
        raise ValueError("out must be contiguous, of query's shape, type and device")
    if lse is not None and (lse[0] != query[0][:2] or lse[2] != torch.float32 or lse[3] != k[3] or not _contiguous(lse)):
        raise ValueError("lse must be a contiguous float32 [sequences, q_heads] tensor on the pools' device")
    tokens = width * pools[4]
    window = min(window, max(tokens, 1)) if window else 0  # one beyond the table is none, and 32 bits hold this
    w_args = wo_args = None
    if weights is not None:
        w_args = _per_slot(weights, "weights", torch.float32, k, batch, tokens)
        wo_args = w_args if weights_out is None else _per_slot(weights_out, "weights_out", torch.float32, k, batch, tokens, w_args[2])
        _own_rows(weights if weights_out is None else weights_out, "weights_out")
    elif weights_out is not None:
        raise ValueError("weights_out without weights")
    size = _workspace_bytes("kvcm_b200_attend_pages", _cabi.lib().kvcm_b200_attend_workspace_bytes(
        batch, n_q_heads, n_kv_heads, dim, tokens, int(weights is not None)))
    return pools, (*q_args[:2], batch, n_q_heads), (table_stride, width), window, w_args, wo_args, size, dim ** -0.5, k[3]


def batch_attend_kv_pages(query: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor,
                          context_lens: torch.Tensor, scale: Optional[float] = None, window: int = 0,
                          out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                          weights: Optional[torch.Tensor] = None, weights_out: Optional[torch.Tensor] = None,
                          status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence over its cached keys and values; returns [sequences, q_heads, dim].

    query [sequences, q_heads, dim]; q_heads is a multiple of the pools' heads and consecutive query heads share a KV head.
    Sequence b attends its last `window` slots (0 = all) of the context_lens[b] in use; slot t lies in page
    block_table[b, t // page_tokens].  The last slots hold the last tokens as long as the cache is in order, that is, until
    batch_evict_kv_pages first moves one; after it attend with window = 0.  A layer that looks back W tokens keeps just
    those with budget = recent = W, evicting between append and attention.  scale defaults to dim ** -0.5.  A sequence
    without tokens gives zeros.  What pages hold behind a sequence's end never takes part, and neither do tokens on pages
    outside the pool; those pages, and lengths beyond the table (cut to it), are counted in `status`.  An attended value that
    is infinite or NaN makes that element of the output infinite or NaN.

    out (default: a new tensor): contiguous, of query's shape and type, memory of its own.
    lse: float32 [sequences, q_heads], receives the logarithm of the softmax sum (negative infinity without tokens).
    weights: float32 [sequences, 1 or kv_heads, >= table tokens]; weights_out (default: weights itself; else memory of its
    own) receives weights plus the attention each token got, summed over the query heads of its KV head or, with one weight
    head, over all of them - what batch_evict_kv_pages ranks by.  A slot in the range whose page lies outside the pool gets
    its weight as it was; entries out of the range are left as they are.

    Each call takes a workspace from torch: 9 to 68 MB for the shares of heads that several CTAs compute (17 MB for heads of
    128 in groups of up to eight) and, with weights, 4 bytes per sequence, query head and token of the block table - of
    the table's width, not of the lengths, which the host does not know.  256 sequences of 64 query heads with a table for
    131,072 tokens take 8.6 GB: pass the part of the table that the longest sequence needs, block_table[:, :pages]."""
    _no_grad(query, k_pool, v_pool, weights, out, lse, weights_out)
    pools, q_args, table_args, window, w_args, wo_args, size, default_scale, device = _attend_plan(
        int(window), out if out is None else _layout(out), lse if lse is None else _layout(lse),
        weights if weights is None else _layout(weights), weights_out if weights_out is None else _layout(weights_out),
        query.shape, query.stride(), query.dtype, query.device, k_pool.shape, k_pool.stride(), k_pool.dtype, k_pool.device,
        v_pool.shape, v_pool.stride(), v_pool.dtype, v_pool.device, block_table.shape, block_table.stride(), block_table.dtype,
        block_table.device, context_lens.shape, context_lens.stride(), context_lens.dtype, context_lens.device)
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    w_all = (0, 0, 0, 0, 0, 0, 0)
    if w_args is not None:
        w_all = (weights.data_ptr(), *w_args[:2], (weights if weights_out is None else weights_out).data_ptr(), *wo_args)
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    _launch("kvcm_b200_attend_pages", device, (k_pool.data_ptr(), v_pool.data_ptr(), *pools), query.data_ptr(), *q_args,
            block_table.data_ptr(), *table_args, context_lens.data_ptr(), default_scale if scale is None else float(scale),
            window, out.data_ptr(), 0 if lse is None else lse.data_ptr(), *w_all, workspace.data_ptr(), size,
            _status_ptr(status, device))
    return out


@functools.lru_cache(maxsize=_REMEMBERED)
def _evict_plan(budget, recent, weights_out, positions_out, *flat):
    k, v, table, lens, weights, positions = _layouts(flat)
    pools = _pools(k, v)
    batch, width, table_stride = _sequences(table, lens, k)
    tokens = width * pools[4]
    if budget < 1 or recent < 0 or recent > budget:
        raise ValueError("0 <= recent <= budget and budget >= 1 are needed, got recent=%r budget=%r" % (recent, budget))
    w_args = _per_slot(weights, "weights", torch.float32, k, batch, tokens)
    heads = w_args[2]
    p_args = _per_slot(positions, "positions", torch.int32, k, batch, tokens, heads)
    wo_args = w_args if weights_out is None else _per_slot(weights_out, "weights_out", torch.float32, k, batch, tokens, heads)
    po_args = p_args if positions_out is None else _per_slot(positions_out, "positions_out", torch.int32, k, batch, tokens, heads)
    _own_rows(weights if weights_out is None else weights_out, "weights_out")
    _own_rows(positions if positions_out is None else positions_out, "positions_out")
    # a budget beyond the table evicts nothing, as the table's size does
    budget = min(budget, max(tokens, 1))
    size = _workspace_bytes("kvcm_b200_evict_pages", _cabi.lib().kvcm_b200_evict_workspace_bytes(batch, heads, tokens, budget))
    return (pools, (table_stride, width), batch, (budget, min(recent, budget), heads), w_args[:2], p_args[:2], wo_args[:2],
            po_args[:2], size, k[3])


def batch_evict_kv_pages(k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor,
                         context_lens: torch.Tensor, weights: torch.Tensor, positions: torch.Tensor, budget: int,
                         recent: int = 0, weights_out: Optional[torch.Tensor] = None,
                         positions_out: Optional[torch.Tensor] = None,
                         status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Cuts every sequence longer than `budget` slots to its `budget` best tokens; returns the new lengths (int32).

    weights float32 and positions int32, both [sequences, 1 or kv_heads, >= table tokens]: of each slot in use the
    accumulated attention (batch_attend_kv_pages) and the position its token has in the text.  Kept are the tokens
    whose position is among the `recent` newest, then the heaviest; among equals the one in the lower slot (NaN counts
    as the heaviest).  Protected tokens are equals: where positions occur more than once and more of them are protected
    than fit, those in the lower slots stay.  With one weight head all KV heads keep the same tokens, else each head its
    own.  Survivors in slots from `budget` on move into the slots freed below it - rows of both pools, weight and position -
    so that the first `budget` slots hold what is kept, in no particular order, and the pages behind them are free.  The
    freed slots get weight 0 and position -1.  Attention over what is left has no use for a window: it would go by slots,
    not by positions.  Results go into `weights` and `positions` themselves unless `weights_out` or `positions_out` are
    given, memory of their own, which then receive every slot in use.

    Pages are packed in place: a page that two sequences share must be copied first, and an evicted page no longer holds
    the tokens that its block hash names, so it must not be stored or matched under that key.  A move from or to a page
    outside the pool is left out and counted in `status`, as is a length beyond the table (cut to it)."""
    _no_grad(k_pool, v_pool, weights, weights_out)
    pools, table_args, batch, sizes, w_args, p_args, wo_args, po_args, size, device = _evict_plan(
        int(budget), int(recent), weights_out if weights_out is None else _layout(weights_out),
        positions_out if positions_out is None else _layout(positions_out), k_pool.shape, k_pool.stride(), k_pool.dtype,
        k_pool.device, v_pool.shape, v_pool.stride(), v_pool.dtype, v_pool.device, block_table.shape, block_table.stride(),
        block_table.dtype, block_table.device, context_lens.shape, context_lens.stride(), context_lens.dtype,
        context_lens.device, weights.shape, weights.stride(), weights.dtype, weights.device, positions.shape,
        positions.stride(), positions.dtype, positions.device)
    new_lens = torch.empty_like(context_lens)
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    _launch("kvcm_b200_evict_pages", device, (k_pool.data_ptr(), v_pool.data_ptr(), *pools), batch, block_table.data_ptr(),
            *table_args, context_lens.data_ptr(), *sizes, weights.data_ptr(), *w_args, positions.data_ptr(), *p_args,
            (weights if weights_out is None else weights_out).data_ptr(), *wo_args,
            (positions if positions_out is None else positions_out).data_ptr(), *po_args, new_lens.data_ptr(),
            workspace.data_ptr(), size, _status_ptr(status, device))
    return new_lens
