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
allocator, so they can be captured into a CUDA graph.  None of them is differentiable; inputs that require gradients
are refused while gradients are recorded.
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


def _pools(k_pool: torch.Tensor, v_pool: torch.Tensor):
    """The fields of kvcm_b200_kv_pools_t."""
    if k_pool.dim() != 4 or k_pool.shape != v_pool.shape or k_pool.stride() != v_pool.stride():
        raise ValueError("the K and V pools must be [pages, page_tokens, heads, dim] tensors of one shape and layout")
    dtype = _DTYPES.get(k_pool.dtype)
    if dtype is None or v_pool.dtype != k_pool.dtype:
        raise ValueError("the pools must hold bfloat16 or float16, got %s and %s" % (k_pool.dtype, v_pool.dtype))
    if not k_pool.is_cuda or v_pool.device != k_pool.device:
        raise ValueError("the pools must live on one GPU")
    pages, page_tokens, heads, dim = k_pool.shape
    sp, st, sh, se = k_pool.stride()
    if page_tokens == 0 or heads == 0 or dim == 0:
        raise ValueError("the pools' pages are empty")
    if se != 1 and dim > 1:
        raise ValueError("the elements of a head must be contiguous in the pools")
    # the stride of an axis of length one says nothing
    sp, st, sh = sp if pages > 1 else 0, st if page_tokens > 1 else 0, sh if heads > 1 else 0
    if (pages > 1 and sp == 0) or (page_tokens > 1 and st == 0) or (heads > 1 and sh == 0):
        raise ValueError("rows of the pools share memory")
    return (k_pool.data_ptr(), v_pool.data_ptr(), pages, sp, st, sh, page_tokens, heads, dim, dtype)


def _no_grad(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("the paged decode operators have no gradient: call them under torch.no_grad()")


def _heads(t: torch.Tensor, name: str, pool: torch.Tensor, count: int):
    if t.dim() != 3 or t.shape[0] != count or t.shape[2] != pool.shape[3]:
        raise ValueError("%s must be [%d, heads, %d], got %s" % (name, count, pool.shape[3], list(t.shape)))
    if t.dtype != pool.dtype or t.device != pool.device:
        raise ValueError("%s must have the pools' type and device" % name)
    if t.stride(2) != 1 and t.shape[2] > 1:
        raise ValueError("the elements of a head must be contiguous in %s" % name)
    return t


def _own_rows(t: torch.Tensor, name: str):
    """A tensor that is written: no two of its rows may be the same memory."""
    for size, stride in zip(t.shape, t.stride()):
        if size > 1 and stride == 0:
            raise ValueError("rows of %s share memory" % name)
    return t


def _sequences(block_table: torch.Tensor, context_lens: torch.Tensor, pool: torch.Tensor):
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.device != pool.device:
        raise ValueError("block_table must be an int32 [sequences, pages] tensor on the pools' device")
    if block_table.stride(1) != 1 and block_table.shape[1] > 1:
        raise ValueError("the pages of a sequence must be contiguous in block_table")
    if (context_lens.dim() != 1 or context_lens.dtype != torch.int32 or context_lens.device != pool.device or
            context_lens.shape[0] != block_table.shape[0] or not context_lens.is_contiguous()):
        raise ValueError("context_lens must be a contiguous int32 [sequences] tensor on the pools' device")
    return block_table.shape[0], block_table.shape[1]


def _per_slot(t: torch.Tensor, name: str, dtype: torch.dtype, pool: torch.Tensor, batch: int, tokens: int, heads=None):
    if (t.dim() != 3 or t.dtype != dtype or t.device != pool.device or t.shape[0] != batch or t.shape[2] < tokens or
            t.shape[1] not in ((1, pool.shape[2]) if heads is None else (heads,)) or (t.stride(2) != 1 and t.shape[2] > 1)):
        raise ValueError("%s must be a %s [%d, %s, >= %d] tensor on the pools' device, contiguous along the last axis, "
                         "with an entry for every token of the block table"
                         % (name, dtype, batch, "1 or %d" % pool.shape[2] if heads is None else heads, tokens))
    return t


def _status_ptr(status: Optional[torch.Tensor], pool: torch.Tensor) -> int:
    if status is None:
        return 0
    if status.numel() < 4 or status.element_size() != 4 or status.device != pool.device or not status.is_contiguous():
        raise ValueError("status must be four 32-bit words on the pools' device")
    return status.data_ptr()


def _launch(name: str, device: torch.device, pools, *args) -> None:
    _cabi.bind_device(device.index)
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == device.index:
        _cabi.call_pages(name, pools, *args, stream)
    else:
        with torch.cuda.device(device):
            _cabi.call_pages(name, pools, *args, stream)


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
    The same slot twice in one call is a data race.  `query_out` may be `query`."""
    _no_grad(query, key, value, inv_freq)
    pools = _pools(k_pool, v_pool)
    tokens = key.shape[0] if key.dim() else 0
    _heads(key, "key", k_pool, tokens)
    _heads(value, "value", k_pool, tokens)
    if key.shape[1] != k_pool.shape[2] or value.shape[1] != k_pool.shape[2]:
        raise ValueError("key and value must have the pools' %d heads" % k_pool.shape[2])
    if not isinstance(slot_indices, torch.Tensor):
        slot_indices = _index_tensor(slot_indices, k_pool.device)
    for t, name in ((positions, "positions"), (slot_indices, "slot_indices")):
        if (t.dim() != 1 or t.dtype not in _INDEX_BYTES or t.shape[0] != tokens or t.device != k_pool.device or
                not t.is_contiguous()):
            raise ValueError("%s must be a contiguous int32 or int64 [%d] tensor on the pools' device" % (name, tokens))
    if (inv_freq.dim() != 1 or inv_freq.dtype != torch.float32 or inv_freq.device != k_pool.device or
            not inv_freq.is_contiguous() or 2 * inv_freq.shape[0] > k_pool.shape[3]):
        raise ValueError("inv_freq must be a contiguous float32 tensor of at most dim / 2 frequencies on the pools' device")
    q_args = (0, 0, 0, 0, 0, 0, 0)
    if query is not None:
        _heads(query, "query", k_pool, tokens)
        if query_out is None:
            query_out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
        elif query_out.shape != query.shape:
            raise ValueError("query_out must have query's shape")
        _own_rows(_heads(query_out, "query_out", k_pool, tokens), "query_out")
        q_args = (query.data_ptr(), query.stride(0), query.stride(1), query.shape[1], query_out.data_ptr(),
                  query_out.stride(0), query_out.stride(1))
    elif query_out is not None:
        raise ValueError("query_out without query")
    _launch("kvcm_b200_append_pages", k_pool.device, pools, *q_args, key.data_ptr(), key.stride(0), key.stride(1),
            value.data_ptr(), value.stride(0), value.stride(1), positions.data_ptr(), _INDEX_BYTES[positions.dtype],
            slot_indices.data_ptr(), _INDEX_BYTES[slot_indices.dtype], tokens, inv_freq.data_ptr(),
            2 * inv_freq.shape[0], int(interleaved), float(attention_factor), _status_ptr(status, k_pool))
    return query_out


@functools.lru_cache(maxsize=4096)
def _attend_workspace_bytes(batch, n_q_heads, n_kv_heads, head_dim, tokens, with_weights):
    return _cabi.lib().kvcm_b200_attend_workspace_bytes(batch, n_q_heads, n_kv_heads, head_dim, tokens, with_weights)


@functools.lru_cache(maxsize=4096)
def _evict_workspace_bytes(batch, heads, tokens, budget):
    return _cabi.lib().kvcm_b200_evict_workspace_bytes(batch, heads, tokens, budget)


def _workspace(size: int, device: torch.device, name: str) -> torch.Tensor:
    if size < 0:
        raise _cabi.KvcmError(_cabi.KVCM_EC_OUT_OF_LIMIT, name)
    return torch.empty(size, dtype=torch.uint8, device=device)


def batch_attend_kv_pages(query: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor,
                          context_lens: torch.Tensor, scale: Optional[float] = None, window: int = 0,
                          out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                          weights: Optional[torch.Tensor] = None, weights_out: Optional[torch.Tensor] = None,
                          status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence over its cached keys and values; returns [sequences, q_heads, dim].

    query [sequences, q_heads, dim]; q_heads is a multiple of the pools' heads and consecutive query heads share a KV head.
    Sequence b attends its last `window` tokens (0 = all) of context_lens[b]; token t lies in page
    block_table[b, t // page_tokens].  scale defaults to dim ** -0.5.  A sequence without tokens gives zeros.  What pages
    hold behind a sequence's end never takes part, and neither do tokens on pages outside the pool; those pages, and
    lengths beyond the table (cut to it), are counted in `status`.

    lse: float32 [sequences, q_heads], receives the logarithm of the softmax sum (negative infinity without tokens).
    weights: float32 [sequences, 1 or kv_heads, >= table tokens]; weights_out (default: weights itself) receives weights plus
    the attention each token got, summed over the query heads of its KV head or, with one weight head, over all of
    them - what batch_evict_kv_pages ranks by.  Entries that are not attended are left as they are."""
    _no_grad(query, k_pool, v_pool, weights)
    pools = _pools(k_pool, v_pool)
    batch, width = _sequences(block_table, context_lens, k_pool)
    _heads(query, "query", k_pool, batch)
    n_q_heads, n_kv_heads, dim = query.shape[1], k_pool.shape[2], k_pool.shape[3]
    if n_q_heads == 0 or n_q_heads % n_kv_heads:
        raise ValueError("%d query heads are not a multiple of %d KV heads" % (n_q_heads, n_kv_heads))
    if window < 0:
        raise ValueError("window must not be negative")
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    elif out.shape != query.shape or out.dtype != query.dtype or out.device != query.device or not out.is_contiguous():
        raise ValueError("out must be contiguous, of query's shape, type and device")
    if lse is not None and (lse.shape != query.shape[:2] or lse.dtype != torch.float32 or lse.device != query.device or
                            not lse.is_contiguous()):
        raise ValueError("lse must be a contiguous float32 [sequences, q_heads] tensor on the pools' device")
    tokens = width * k_pool.shape[1]
    w_args = (0, 0, 0, 0, 0, 0, 0)
    if weights is not None:
        _per_slot(weights, "weights", torch.float32, k_pool, batch, tokens)
        if weights_out is None:
            weights_out = weights
        else:
            _per_slot(weights_out, "weights_out", torch.float32, k_pool, batch, tokens, weights.shape[1])
        _own_rows(weights_out, "weights_out")
        w_args = (weights.data_ptr(), weights.stride(0), weights.stride(1), weights_out.data_ptr(),
                  weights_out.stride(0), weights_out.stride(1), weights.shape[1])
    elif weights_out is not None:
        raise ValueError("weights_out without weights")
    size = _attend_workspace_bytes(batch, n_q_heads, n_kv_heads, dim, tokens, int(weights is not None))
    workspace = _workspace(size, k_pool.device, "kvcm_b200_attend_pages")
    _launch("kvcm_b200_attend_pages", k_pool.device, pools, query.data_ptr(), query.stride(0), query.stride(1), batch,
            n_q_heads, block_table.data_ptr(), block_table.stride(0), width, context_lens.data_ptr(),
            dim ** -0.5 if scale is None else float(scale), int(window), out.data_ptr(),
            0 if lse is None else lse.data_ptr(), *w_args, workspace.data_ptr(), size, _status_ptr(status, k_pool))
    return out


def batch_evict_kv_pages(k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor,
                         context_lens: torch.Tensor, weights: torch.Tensor, positions: torch.Tensor, budget: int,
                         recent: int = 0, weights_out: Optional[torch.Tensor] = None,
                         positions_out: Optional[torch.Tensor] = None,
                         status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Cuts every sequence longer than `budget` slots to its `budget` best tokens; returns the new lengths (int32).

    weights float32 and positions int32, both [sequences, 1 or kv_heads, >= table tokens]: of each slot in use the
    accumulated attention (batch_attend_kv_pages) and the position its token has in the text.  Kept are the tokens
    whose position is among the `recent` newest, then the heaviest; among equals the one in the lower slot (NaN counts
    as the heaviest).  With one weight head all KV heads keep the same tokens, else each head its own.  Survivors in
    slots from `budget` on move into the slots freed below it - rows of both pools, weight and position - so that
    the first `budget` slots hold what is kept, in no particular order, and the pages behind them are free.  The freed
    slots get weight 0 and position -1.  Results go into `weights` and `positions` themselves unless `weights_out` or
    `positions_out` are given, which then receive every slot in use.

    Pages are packed in place: a page that two sequences share must be copied first.  A move from or to a page outside
    the pool is left out and counted in `status`, as is a length beyond the table (cut to it)."""
    _no_grad(k_pool, v_pool, weights)
    pools = _pools(k_pool, v_pool)
    batch, width = _sequences(block_table, context_lens, k_pool)
    tokens = width * k_pool.shape[1]
    if budget < 1 or recent < 0 or recent > budget:
        raise ValueError("0 <= recent <= budget and budget >= 1 are needed, got recent=%r budget=%r" % (recent, budget))
    _per_slot(weights, "weights", torch.float32, k_pool, batch, tokens)
    heads = weights.shape[1]
    _per_slot(positions, "positions", torch.int32, k_pool, batch, tokens, heads)
    if weights_out is None:
        weights_out = weights
    else:
        _per_slot(weights_out, "weights_out", torch.float32, k_pool, batch, tokens, heads)
    if positions_out is None:
        positions_out = positions
    else:
        _per_slot(positions_out, "positions_out", torch.int32, k_pool, batch, tokens, heads)
    _own_rows(weights_out, "weights_out")
    _own_rows(positions_out, "positions_out")
    new_lens = torch.empty(batch, dtype=torch.int32, device=k_pool.device)
    budget = min(int(budget), max(tokens, 1))
    size = _evict_workspace_bytes(batch, heads, tokens, budget)
    workspace = _workspace(size, k_pool.device, "kvcm_b200_evict_pages")
    _launch("kvcm_b200_evict_pages", k_pool.device, pools, batch, block_table.data_ptr(), block_table.stride(0), width,
            context_lens.data_ptr(), budget, min(int(recent), budget), heads, weights.data_ptr(), weights.stride(0),
            weights.stride(1), positions.data_ptr(), positions.stride(0), positions.stride(1), weights_out.data_ptr(),
            weights_out.stride(0), weights_out.stride(1), positions_out.data_ptr(), positions_out.stride(0),
            positions_out.stride(1), new_lens.data_ptr(), workspace.data_ptr(), size, _status_ptr(status, k_pool))
    return new_lens
