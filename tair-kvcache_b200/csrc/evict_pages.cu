// Eviction from a paged cache by accumulated attention weight.
//
// Per sequence and weight head: rank the slots in use - protected ones (the newest tokens) first, then by weight, ties to
// the lower slot - keep the first `budget`, and pack the survivors into the first `budget` slots.  Survivors below
// `budget` stay; the others move into the holes.  Sources lie at or above `budget`, destinations below, so all moves of
// a head are independent of one another, and only as many rows move as there are holes: one per step in a cache that
// grows by one token per step, where packing in order would move up to the whole cache.
//
// The rank is not sorted out: the weight becomes a 32-bit key whose unsigned order is the rank, and the budget-th largest
// key is found by counting digits (11, 11 and 10 bits) in shared memory.  One thread-block cluster takes one head of
// one sequence; each CTA holds its slice of the keys in shared memory, and the digit counts are added up over distributed
// shared memory.  That kernel is a chain of short phases, bound by their latencies; it leaves a list of moves.  The
// second kernel is bound by HBM: it spreads the moves of all heads over the whole GPU, so that one long sequence is
// packed by every SM.  (One kernel for both left the rows of a head to the cluster that ranked it: 703 us instead of 61
// for 131,072 slots of eight heads.)
#include <cooperative_groups.h>

#include "paged_kv.cuh"

namespace cg = cooperative_groups;

namespace kvcm {
namespace {

constexpr int kEvictThreads = 512;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr uint32_t kKeyProtected = 0xFFFFFFFFu;
constexpr uint32_t kKeyNan = 0xFFFFFFFEu;
// Keys a CTA keeps in shared memory; longer slices are read again from global memory in every pass.
constexpr int kMaxCachedKeys = 49152;
constexpr int kMoveThreads = 256;
constexpr int kMovePieces = 4096;  // 16-byte pieces a block copies at a time, about
constexpr int kMaxMovesAtOnce = 128;

struct EvictParams {
    PagedPools pools;
    const int32_t *table;
    const int32_t *lens;
    const float *weights;
    const int32_t *positions;
    float *weights_out;
    int32_t *positions_out;
    int32_t *new_lens;
    int2 *moves;        // [batch * heads][max_moves], {source slot, destination slot}
    int32_t *n_moves;   // [batch * heads]
    uint32_t *status;
    int64_t table_stride;
    int64_t w_batch, w_head, p_batch, p_head, wo_batch, wo_head, po_batch, po_head;
    int64_t max_moves;
    int32_t table_width;
    int32_t table_tokens;
    int32_t n_heads;         // weight heads
    int32_t heads_per_move;  // KV heads that move together
    int32_t budget, recent;
    int32_t chunks;  // 16-byte pieces of a row
    int32_t separate_out;
    int32_t units;           // batch * weight heads
    int32_t moves_at_once;   // of a block of the second kernel
    int32_t blocks_per_unit;
};

struct EvictShared {
    uint32_t hist[kBins];
    uint32_t warp_sum[kEvictWarps];
    uint32_t prefix;   // digits found so far
    uint32_t above;    // keys still to be kept within the prefix
    uint32_t counts;   // this CTA's keys equal to the threshold
    uint32_t holes;    // this CTA's holes
    uint32_t movers;   // this CTA's movers
    int32_t newest;
    uint32_t total;
};

// Unsigned order of the result = order of the weights; both zeros are equal, NaN is the largest.
__device__ __forceinline__ uint32_t WeightKey(float w) {
    if (w != w) return kKeyNan;
    const uint32_t u = __float_as_uint(w + 0.0f);  // -0 becomes +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive scan of one value per thread; every thread also gets the total.
__device__ __forceinline__ uint32_t BlockExclusive(uint32_t value, EvictShared &sh, uint32_t *total) {
    const uint32_t lane = LaneId(), warp = threadIdx.x >> 5;
    uint32_t inclusive = value;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, inclusive, d);
        if (lane >= d) inclusive += up;
    }
    __syncthreads();
    if (lane == 31) sh.warp_sum[warp] = inclusive;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kEvictWarps; ++w) {
        const uint32_t s = sh.warp_sum[w];
        if (w < static_cast<int>(warp)) before += s;
        all += s;
    }
    *total = all;
    return before + inclusive - value;
}

template <bool kCached>
__global__ void __launch_bounds__(kEvictThreads, 2) EvictPagesKernel(const EvictParams p) {
    extern __shared__ uint32_t keys[];
    __shared__ EvictShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t n_ranks = cluster.num_blocks();
    const uint32_t rank = cluster.block_rank();
    const uint32_t unit = blockIdx.x / n_ranks;
    const uint32_t seq = unit / p.n_heads;
    const uint32_t head = unit - seq * p.n_heads;
    const uint32_t tid = threadIdx.x, lane = LaneId();
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");

    int32_t n = __ldg(p.lens + seq);
    if (n > p.table_tokens) {
        if (head == 0 && rank == 0 && tid == 0) CountSkipped(p.status, seq, 1u);
        n = p.table_tokens;
    }
    n = max(n, 0);
    const int32_t k = min(n, p.budget);
    if (head == 0 && rank == 0 && tid == 0) p.new_lens[seq] = k;
    const float *w_in = p.weights + seq * p.w_batch + head * p.w_head;
    const int32_t *pos_in = p.positions + seq * p.p_batch + head * p.p_head;
    float *w_out = p.weights_out + seq * p.wo_batch + head * p.wo_head;
    int32_t *pos_out = p.positions_out + seq * p.po_batch + head * p.po_head;
    if (n <= p.budget) {
        if (rank == 0 && tid == 0) p.n_moves[unit] = 0;
        if (p.separate_out) {
            for (int32_t i = rank * kEvictThreads + tid; i < n; i += n_ranks * kEvictThreads) {
                w_out[i] = w_in[i];
                pos_out[i] = pos_in[i];
            }
        }
        return;  // every CTA of the cluster leaves here
    }

    // This CTA's slice of the slots; within it a thread owns `per` consecutive ones, an odd number so that a warp's
    // reads of the key array spread over the banks.
    const int32_t slice = (n + n_ranks - 1) / n_ranks;
    const int32_t per = ((slice + kEvictThreads - 1) / kEvictThreads) | 1;
    const int32_t first = min(n, static_cast<int32_t>(rank) * slice);
    const int32_t count = min(n, first + slice) - first;

    // The largest position in use, over the cluster.
    int32_t newest = INT32_MIN;
    for (int32_t i = tid; i < count; i += kEvictThreads) newest = max(newest, pos_in[first + i]);
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (tid == 0) sh.newest = INT32_MIN;
    __syncthreads();
    if (lane == 0) atomicMax(&sh.newest, newest);
    cluster.sync();
    newest = INT32_MIN;
    for (uint32_t r = 0; r < n_ranks; ++r) newest = max(newest, cluster.map_shared_rank(&sh, r)->newest);
    const int64_t oldest_safe = static_cast<int64_t>(newest) - p.recent;  // protected: position > oldest_safe

    auto make_key = [&](int32_t i) -> uint32_t {
        return pos_in[first + i] > oldest_safe ? kKeyProtected : WeightKey(w_in[first + i]);
    };
    auto key_at = [&](int32_t i) -> uint32_t { return kCached ? keys[i] : make_key(i); };
    if (kCached) {
        for (int32_t i = tid; i < count; i += kEvictThreads) keys[i] = make_key(i);
    }

    // The k-th largest key, digit by digit from the top.
    if (tid == 0) {
        sh.prefix = 0;
        sh.above = static_cast<uint32_t>(k);
    }
    uint32_t mask = 0;  // bits of the key settled so far
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
        const uint32_t bins = pass == 2 ? 1024u : 2048u;
        for (uint32_t b = tid; b < kBins; b += kEvictThreads) sh.hist[b] = 0;
        __syncthreads();
        const uint32_t prefix = sh.prefix;
        for (int32_t i = tid; i < count; i += kEvictThreads) {
            const uint32_t key = key_at(i);
            if ((key & mask) == prefix) atomicAdd(&sh.hist[(key >> shift) & (bins - 1)], 1u);
        }
        cluster.sync();
        // Thread t adds up bins 4t' .. of the whole cluster, from the top bin down.
        constexpr int kPer = kBins / kEvictThreads;
        uint32_t sums[kPer];
        uint32_t mine = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const uint32_t bin = kBins - 1 - (tid * kPer + j);
            sums[j] = 0;
            for (uint32_t r = 0; r < n_ranks; ++r) sums[j] += cluster.map_shared_rank(&sh, r)->hist[bin];
            mine += sums[j];
        }
        uint32_t total;
        uint32_t before = BlockExclusive(mine, sh, &total);
        const uint32_t wanted = sh.above;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const uint32_t bin = kBins - 1 - (tid * kPer + j);
            if (before < wanted && before + sums[j] >= wanted) {
                sh.prefix = prefix | (bin << shift);
                sh.above = wanted - before;
                sh.counts = sh.hist[bin];  // of this CTA
            }
            before += sums[j];
        }
        mask |= (bins - 1) << shift;
        cluster.sync();  // the counts are read by all before they are cleared
    }
    const uint32_t threshold = sh.prefix;
    const uint32_t equal_kept = sh.above;  // of the keys equal to the threshold, those in the lowest slots

    // Which slots are holes and which are movers, in slot order.
    uint32_t equal_base = 0;
    for (uint32_t r = 0; r < rank; ++r) equal_base += cluster.map_shared_rank(&sh, r)->counts;
    const int32_t begin = min(count, static_cast<int32_t>(tid) * per);
    const int32_t end = min(count, begin + per);
    uint32_t equal = 0;
    for (int32_t i = begin; i < end; ++i) equal += key_at(i) == threshold;
    uint32_t total;
    const uint32_t equal_first = equal_base + BlockExclusive(equal, sh, &total);
    uint32_t holes = 0, movers = 0, seen = equal_first;
    for (int32_t i = begin; i < end; ++i) {
        const uint32_t key = key_at(i);
        const bool kept = key > threshold || (key == threshold && seen++ < equal_kept);
        holes += !kept && first + i < k;
        movers += kept && first + i >= k;
    }
    uint32_t all_holes, all_movers;
    uint32_t hole_at = BlockExclusive(holes, sh, &all_holes);
    uint32_t mover_at = BlockExclusive(movers, sh, &all_movers);
    if (tid == 0) {
        sh.holes = all_holes;
        sh.movers = all_movers;
    }
    cluster.sync();
    uint32_t n_moves = 0;
    for (uint32_t r = 0; r < n_ranks; ++r) {
        const EvictShared *peer = cluster.map_shared_rank(&sh, r);
        if (r < rank) {
            hole_at += peer->holes;
            mover_at += peer->movers;
        }
        n_moves += peer->movers;
    }
    if (rank == 0 && tid == 0) p.n_moves[unit] = static_cast<int32_t>(n_moves);
    cluster.sync();  // a CTA's shared memory may go once its peers have read it
    int2 *moves = p.moves + static_cast<int64_t>(unit) * p.max_moves;
    seen = equal_first;
    for (int32_t i = begin; i < end; ++i) {
        const uint32_t key = key_at(i);
        const bool kept = key > threshold || (key == threshold && seen++ < equal_kept);
        const int32_t slot = first + i;
        if (slot < k) {
            if (!kept) {
                moves[hole_at++].y = slot;
            } else if (p.separate_out) {
                w_out[slot] = w_in[slot];
                pos_out[slot] = pos_in[slot];
            }
        } else if (kept) {
            moves[mover_at++].x = slot;
        } else {
            w_out[slot] = 0.0f;
            pos_out[slot] = -1;
        }
    }
}

// The moves: rows of K and V in 16-byte pieces, weight and position; the slot a token leaves becomes free.
__global__ void __launch_bounds__(kMoveThreads) MoveSlotsKernel(const EvictParams p) {
    __shared__ int64_t from_row[kMaxMovesAtOnce], to_row[kMaxMovesAtOnce];
    const uint32_t tid = threadIdx.x;
    const uint32_t pieces = 2u * p.chunks * p.heads_per_move;  // of one move: K and V rows of every head that moves
    const int64_t blocks = static_cast<int64_t>(p.units) * p.blocks_per_unit;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
        const int32_t unit = static_cast<int32_t>(block / p.blocks_per_unit);
        const int32_t at = static_cast<int32_t>(block - static_cast<int64_t>(unit) * p.blocks_per_unit) * p.moves_at_once;
        const int32_t here = min(p.moves_at_once, __ldcg(p.n_moves + unit) - at);
        if (here <= 0) continue;
        const int32_t seq = unit / p.n_heads, head = unit - seq * p.n_heads;
        __syncthreads();
        if (static_cast<int32_t>(tid) < here) {
            const int2 m = __ldcg(p.moves + static_cast<int64_t>(unit) * p.max_moves + at + tid);
            const int32_t *table = p.table + seq * p.table_stride;
            const int32_t sp = m.x / p.pools.page_tokens, dp = m.y / p.pools.page_tokens;
            const int64_t src_page = __ldg(table + sp), dst_page = __ldg(table + dp);
            const int64_t w_from = seq * p.w_batch + head * p.w_head, p_from = seq * p.p_batch + head * p.p_head;
            const float w = p.weights[w_from + m.x];
            const int32_t position = p.positions[p_from + m.x];
            int64_t src = -1, dst = -1;
            if (src_page >= 0 && src_page < p.pools.pool_pages && dst_page >= 0 && dst_page < p.pools.pool_pages) {
                const int64_t head_off = p.n_heads > 1 ? head * p.pools.head_stride : 0;
                src = src_page * p.pools.page_stride + (m.x - sp * p.pools.page_tokens) * p.pools.token_stride + head_off;
                dst = dst_page * p.pools.page_stride + (m.y - dp * p.pools.page_tokens) * p.pools.token_stride + head_off;
            } else {
                CountSkipped(p.status, static_cast<uint32_t>(seq), 1u);
            }
            from_row[tid] = src;
            to_row[tid] = dst;
            float *w_out = p.weights_out + seq * p.wo_batch + head * p.wo_head;
            int32_t *pos_out = p.positions_out + seq * p.po_batch + head * p.po_head;
            w_out[m.y] = w;
            pos_out[m.y] = position;
            w_out[m.x] = 0.0f;
            pos_out[m.x] = -1;
        }
        __syncthreads();
        const uint32_t n_pieces = static_cast<uint32_t>(here) * pieces;
        constexpr int kUnroll = 4;
        for (uint32_t base = tid; base < n_pieces; base += kMoveThreads * kUnroll) {
            uint4 data[kUnroll];
            uint8_t *to[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const uint32_t f = base + u * kMoveThreads;
                to[u] = nullptr;
                if (f < n_pieces) {
                    const uint32_t m = f / pieces;
                    const uint32_t within = f - m * pieces;
                    const uint32_t row = within / p.chunks;
                    const int64_t off = static_cast<int64_t>(row >> 1) * p.pools.head_stride +
                                        static_cast<int64_t>(within - row * p.chunks) * 16;
                    uint8_t *pool = (row & 1) ? p.pools.v : p.pools.k;
                    if (from_row[m] >= 0) {
                        data[u] = __ldcs(reinterpret_cast<const uint4 *>(pool + from_row[m] + off));
                        to[u] = pool + to_row[m] + off;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if (to[u] != nullptr) *reinterpret_cast<uint4 *>(to[u]) = data[u];
            }
        }
    }
}

int64_t EvictMaxMoves(int64_t table_tokens, int32_t budget) {
    return std::max<int64_t>(0, std::min<int64_t>(budget, table_tokens - budget));
}

// The workspace: the lists of moves, then their lengths.
int64_t EvictMovesBytes(int64_t units, int64_t table_tokens, int32_t budget) {
    return (units * EvictMaxMoves(table_tokens, budget) * 8 + 255) / 256 * 256;
}

}  // namespace
}  // namespace kvcm

extern "C" {

int64_t kvcm_b200_evict_workspace_bytes(int32_t batch, int32_t n_weight_heads, int64_t table_tokens, int32_t budget) {
    if (batch < 0 || n_weight_heads <= 0 || table_tokens < 0 || table_tokens > kvcm::kMaxTableTokens || budget <= 0) return -1;
    const int64_t units = static_cast<int64_t>(batch) * n_weight_heads;
    return kvcm::EvictMovesBytes(units, table_tokens, budget) + std::max<int64_t>(256, (units * 4 + 255) / 256 * 256);
}

int32_t kvcm_b200_evict_pages(const kvcm_b200_kv_pools_t *pools, int32_t batch, const int32_t *d_block_table,
                              int64_t table_stride, int32_t table_width, const int32_t *d_context_lens, int32_t budget,
                              int32_t recent, int32_t n_weight_heads, const float *d_weights, int64_t w_batch_stride,
                              int64_t w_head_stride, const int32_t *d_positions, int64_t p_batch_stride,
                              int64_t p_head_stride, float *d_weights_out, int64_t wo_batch_stride,
                              int64_t wo_head_stride, int32_t *d_positions_out, int64_t po_batch_stride,
                              int64_t po_head_stride, int32_t *d_new_lens, void *d_workspace, int64_t workspace_bytes,
                              uint32_t *d_status, kvcm_stream_t stream) {
    using namespace kvcm;
    const int32_t rc = CheckPools(pools, INT32_MAX);
    if (rc != KVCM_OK) return rc;
    const int64_t table_tokens = static_cast<int64_t>(table_width) * pools->page_tokens;
    if (batch < 0 || table_width < 0 || budget < 1 || recent < 0 || recent > budget ||
        (n_weight_heads != 1 && n_weight_heads != pools->n_kv_heads)) {
        return KVCM_ER_INVALID_PARAMS;
    }
    if (table_tokens > kMaxTableTokens || static_cast<int64_t>(batch) * n_weight_heads > (1 << 27)) return KVCM_EC_OUT_OF_LIMIT;
    const bool any_slots = batch > 0 && table_width > 0;
    if ((any_slots && (d_block_table == nullptr || d_weights == nullptr || d_positions == nullptr ||
                       d_weights_out == nullptr || d_positions_out == nullptr)) ||
        (batch > 0 && (d_context_lens == nullptr || d_new_lens == nullptr || d_workspace == nullptr)) ||
        !RowsAre16ByteAligned(*pools) || (reinterpret_cast<uintptr_t>(d_workspace) & 15u) != 0) {
        return KVCM_ER_INVALID_ADDRESS;
    }
    // The lengths are read by every CTA of a sequence at its own time, so the new ones go elsewhere; arrays updated in
    // place are updated entry by entry.
    const uintptr_t lens_at = reinterpret_cast<uintptr_t>(d_context_lens), new_at = reinterpret_cast<uintptr_t>(d_new_lens);
    if ((new_at < lens_at ? lens_at - new_at : new_at - lens_at) < static_cast<uintptr_t>(batch) * 4 ||
        (d_weights_out == d_weights && (wo_batch_stride != w_batch_stride || wo_head_stride != w_head_stride)) ||
        (d_positions_out == d_positions && (po_batch_stride != p_batch_stride || po_head_stride != p_head_stride))) {
        return KVCM_ER_INVALID_PARAMS;
    }
    if (workspace_bytes < kvcm_b200_evict_workspace_bytes(batch, n_weight_heads, table_tokens, budget)) {
        return KVCM_ER_INVALID_PARAMS;
    }
    if (!HaveDevice()) return KVCM_ER_NO_DEVICE;
    if (batch == 0) return KVCM_OK;
    EvictParams p = {};
    p.pools = AsPagedPools(*pools);
    p.table = d_block_table;
    p.lens = d_context_lens;
    p.weights = d_weights;
    p.positions = d_positions;
    p.weights_out = d_weights_out;
    p.positions_out = d_positions_out;
    p.new_lens = d_new_lens;
    p.moves = static_cast<int2 *>(d_workspace);
    p.status = d_status;
    p.table_stride = table_stride;
    p.w_batch = w_batch_stride;
    p.w_head = w_head_stride;
    p.p_batch = p_batch_stride;
    p.p_head = p_head_stride;
    p.wo_batch = wo_batch_stride;
    p.wo_head = wo_head_stride;
    p.po_batch = po_batch_stride;
    p.po_head = po_head_stride;
    p.max_moves = EvictMaxMoves(table_tokens, budget);
    p.table_width = table_width;
    p.table_tokens = static_cast<int32_t>(table_tokens);
    p.n_heads = n_weight_heads;
    p.heads_per_move = n_weight_heads == 1 ? pools->n_kv_heads : 1;
    p.budget = budget;
    p.recent = recent;
    p.chunks = pools->head_dim / 8;
    p.separate_out = d_weights_out != d_weights || d_positions_out != d_positions;

    // As many CTAs as fit two to an SM, but none with fewer than about a thousand slots, and slices that fit shared memory.
    const int64_t units = static_cast<int64_t>(batch) * n_weight_heads;
    const int32_t sm_count = GetDeviceInfo().sm_count;
    int cluster = 1;
    while (cluster < kMaxCluster && units * cluster * 2 <= 2 * sm_count && table_tokens / (cluster * 2) >= 1024) cluster *= 2;
    while (cluster < kMaxCluster && (table_tokens + cluster - 1) / cluster > kMaxCachedKeys) cluster *= 2;
    const int64_t slice = (table_tokens + cluster - 1) / cluster;
    const bool cached = slice <= kMaxCachedKeys;
    p.units = static_cast<int32_t>(units);
    p.n_moves = reinterpret_cast<int32_t *>(static_cast<uint8_t *>(d_workspace) + EvictMovesBytes(units, table_tokens, budget));
    const int32_t pieces = 2 * p.chunks * p.heads_per_move;
    p.moves_at_once = std::min(kMaxMovesAtOnce, std::max(1, kMovePieces / pieces));
    p.blocks_per_unit = static_cast<int32_t>((p.max_moves + p.moves_at_once - 1) / p.moves_at_once);

    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<uint32_t>(units * cluster));
    cfg.blockDim = dim3(kEvictThreads);
    cfg.dynamicSmemBytes = cached ? static_cast<size_t>(slice) * 4 : 0;
    cfg.stream = AsStream(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cached) {
        EnsureDynamicSmem(EvictPagesKernel<true>, kMaxCachedKeys * 4);
        cudaLaunchKernelEx(&cfg, EvictPagesKernel<true>, p);
    } else {
        cudaLaunchKernelEx(&cfg, EvictPagesKernel<false>, p);
    }
    if (p.blocks_per_unit == 0) return LaunchStatus();  // the budget is not below what the table holds
    cudaLaunchConfig_t move = {};
    move.gridDim = dim3(static_cast<uint32_t>(std::min<int64_t>(units * p.blocks_per_unit, 8 * sm_count)));
    move.blockDim = dim3(kMoveThreads);
    move.stream = cfg.stream;
    cudaLaunchAttribute early[1];
    early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early[0].val.programmaticStreamSerializationAllowed = 1;
    move.attrs = early;
    move.numAttrs = 1;
    cudaLaunchKernelEx(&move, MoveSlotsKernel, p);
    return LaunchStatus();
}

}  // extern "C"
