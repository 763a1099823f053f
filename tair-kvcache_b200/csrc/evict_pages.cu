// Eviction from a paged cache by accumulated attention weight.
//
// Per sequence and weight head: rank the slots in use - protected ones (the newest tokens) first, then by weight, ties to
// the lower slot - keep the first `budget`, and pack the survivors into the first `budget` slots.  Survivors below
// `budget` stay; the others move into the holes.  Sources lie at or above `budget`, destinations below, so all moves of
// a head are independent of one another, and only as many rows move as there are holes: one per step in a cache that
// grows by one token per step, where packing in order would move up to the whole cache.
//
// The rank is not sorted out: the weight becomes a 32-bit key whose unsigned order is the rank, and the budget-th largest
// key is found by counting its four bytes, from the top, in shared memory.  One CTA takes one head of one sequence, or a
// thread-block cluster does, each CTA with a slice of the keys in shared memory and the counts added up over distributed
// shared memory.  That kernel is a chain of short phases, bound by their latencies; it leaves a list of moves.  The
// second kernel is bound by HBM: it spreads the moves of all heads over the whole GPU, so that one long sequence is
// packed by every SM.  (One kernel for both left the rows of a head to the cluster that ranked it: 703 us for 131,072
// slots of eight heads instead of 59.)
//
// 128 heads of 6001 to 8192 slots cut to 4096, rows of 256 bytes: 64 us, 18 to rank, 45 to move (5.4 TB/s read and
// written, 83 % of a plain copy: 256-byte rows scattered on both sides).  One sequence of 131,072 slots cut to 32,768, all
// heads together: 23 us and 33 us (96 %).  256 heads one slot over their budget: 14 us together, a chain of latencies.
// Counting with warp-wide matches instead of four copies of the counts took 29 and 61 us to rank the first two; reading
// all four copies of every peer instead of their sum 22 and 37; moving with plain instead of streaming stores 49 and 36.
#include <cooperative_groups.h>

#include <cstddef>

#include "paged_kv.cuh"

namespace cg = cooperative_groups;

namespace kvcm {
namespace {

constexpr int kEvictThreads = 512;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kBins = 256;
constexpr int kPasses = 4;
constexpr int kCopies = 4;  // of the counts, for lanes that count the same byte: weights share their high ones
constexpr int kMaxCluster = 16;
constexpr int kPortableCluster = 8;  // beyond it a launch opts in
constexpr uint32_t kKeyProtected = 0xFFFFFFFFu;
constexpr uint32_t kKeyNan = 0xFFFFFFFEu;
constexpr uint32_t kAll = 0xFFFFFFFFu;
// Slots a CTA keeps in shared memory, key and position; longer slices are read again from global memory in every pass.
constexpr int kMaxCachedSlots = 22528;
constexpr int kLoads = 8;  // loads of a thread in flight together
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
    int32_t table_tokens;
    int32_t n_heads;         // weight heads
    int32_t heads_per_move;  // KV heads that move together
    int32_t budget, recent;
    int32_t separate_out;
    FastDivide pieces;       // 16-byte pieces of one move: K and V rows of every head that moves
    FastDivide row_pieces;   // of a row
    int32_t units;           // batch * weight heads
    int32_t moves_at_once;   // of a block of the second kernel
    int32_t blocks_per_unit;
};

template <bool kCluster>
struct alignas(16) EvictShared {
    uint32_t counts[kCluster ? kPasses : 1][kBins];  // of this CTA, the copies added up, for its peers
    uint32_t total[kBins];                           // of the cluster, in the pass at hand; read 16 bytes at a time
    uint32_t hist[kPasses][kCopies][kBins + 8];
    uint2 warp_sum[kEvictWarps];
    uint32_t prefix;  // bytes found so far
    uint32_t wanted;  // keys still to be kept within the prefix
    uint32_t equal;   // this CTA's keys equal to the threshold
    uint32_t holes;   // this CTA's holes
    uint32_t movers;  // this CTA's movers
    int32_t newest;
};
static_assert(alignof(EvictShared<true>) == 16 && offsetof(EvictShared<true>, total) % 16 == 0, "total is read as uint4");
static_assert(alignof(EvictShared<false>) == 16 && offsetof(EvictShared<false>, total) % 16 == 0, "total is read as uint4");

// Unsigned order of the result = order of the weights; both zeros are equal, NaN is the largest.
__device__ __forceinline__ uint32_t WeightKey(float w) {
    if (w != w) return kKeyNan;
    const uint32_t u = __float_as_uint(w + 0.0f);  // -0 becomes +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive sums over the warps of two values that each warp's lanes agree on; every thread also gets the totals.
template <bool kCluster>
__device__ __forceinline__ uint2 WarpsExclusive(uint2 value, EvictShared<kCluster> &sh, uint2 *total) {
    const uint32_t warp = threadIdx.x >> 5;
    __syncthreads();
    if (LaneId() == 0) sh.warp_sum[warp] = value;
    __syncthreads();
    uint2 before = make_uint2(0, 0), all = make_uint2(0, 0);
#pragma unroll
    for (int w = 0; w < kEvictWarps; ++w) {
        const uint2 s = sh.warp_sum[w];
        if (w < static_cast<int>(warp)) {
            before.x += s.x;
            before.y += s.y;
        }
        all.x += s.x;
        all.y += s.y;
    }
    *total = all;
    return before;
}

template <bool kCluster, bool kCached>
__global__ void __launch_bounds__(kEvictThreads, 2) EvictPagesKernel(const __grid_constant__ EvictParams p) {
    extern __shared__ uint32_t slots[];  // keys, then positions, of this CTA's slice
    __shared__ EvictShared<kCluster> sh;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t n_ranks = kCluster ? cluster.num_blocks() : 1;
    const uint32_t rank = kCluster ? cluster.block_rank() : 0;
    auto sync_all = [&]() {
        if (kCluster) {
            cluster.sync();
        } else {
            __syncthreads();
        }
    };
    auto peer = [&](uint32_t r) -> const EvictShared<kCluster> & { return kCluster ? *cluster.map_shared_rank(&sh, r) : sh; };
    const uint32_t unit = blockIdx.x / n_ranks;
    const uint32_t seq = unit / p.n_heads;
    const uint32_t head = unit - seq * p.n_heads;
    const uint32_t tid = threadIdx.x, lane = LaneId(), warp = tid >> 5;
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

    const int32_t slice = (n + n_ranks - 1) / n_ranks;  // of the slots; the last one's may be shorter
    const int32_t first = min(n, static_cast<int32_t>(rank) * slice);
    const int32_t count = min(n, first + slice) - first;
    w_in += first;
    pos_in += first;
    uint32_t *keys = slots;
    int32_t *ages = reinterpret_cast<int32_t *>(slots + slice);
    uint32_t *kept_bits = slots + slice;  // in the place of the positions, once the keys account for them

    // Weights and positions into shared memory; the largest position in use, over the cluster.
    for (uint32_t i = tid; i < sizeof(sh.hist) / 4; i += kEvictThreads) (&sh.hist[0][0][0])[i] = 0;
    if (tid == 0) {
        sh.newest = INT32_MIN;
        sh.prefix = 0;
        sh.wanted = static_cast<uint32_t>(k);
    }
    int32_t newest = INT32_MIN;
    for (int32_t i0 = tid; i0 < count; i0 += kLoads * kEvictThreads) {
        float w[kLoads];
        int32_t age[kLoads];
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int32_t i = i0 + j * kEvictThreads;
            age[j] = INT32_MIN;
            if (i < count) {
                age[j] = pos_in[i];
                if (kCached) w[j] = w_in[i];
            }
        }
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int32_t i = i0 + j * kEvictThreads;
            newest = max(newest, age[j]);
            if (kCached && i < count) {
                keys[i] = WeightKey(w[j]);
                ages[i] = age[j];
            }
        }
    }
    newest = __reduce_max_sync(0xffffffffu, newest);
    __syncthreads();
    if (lane == 0) atomicMax(&sh.newest, newest);
    sync_all();
    newest = sh.newest;
    if (kCluster) {
        for (uint32_t r = 0; r < n_ranks; ++r) newest = max(newest, peer(r).newest);
    }
    const int64_t oldest_safe = static_cast<int64_t>(newest) - p.recent;  // protected: position > oldest_safe

    auto key_at = [&](int32_t i) -> uint32_t {
        if (kCached) return keys[i];
        return pos_in[i] > oldest_safe ? kKeyProtected : WeightKey(w_in[i]);
    };

    // The k-th largest key, byte by byte from the top.
    uint32_t prefix = 0, wanted = static_cast<uint32_t>(k);
#pragma unroll 1
    for (int pass = 0; pass < kPasses; ++pass) {
        const int shift = 24 - 8 * pass;
        const uint32_t mask = pass == 0 ? 0u : 0xffffffffu << (shift + 8);
        uint32_t *hist = sh.hist[pass][lane % kCopies];
#pragma unroll 4
        for (int32_t i = tid; i < count; i += kEvictThreads) {
            uint32_t key = key_at(i);
            if (kCached && pass == 0 && ages[i] > oldest_safe) keys[i] = key = kKeyProtected;
            if ((key & mask) == prefix) atomicAdd(hist + ((key >> shift) & 0xffu), 1u);
        }
        __syncthreads();
        uint32_t counted = 0;  // of byte tid, first in this CTA, then in the cluster
        if (tid < kBins) {
#pragma unroll
            for (int c = 0; c < kCopies; ++c) counted += sh.hist[pass][c][tid];
            if (kCluster) sh.counts[pass][tid] = counted;
        }
        if (kCluster) {
            cluster.sync();
            if (tid < kBins) {
                counted = 0;
#pragma unroll 4
                for (uint32_t r = 0; r < n_ranks; ++r) counted += peer(r).counts[pass][tid];
            }
        }
        if (tid < kBins) sh.total[tid] = counted;
        __syncthreads();
        if (warp == 0) {
            // Lane t takes the eight bytes 255 - 8 t .. 248 - 8 t, from the top down.
            const uint4 lo = *reinterpret_cast<const uint4 *>(&sh.total[248 - 8 * lane]);
            const uint4 hi = *reinterpret_cast<const uint4 *>(&sh.total[252 - 8 * lane]);
            const uint32_t sums[8] = {hi.w, hi.z, hi.y, hi.x, lo.w, lo.z, lo.y, lo.x};
            uint32_t mine = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) mine += sums[j];
            uint32_t inclusive = mine;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, inclusive, d);
                if (lane >= d) inclusive += up;
            }
            uint32_t before = inclusive - mine;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (before < wanted && before + sums[j] >= wanted) {
                    const uint32_t byte = 255 - (8 * lane + j);
                    sh.prefix = prefix | (byte << shift);
                    sh.wanted = before + sums[j] == wanted ? kAll : wanted - before;
                    // after the last pass, keys of this CTA that are equal to the threshold
                    sh.equal = kCluster ? sh.counts[pass][byte] : sums[j];
                }
                before += sums[j];
            }
        }
        __syncthreads();
        prefix = sh.prefix;
        wanted = sh.wanted;
        if (wanted == kAll) break;  // every key that begins with these bytes is kept: nothing is left to tell apart
    }
    const uint32_t threshold = prefix;
    const uint32_t equal_kept = wanted;  // of the keys equal to the threshold, those in the lowest slots
    const bool ties = wanted != kAll;

    // Which slots are holes and which are movers, in slot order: each warp goes through a stretch of the slice, 32
    // slots at a time.
    const int32_t stretch = ((count + kEvictWarps - 1) / kEvictWarps + 31) & ~31;
    const int32_t begin = min(count, static_cast<int32_t>(warp) * stretch), end = min(count, begin + stretch);
    const uint32_t below = (1u << lane) - 1u;
    uint32_t equal_before = 0;
    if (ties) {
        sync_all();
        if (kCluster) {
            for (uint32_t r = 0; r != rank; ++r) equal_before += peer(r).equal;
        }
        uint32_t equal = 0;
        for (int32_t i0 = begin; i0 < end; i0 += 32) {
            const int32_t i = i0 + static_cast<int32_t>(lane);
            equal += __popc(__ballot_sync(0xffffffffu, i < end && key_at(i) == threshold));
        }
        uint2 total;
        equal_before += WarpsExclusive(make_uint2(equal, 0), sh, &total).x;
    }
    // Whether the lane's slot is kept; `seen` counts the keys equal to the threshold so far.
    auto is_kept = [&](int32_t i, uint32_t &seen) -> bool {
        const uint32_t key = i < end ? key_at(i) : 0u;
        if (!ties) return i < end && key >= threshold;
        const bool equals = i < end && key == threshold;
        const uint32_t equals_mask = __ballot_sync(0xffffffffu, equals);
        const bool kept = i < end && (key > threshold || (equals && seen + __popc(equals_mask & below) < equal_kept));
        seen += __popc(equals_mask);
        return kept;
    };
    uint32_t holes = 0, movers = 0, seen = equal_before;
    for (int32_t i0 = begin; i0 < end; i0 += 32) {
        const int32_t i = i0 + static_cast<int32_t>(lane), slot = first + i;
        const bool kept = is_kept(i, seen);
        const uint32_t kept_mask = __ballot_sync(0xffffffffu, kept);
        const uint32_t low_mask = __ballot_sync(0xffffffffu, i < end && slot < k);
        holes += __popc(low_mask & ~kept_mask);
        movers += __popc(kept_mask & ~low_mask);
        if (kCached && lane == 0) kept_bits[i0 >> 5] = kept_mask;
    }
    uint2 all;
    const uint2 mine_at = WarpsExclusive(make_uint2(holes, movers), sh, &all);
    uint32_t hole_at = mine_at.x, mover_at = mine_at.y;
    if (tid == 0) {
        sh.holes = all.x;
        sh.movers = all.y;
    }
    uint32_t n_moves = all.y;
    if (kCluster) {
        cluster.sync();
        n_moves = 0;
        for (uint32_t r = 0; r < n_ranks; ++r) {
            if (kCluster && r < rank) {
                hole_at += peer(r).holes;
                mover_at += peer(r).movers;
            }
            n_moves += peer(r).movers;
        }
        cluster.barrier_arrive();  // a CTA's shared memory may go once its peers have read it: they wait at the end
    }
    if (rank == 0 && tid == 0) p.n_moves[unit] = static_cast<int32_t>(n_moves);
    int2 *moves = p.moves + static_cast<int64_t>(unit) * p.max_moves;
    seen = equal_before;
    for (int32_t i0 = begin; i0 < end; i0 += 32) {
        const int32_t i = i0 + static_cast<int32_t>(lane), slot = first + i;
        const bool kept = kCached ? (kept_bits[i0 >> 5] >> lane) & 1u : is_kept(i, seen);
        const bool hole = i < end && !kept && slot < k, mover = kept && slot >= k;
        const uint32_t hole_mask = __ballot_sync(0xffffffffu, hole), mover_mask = __ballot_sync(0xffffffffu, mover);
        if (hole) moves[hole_at + __popc(hole_mask & below)].y = slot;
        if (mover) moves[mover_at + __popc(mover_mask & below)].x = slot;
        hole_at += __popc(hole_mask);
        mover_at += __popc(mover_mask);
        if (i < end && !kept && slot >= k) {
            w_out[slot] = 0.0f;
            pos_out[slot] = -1;
        } else if (!kCached && p.separate_out && kept && slot < k) {
            w_out[slot] = w_in[i];
            pos_out[slot] = pos_in[i];
        }
    }
    if (kCached && p.separate_out) {  // survivors that stay
        __syncthreads();
        const int32_t low = min(count, k - first);
        for (int32_t i0 = tid; i0 < low; i0 += kLoads * kEvictThreads) {
            float w[kLoads];
            int32_t age[kLoads];
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int32_t i = i0 + j * kEvictThreads;
                if (i < low && ((kept_bits[i >> 5] >> (i & 31)) & 1u)) {
                    w[j] = w_in[i];
                    age[j] = pos_in[i];
                }
            }
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int32_t i = i0 + j * kEvictThreads;
                if (i < low && ((kept_bits[i >> 5] >> (i & 31)) & 1u)) {
                    w_out[first + i] = w[j];
                    pos_out[first + i] = age[j];
                }
            }
        }
    }
    if (kCluster) cluster.barrier_wait();
}

// The moves: rows of K and V in 16-byte pieces, weight and position; the slot a token leaves becomes free.
__global__ void __launch_bounds__(kMoveThreads) MoveSlotsKernel(const __grid_constant__ EvictParams p) {
    __shared__ int64_t from_row[kMaxMovesAtOnce], to_row[kMaxMovesAtOnce];
    const uint32_t tid = threadIdx.x;
    const int64_t blocks = static_cast<int64_t>(p.units) * p.blocks_per_unit;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
        // the first moves of every head, then the second ones: heads with fewer moves than there is room for run out last
        const int64_t turn = block / p.units;
        const int32_t unit = static_cast<int32_t>(block - turn * p.units);
        const int32_t at = static_cast<int32_t>(turn) * p.moves_at_once;
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
        const uint32_t n_pieces = static_cast<uint32_t>(here) * p.pieces.d;
        constexpr int kUnroll = 8;
        for (uint32_t base = tid; base < n_pieces; base += kMoveThreads * kUnroll) {
            uint4 data[kUnroll];
            uint8_t *to[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const uint32_t f = base + u * kMoveThreads;
                to[u] = nullptr;
                if (f < n_pieces) {
                    const uint32_t m = p.pieces(f);
                    const uint32_t within = f - m * p.pieces.d;
                    const uint32_t row = p.row_pieces(within);
                    const int64_t off = static_cast<int64_t>(row >> 1) * p.pools.head_stride +
                                        static_cast<int64_t>(within - row * p.row_pieces.d) * 16;
                    uint8_t *pool = (row & 1) ? p.pools.v : p.pools.k;
                    if (from_row[m] >= 0) {
                        data[u] = __ldcs(reinterpret_cast<const uint4 *>(pool + from_row[m] + off));
                        to[u] = pool + to_row[m] + off;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if (to[u] != nullptr) __stcs(reinterpret_cast<uint4 *>(to[u]), data[u]);
            }
        }
    }
}

// The opt-in to clusters of more than eight CTAs is per device and per kernel, like the one to large shared memory.
template <typename Kernel>
cudaError_t AllowLargeClusters(Kernel kernel) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}

// The largest cluster to launch: sixteen CTAs, each with an SM's shared memory, where the device (or the partition of it
// that the process has) can place that many side by side, else the eight that any can.  Asked once per device.
int LargestCluster() {
    static std::mutex mu;
    static std::vector<std::pair<int, int>> known;  // by device ordinal
    int device = 0;
    cudaGetDevice(&device);
    std::lock_guard<std::mutex> lock(mu);
    for (const auto &k : known) {
        if (k.first == device) return k.second;
    }
    auto *kernel = EvictPagesKernel<true, true>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kMaxCluster);
    cfg.blockDim = dim3(kEvictThreads);
    cfg.dynamicSmemBytes = kMaxCachedSlots * 8;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kMaxCluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    const bool placed = EnsureDynamicSmem(kernel, kMaxCachedSlots * 8) == cudaSuccess &&
                        AllowLargeClusters(kernel) == cudaSuccess &&
                        cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess && clusters > 0;
    if (!placed) cudaGetLastError();
    known.emplace_back(device, placed ? kMaxCluster : kPortableCluster);
    return known.back().second;
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
    EvictParams p{};
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
    p.table_tokens = static_cast<int32_t>(table_tokens);
    p.n_heads = n_weight_heads;
    p.heads_per_move = n_weight_heads == 1 ? pools->n_kv_heads : 1;
    p.budget = budget;
    p.recent = recent;
    p.row_pieces = FastDivide(static_cast<uint32_t>(pools->head_dim / 8));
    p.pieces = FastDivide(2 * p.row_pieces.d * static_cast<uint32_t>(p.heads_per_move));
    p.separate_out = d_weights_out != d_weights || d_positions_out != d_positions;

    // As many CTAs as fit two to an SM, but none with fewer than about a thousand slots, and slices that fit shared memory.
    const int64_t units = static_cast<int64_t>(batch) * n_weight_heads;
    const int32_t sm_count = GetDeviceInfo().sm_count;
    const int largest = LargestCluster();
    int cluster = 1;
    while (cluster < largest && units * cluster * 2 <= 2 * sm_count && table_tokens / (cluster * 2) >= 1024) cluster *= 2;
    while (cluster < largest && (table_tokens + cluster - 1) / cluster > kMaxCachedSlots) cluster *= 2;
    const int64_t slice = (table_tokens + cluster - 1) / cluster;
    const bool cached = slice <= kMaxCachedSlots;
    p.units = static_cast<int32_t>(units);
    p.n_moves = reinterpret_cast<int32_t *>(static_cast<uint8_t *>(d_workspace) + EvictMovesBytes(units, table_tokens, budget));
    p.moves_at_once = std::min(kMaxMovesAtOnce, std::max(1, kMovePieces / static_cast<int>(p.pieces.d)));
    p.blocks_per_unit = static_cast<int32_t>((p.max_moves + p.moves_at_once - 1) / p.moves_at_once);

    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<uint32_t>(units * cluster));
    cfg.blockDim = dim3(kEvictThreads);
    cfg.dynamicSmemBytes = cached ? static_cast<size_t>(slice) * 8 : 0;
    cfg.stream = AsStream(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    Requests requests;
    auto launch = [&](auto kernel) {
        if (cached) requests.Make([&] { return EnsureDynamicSmem(kernel, kMaxCachedSlots * 8); });
        if (cluster > kPortableCluster) requests.Make([&] { return AllowLargeClusters(kernel); });
        requests.Make([&] { return cudaLaunchKernelEx(&cfg, kernel, p); });
    };
    if (cluster > 1) {
        cached ? launch(EvictPagesKernel<true, true>) : launch(EvictPagesKernel<true, false>);
    } else {
        launch(EvictPagesKernel<false, true>);  // a slice too long for shared memory has made a cluster above
    }
    if (p.blocks_per_unit == 0) return requests.Status();  // the budget is not below what the table holds
    cudaLaunchConfig_t move = {};
    move.gridDim = dim3(static_cast<uint32_t>(std::min<int64_t>(units * p.blocks_per_unit, 8 * sm_count)));
    move.blockDim = dim3(kMoveThreads);
    move.stream = cfg.stream;
    cudaLaunchAttribute early[1];
    early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early[0].val.programmaticStreamSerializationAllowed = 1;
    move.attrs = early;
    move.numAttrs = 1;
    requests.Make([&] { return cudaLaunchKernelEx(&move, MoveSlotsKernel, p); });
    return requests.Status();
}

}  // extern "C"
