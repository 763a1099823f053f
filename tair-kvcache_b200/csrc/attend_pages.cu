// Attention of one new token per sequence over its paged keys and values, with the attention weights accumulated per
// cached token on request.
//
//   o_h = sum_t p_t V[t],  p = softmax_t(scale * q_h . K[t]),  t over the sequence's last `window` tokens or all.
//
// Bound by HBM: every K and V row is read once (512 bytes per token and KV head of 128), used by the group of query heads
// that share the KV head, 2 to 32 multiplications per byte.  One pass with a running maximum and sum; K and V rows go
// from HBM to shared memory by 16-byte asynchronous copies, each warp with a ring of its own, and from there by ldmatrix
// into 16x8x16 matrix instructions whose 16 rows are the group's query heads.  A group is far too small for the 128
// rows of the tcgen05 instructions, and the tensor pipe is idle most of the time as it is.
//
// Probabilities enter the second product as two 16-bit halves, p = hi + lo, whose sum carries 16 (bf16) or more bits,
// so the output is rounded once.  With a group of at most eight the halves cost nothing: hi takes rows 0-7 of the
// matrix instruction, lo the rows 8-15 that the group leaves free.
//
// The work is cut by tokens, not by sequences: the steps (kStep tokens of one KV head of one sequence) of the whole
// batch are numbered through, and each of the persistent CTAs takes an equal run of them, found from the lengths on the
// device.  A head that lies within one run is finished there; the runs of a head that is cut leave their unnormalised
// sums and statistics in the workspace, and the second kernel joins them, in order, so results do not depend on timing.
#include "paged_kv.cuh"

namespace kvcm {
namespace {

constexpr int kAttendWarps = 4;
constexpr int kAttendThreads = kAttendWarps * 32;
constexpr int kTile = 16;                     // tokens a warp takes per step
constexpr int kStep = kTile * kAttendWarps;   // tokens a CTA takes per step
constexpr int kMaxWorkers = 1024;
constexpr int kMaxAttendHeadDim = 256;
constexpr int kJoinThreads = 512;
constexpr int kWeightThreads = kJoinThreads;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;

struct AttendParams {
    PagedPools pools;
    const uint8_t *query;
    int64_t q_batch, q_head;  // in elements
    const int32_t *table;
    int64_t table_stride;
    const int32_t *lens;
    uint8_t *out;
    float *lse;
    uint32_t *status;
    const float *weights;
    float *weights_out;
    int64_t w_batch, w_head, wo_batch, wo_head;
    int32_t n_weight_heads;
    // workspace
    int64_t *steps_before;  // [batch + 1] steps of all sequences before this one, one KV head and row tile counted
    float *part_o;          // [workers * 2][rows][dim]
    float2 *part_ml;        // [workers * 2][rows] maximum and sum of a share, the maximum in units of log2
    float2 *whole_ml;       // [batch][n_q_heads], heads that one CTA finished
    float *scores;          // [batch][n_q_heads][score_stride], in units of log2; null without weights
    int64_t score_stride;
    int32_t batch, n_q_heads, group;
    int32_t row_tiles;  // tiles of kRows query heads per KV head
    int32_t units;      // KV heads * row tiles
    int32_t table_tokens;
    int32_t window;
    float scale_log2;
    int32_t workers;
};

struct Span {
    int32_t first, len;  // attended tokens [first, len)
    int32_t steps;
};

__device__ __forceinline__ Span SpanOf(const AttendParams &p, int32_t b) {
    Span s;
    s.len = max(0, min(__ldg(p.lens + b), p.table_tokens));
    s.first = p.window > 0 ? max(0, s.len - p.window) : 0;
    s.steps = (s.len - s.first + kStep - 1) / kStep;
    return s;
}

// Steps per worker, the same in both kernels.
__device__ __forceinline__ int64_t StepsPerWorker(int64_t all, int32_t workers) {
    const int64_t per = (all + workers - 1) / workers;
    return per > 0 ? per : 1;
}

__device__ __forceinline__ void CopyAsync16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void CopyCommit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void CopyWait() {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ void LoadMatrix(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void LoadMatrixTransposed(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <typename T>
__device__ __forceinline__ void MatrixMultiply(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void MatrixMultiply<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                                              uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void MatrixMultiply<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                       uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// p0, p1 as 16-bit halves: hi is p rounded, lo what the rounding left over, rounded again.
template <typename T>
__device__ __forceinline__ void SplitPair(float p0, float p1, uint32_t &hi, uint32_t &lo) {
    const auto h = Half16<T>::FromFloat2(p0, p1);
    const float2 back = Half16<T>::ToFloat2(h);
    const auto l = Half16<T>::FromFloat2(p0 - back.x, p1 - back.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

// Shapes of the main kernel: kDim (64, 128, 256) is head_dim rounded up, kRows (8, 16) the query heads of a row tile.
template <int kDim, int kRows>
struct AttendShape {
    static constexpr int kRowBytes = kDim * 2;
    static constexpr int kTileBytes = kTile * kRowBytes;  // of K, and again of V
    static constexpr int kStages = kDim == 64 ? 4 : (kDim == 256 && kRows == 16 ? 2 : 3);
    static constexpr int kRingBytes = kAttendWarps * kStages * 2 * kTileBytes;
    static constexpr int kSmemBytes = kRingBytes + kAttendWarps * kRows * kDim * 4;  // + the warps' sums
    // an SM's 228 KB, of which every CTA takes 1 KB for itself and the kernel's small arrays
    static constexpr int kFit = 228 * 1024 / (kSmemBytes + 1024 + 640);
    static constexpr int kCtasPerSm = kFit < 2 ? kFit : 2;
};

template <typename T, int kDim, int kRows, bool kScores>
__global__ void __launch_bounds__(kAttendThreads, AttendShape<kDim, kRows>::kCtasPerSm) AttendPagesKernel(const AttendParams p) {
    using Shape = AttendShape<kDim, kRows>;
    constexpr int kStages = Shape::kStages;
    constexpr int kPieces = kDim / 8;               // 16-byte pieces of a row
    constexpr int kRowsPerCopy = 32 / kPieces;      // rows one copy instruction of a warp covers
    constexpr int kCopies = kTile / kRowsPerCopy;   // copy instructions per tile of K
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t scan_warp[kAttendWarps];
    __shared__ int64_t found_before;
    __shared__ int32_t found_b;
    __shared__ uint32_t valid_masks[kAttendWarps][kStages];
    __shared__ float2 join_ml[kAttendWarps][kRows];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float *join_o = reinterpret_cast<float *>(smem + Shape::kRingBytes);  // [warps][kRows][kDim]

    // ---- the steps of this CTA: [begin, begin + n_steps) of all steps, found by a scan over the sequences
    const int32_t chunk = (p.batch + kAttendThreads - 1) / kAttendThreads;
    const int32_t b_first = min(p.batch, static_cast<int32_t>(tid) * chunk), b_last = min(p.batch, b_first + chunk);
    int64_t mine = 0;
    for (int32_t b = b_first; b < b_last; ++b) mine += SpanOf(p, b).steps;
    int64_t inclusive = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int64_t up = __shfl_up_sync(0xffffffffu, inclusive, d);
        if (lane >= d) inclusive += up;
    }
    if (lane == 31) scan_warp[warp] = inclusive;
    __syncthreads();
    int64_t before = inclusive - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kAttendWarps; ++w) {
        if (w < static_cast<int>(warp)) before += scan_warp[w];
        all += scan_warp[w];
    }
    const int64_t total = all * p.units;
    const int64_t per = StepsPerWorker(total, p.workers);
    const int64_t begin = blockIdx.x * per;
    if (blockIdx.x == 0) {  // the second kernel reads where each sequence begins
        int64_t at = before;
        for (int32_t b = b_first; b < b_last; ++b) {
            p.steps_before[b] = at;
            at += SpanOf(p, b).steps;
            if (p.status != nullptr && __ldg(p.lens + b) > p.table_tokens) CountSkipped(p.status, b, 1u);
        }
        if (tid == 0) p.steps_before[p.batch] = all;
    }
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    if (begin >= total) return;
    if (before * p.units <= begin && begin < (before + mine) * p.units) {
        int64_t at = before;
        int32_t b = b_first;
        for (;; ++b) {
            const int32_t steps = SpanOf(p, b).steps;
            if (begin < (at + steps) * p.units) break;
            at += steps;
        }
        found_b = b;
        found_before = at * p.units;
    }
    __syncthreads();
    const int32_t n_steps = static_cast<int32_t>(min(per, total - begin));

    // A place in this CTA's run of steps.
    struct Cursor {
        int32_t b, unit, step;
        Span span;
        __device__ __forceinline__ void Next(const AttendParams &p, bool more) {
            if (++step < span.steps) return;
            step = 0;
            if (++unit < p.units || !more) return;
            unit = 0;
            do {
                span = SpanOf(p, ++b);
            } while (span.steps == 0);
        }
    };
    Cursor now;
    now.b = found_b;
    now.span = SpanOf(p, now.b);
    const int64_t inside = begin - found_before;
    now.unit = static_cast<int32_t>(inside / now.span.steps);
    now.step = static_cast<int32_t>(inside - static_cast<int64_t>(now.unit) * now.span.steps);
    Cursor ahead = now;

    const uint32_t ring = SmemAddr(smem) + warp * (kStages * 2 * Shape::kTileBytes);
    const uint32_t copy_piece = lane % kPieces, copy_row = lane / kPieces;
    const uint32_t copy_bytes = copy_piece * 8 < static_cast<uint32_t>(p.pools.head_dim) ? 16u : 0u;

    // Starts the copies of this warp's 16 tokens of step `ahead` into a stage.  Rows that take no part are filled with
    // zeros, so that whatever lies there cannot reach a product.
    auto fetch = [&](int stage) {
        const int32_t kv = ahead.unit / p.row_tiles;
        const int32_t t = ahead.span.first + ahead.step * kStep + static_cast<int32_t>(warp) * kTile +
                          static_cast<int32_t>(lane & (kTile - 1));
        int64_t off = -1;
        if (t < ahead.span.len) {
            const int32_t page_i = t / p.pools.page_tokens;
            const int32_t within = t - page_i * p.pools.page_tokens;
            const int64_t page = __ldg(p.table + ahead.b * p.table_stride + page_i);
            if (page >= 0 && page < p.pools.pool_pages) {
                off = page * p.pools.page_stride + within * p.pools.token_stride + kv * p.pools.head_stride;
            } else if (ahead.unit == 0 && lane < kTile && (within == 0 || t == ahead.span.first)) {
                CountSkipped(p.status, static_cast<uint32_t>(ahead.b), 1u);
            }
        }
        const uint32_t valid = __ballot_sync(0xffffffffu, off >= 0) & 0xffffu;
        if (lane == 0) valid_masks[warp][stage] = valid;
        const uint32_t k_to = ring + stage * 2 * Shape::kTileBytes;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const uint32_t row = i * kRowsPerCopy + copy_row;
            const int64_t row_off = __shfl_sync(0xffffffffu, off, row);
            const uint32_t bytes = row_off >= 0 ? copy_bytes : 0u;
            const int64_t from = bytes != 0 ? row_off + copy_piece * 16 : 0;
            const uint32_t to = k_to + row * Shape::kRowBytes + ((copy_piece ^ (row & 7)) * 16);
            CopyAsync16(to, p.pools.k + from, bytes);
            CopyAsync16(to + Shape::kTileBytes, p.pools.v + from, bytes);
        }
    };

    constexpr int kOut = kDim / 8;
    float o[kOut][4];
    uint32_t qa[kDim / 16][kRows == 8 ? 2 : 4];
    float top[2], sum[2];  // of rows lane / 4 and lane / 4 + 8

#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
        if (s < n_steps) {
            fetch(s);
            ahead.Next(p, s + 1 < n_steps);
        }
        CopyCommit();
    }
    bool fresh = true;
    int32_t share_first = now.step;
    int stage = 0;
    for (int32_t s = 0; s < n_steps; ++s) {
        CopyWait<kStages - 2>();
        __syncwarp();
        if (s + kStages - 1 < n_steps) {
            fetch(stage == 0 ? kStages - 1 : stage - 1);
            ahead.Next(p, s + kStages < n_steps);
        }
        CopyCommit();

        const int32_t kv = now.unit / p.row_tiles;
        const int32_t row_tile = now.unit - kv * p.row_tiles;
        const int32_t head0 = kv * p.group + row_tile * kRows;             // first query head of this tile
        const int32_t rows = min(kRows, p.group - row_tile * kRows);       // query heads of this tile
        if (fresh) {
            fresh = false;
            share_first = now.step;
            const T *q = reinterpret_cast<const T *>(p.query) + now.b * p.q_batch + head0 * p.q_head;
#pragma unroll
            for (int ks = 0; ks < kDim / 16; ++ks) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int col = ks * 16 + half * 8 + (lane & 3) * 2;
#pragma unroll
                    for (int r = 0; r < kRows / 8; ++r) {
                        const int row = static_cast<int>(lane >> 2) + r * 8;
                        uint32_t x = 0;
                        if (row < rows && col < p.pools.head_dim) x = __ldg(reinterpret_cast<const uint32_t *>(q + row * p.q_head + col));
                        qa[ks][half * (kRows / 8) + r] = x;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < kOut; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
            top[0] = top[1] = -INFINITY;
            sum[0] = sum[1] = 0.0f;
        }

        const uint32_t valid = valid_masks[warp][stage];
        // where this thread's scores of row lane / 4 go: two pairs of tokens, eight apart
        const int64_t score_at = kScores ? (static_cast<int64_t>(now.b) * p.n_q_heads + head0 + (lane >> 2)) * p.score_stride +
                                               static_cast<int64_t>(now.step) * kStep + warp * kTile + (lane & 3) * 2
                                         : 0;
        if (kScores && valid == 0) {
#pragma unroll
            for (int r = 0; r < kRows / 8; ++r) {
                if (static_cast<int>(lane >> 2) + r * 8 < rows) {
                    float *to = p.scores + score_at + r * 8 * p.score_stride;
                    *reinterpret_cast<float2 *>(to) = make_float2(-INFINITY, -INFINITY);
                    *reinterpret_cast<float2 *>(to + 8) = make_float2(-INFINITY, -INFINITY);
                }
            }
        }
        if (valid != 0) {
            // ---- scores of 16 tokens: two 16x8 products over the head dimension
            const uint32_t k_at = ring + stage * 2 * Shape::kTileBytes;
            float c[2][2][4] = {};
            {
                const uint32_t row = (lane & 7) + ((lane >> 4) << 3);
                const uint32_t row_at = k_at + row * Shape::kRowBytes;
                const uint32_t piece = (lane >> 3) & 1;
#pragma unroll
                for (int ks = 0; ks < kDim / 16; ++ks) {
                    uint32_t kb[4];
                    LoadMatrix(kb, row_at + (((ks * 2 + piece) ^ (row & 7)) * 16));
                    if constexpr (kRows == 8) {
                        MatrixMultiply<T>(c[ks & 1][0], qa[ks][0], 0u, qa[ks][1], 0u, kb[0], kb[1]);
                        MatrixMultiply<T>(c[ks & 1][1], qa[ks][0], 0u, qa[ks][1], 0u, kb[2], kb[3]);
                    } else {
                        MatrixMultiply<T>(c[ks & 1][0], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], kb[0], kb[1]);
                        MatrixMultiply<T>(c[ks & 1][1], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], kb[2], kb[3]);
                    }
                }
            }
            float x[2][4];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t col = nt * 8 + (lane & 3) * 2 + (e & 1);
                    const float v = (c[0][nt][e] + c[1][nt][e]) * p.scale_log2;
                    x[nt][e] = (valid >> col) & 1u ? v : -INFINITY;
                }
            }
            if (kScores) {
#pragma unroll
                for (int r = 0; r < kRows / 8; ++r) {
                    if (static_cast<int>(lane >> 2) + r * 8 < rows) {
                        float *to = p.scores + score_at + r * 8 * p.score_stride;
                        *reinterpret_cast<float2 *>(to) = make_float2(x[0][r * 2], x[0][r * 2 + 1]);
                        *reinterpret_cast<float2 *>(to + 8) = make_float2(x[1][r * 2], x[1][r * 2 + 1]);
                    }
                }
            }
            // ---- running maximum and sum
            uint32_t pa[4], pl[4];
            float scale_o[2] = {1.0f, 1.0f};
#pragma unroll
            for (int r = 0; r < kRows / 8; ++r) {
                float m = fmaxf(fmaxf(x[0][r * 2], x[0][r * 2 + 1]), fmaxf(x[1][r * 2], x[1][r * 2 + 1]));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                m = fmaxf(m, top[r]);
                const float use = m == -INFINITY ? 0.0f : m;  // nothing but negative infinity so far
                scale_o[r] = exp2f(top[r] - use);
                top[r] = m;
                float e[2][2];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    e[nt][0] = exp2f(x[nt][r * 2] - use);
                    e[nt][1] = exp2f(x[nt][r * 2 + 1] - use);
                }
                sum[r] = sum[r] * scale_o[r] + ((e[0][0] + e[0][1]) + (e[1][0] + e[1][1]));
                SplitPair<T>(e[0][0], e[0][1], pa[r], pl[r]);
                SplitPair<T>(e[1][0], e[1][1], pa[2 + r], pl[2 + r]);
            }
            if constexpr (kRows == 8) {  // the second half of every pair takes the free rows
                pa[1] = pl[0];
                pa[3] = pl[2];
                scale_o[1] = scale_o[0];
            }
            if (__any_sync(0xffffffffu, scale_o[0] != 1.0f || scale_o[1] != 1.0f)) {
#pragma unroll
                for (int j = 0; j < kOut; ++j) {
                    o[j][0] *= scale_o[0];
                    o[j][1] *= scale_o[0];
                    o[j][2] *= scale_o[1];
                    o[j][3] *= scale_o[1];
                }
            }
            // ---- the product with V
            {
                const uint32_t row = lane & 15;
                const uint32_t row_at = k_at + Shape::kTileBytes + row * Shape::kRowBytes;
                const uint32_t piece = lane >> 4;
#pragma unroll
                for (int j = 0; j < kDim / 16; ++j) {
                    uint32_t vb[4];
                    LoadMatrixTransposed(vb, row_at + (((j * 2 + piece) ^ (row & 7)) * 16));
                    MatrixMultiply<T>(o[2 * j], pa[0], pa[1], pa[2], pa[3], vb[0], vb[1]);
                    MatrixMultiply<T>(o[2 * j + 1], pa[0], pa[1], pa[2], pa[3], vb[2], vb[3]);
                    if constexpr (kRows == 16) {
                        MatrixMultiply<T>(o[2 * j], pl[0], pl[1], pl[2], pl[3], vb[0], vb[1]);
                        MatrixMultiply<T>(o[2 * j + 1], pl[0], pl[1], pl[2], pl[3], vb[2], vb[3]);
                    }
                }
            }
        }
        __syncwarp();  // the stage may be filled again
        stage = stage + 1 == kStages ? 0 : stage + 1;

        if (now.step + 1 == now.span.steps || s + 1 == n_steps) {
            // ---- the share is complete: the warps' sums are joined in shared memory
            fresh = true;
#pragma unroll
            for (int r = 0; r < kRows / 8; ++r) {
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
                if ((lane & 3) == 0) join_ml[warp][(lane >> 2) + r * 8] = make_float2(top[r], sum[r]);
            }
            float *mine_o = join_o + (warp * kRows + (lane >> 2)) * kDim + (lane & 3) * 2;
#pragma unroll
            for (int j = 0; j < kOut; ++j) {
                if constexpr (kRows == 8) {
                    *reinterpret_cast<float2 *>(mine_o + j * 8) = make_float2(o[j][0] + o[j][2], o[j][1] + o[j][3]);
                } else {
                    *reinterpret_cast<float2 *>(mine_o + j * 8) = make_float2(o[j][0], o[j][1]);
                    *reinterpret_cast<float2 *>(mine_o + 8 * kDim + j * 8) = make_float2(o[j][2], o[j][3]);
                }
            }
            __syncthreads();
            const bool whole = share_first == 0 && now.step + 1 == now.span.steps;
            // a share that begins where the run does is the run's first; any other begins at its unit's first step
            const bool begins_run = s + 1 - (now.step + 1 - share_first) == 0;
            const int64_t slot = (static_cast<int64_t>(blockIdx.x) * 2 + (begins_run ? 0 : 1)) * kRows;
            for (uint32_t i = tid; i < static_cast<uint32_t>(rows) * (kDim / 2); i += kAttendThreads) {
                const uint32_t row = i / (kDim / 2);
                const uint32_t d = (i - row * (kDim / 2)) * 2;
                float m = -INFINITY;
#pragma unroll
                for (int w = 0; w < kAttendWarps; ++w) m = fmaxf(m, join_ml[w][row].x);
                float l = 0.0f;
                float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kAttendWarps; ++w) {
                    const float2 ml = join_ml[w][row];
                    const float f = exp2f(ml.x - (m == -INFINITY ? 0.0f : m));
                    const float2 part = *reinterpret_cast<const float2 *>(join_o + (w * kRows + row) * kDim + d);
                    l += ml.y * f;
                    acc.x += part.x * f;
                    acc.y += part.y * f;
                }
                if (whole) {
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    const int64_t head_at = static_cast<int64_t>(now.b) * p.n_q_heads + head0 + row;
                    if (d < static_cast<uint32_t>(p.pools.head_dim)) {
                        T *to = reinterpret_cast<T *>(p.out) + head_at * p.pools.head_dim + d;
                        *reinterpret_cast<typename Half16<T>::Pair *>(to) = Half16<T>::FromFloat2(acc.x * inv, acc.y * inv);
                    }
                    if (d == 0) {
                        if (kScores) p.whole_ml[head_at] = make_float2(m, l);
                        if (p.lse != nullptr) p.lse[head_at] = l == 0.0f ? -INFINITY : m * kLn2 + logf(l);
                    }
                } else {
                    *reinterpret_cast<float2 *>(p.part_o + (slot + row) * kDim + d) = acc;
                    if (d == 0) p.part_ml[slot + row] = make_float2(m, l);
                }
            }
            __syncthreads();
        }
        now.Next(p, s + 1 < n_steps);
    }
    CopyWait<0>();
}

// Where the shares of a unit lie: workers [first, last]; share w is in slot 2 w + (its unit begins within the run).
struct Shares {
    int64_t t0, per;
    int32_t first, last;
    __device__ __forceinline__ int64_t Slot(int32_t w) const { return 2 * static_cast<int64_t>(w) + (t0 > w * per ? 1 : 0); }
};

__device__ __forceinline__ Shares SharesOf(const AttendParams &p, int64_t before, int64_t steps, int64_t per, int32_t unit) {
    Shares s;
    s.t0 = before * p.units + unit * steps;
    s.per = per;
    s.first = static_cast<int32_t>(s.t0 / per);
    s.last = static_cast<int32_t>((s.t0 + steps - 1) / per);
    return s;
}

// Joins the shares of heads that were cut, writes zeros for sequences without tokens, and, in the blocks behind those,
// adds the attention every token received to its weight.  One block per query head, then kWeightThreads tokens of one
// weight head per block.
template <typename T, int kDim, int kRows>
__global__ void __launch_bounds__(kJoinThreads) JoinSharesKernel(const AttendParams p, uint32_t join_blocks, uint32_t weight_chunks) {
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const int64_t total = p.steps_before[p.batch] * p.units;
    const int64_t per = StepsPerWorker(total, p.workers);
    const uint32_t tid = threadIdx.x;
    if (blockIdx.x < join_blocks) {
        constexpr int kLanes = kDim / 2;                      // threads across a head, two elements each
        constexpr int kParts = kJoinThreads / kLanes;         // shares summed side by side
        __shared__ float2 sums[kParts][kLanes];
        __shared__ float part_l[kParts];
        const int32_t b = blockIdx.x / p.n_q_heads, head = blockIdx.x - b * p.n_q_heads;
        const int64_t head_at = static_cast<int64_t>(b) * p.n_q_heads + head;
        T *out = reinterpret_cast<T *>(p.out) + head_at * p.pools.head_dim;
        const int64_t before = p.steps_before[b], steps = p.steps_before[b + 1] - before;
        if (steps == 0) {
            for (uint32_t d = tid; d < static_cast<uint32_t>(p.pools.head_dim); d += kJoinThreads) out[d] = Half16<T>::FromFloat(0.0f);
            if (tid == 0 && p.lse != nullptr) p.lse[head_at] = -INFINITY;
            return;
        }
        const int32_t kv = head / p.group, in_group = head - kv * p.group;
        const int32_t row = in_group % kRows;
        const Shares sh = SharesOf(p, before, steps, per, kv * p.row_tiles + in_group / kRows);
        if (sh.first == sh.last) return;  // finished by the CTA that had it whole
        __shared__ float warp_max[kJoinThreads / 32];
        float m = -INFINITY;
        for (int32_t w = sh.first + tid; w <= sh.last; w += kJoinThreads) m = fmaxf(m, p.part_ml[sh.Slot(w) * kRows + row].x);
#pragma unroll
        for (int d = 16; d > 0; d /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        if ((tid & 31) == 0) warp_max[tid >> 5] = m;
        __syncthreads();
        m = warp_max[0];
        for (int w = 1; w < kJoinThreads / 32; ++w) m = fmaxf(m, warp_max[w]);
        const float use = m == -INFINITY ? 0.0f : m;
        const uint32_t part = tid / kLanes, at = tid % kLanes;
        float2 acc = make_float2(0.0f, 0.0f);
        float l = 0.0f;
#pragma unroll 4
        for (int32_t w = sh.first + part; w <= sh.last; w += kParts) {
            const int64_t slot = sh.Slot(w) * kRows + row;
            const float2 ml = p.part_ml[slot];
            const float2 v = *reinterpret_cast<const float2 *>(p.part_o + slot * kDim + at * 2);
            const float f = exp2f(ml.x - use);
            l += ml.y * f;
            acc.x += v.x * f;
            acc.y += v.y * f;
        }
        sums[part][at] = acc;
        if (at == 0) part_l[part] = l;
        __syncthreads();
        if (part == 0) {
            l = 0.0f;
            acc = make_float2(0.0f, 0.0f);
            for (int i = 0; i < kParts; ++i) {
                l += part_l[i];
                acc.x += sums[i][at].x;
                acc.y += sums[i][at].y;
            }
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            if (at * 2 < static_cast<uint32_t>(p.pools.head_dim)) {
                *reinterpret_cast<typename Half16<T>::Pair *>(out + at * 2) = Half16<T>::FromFloat2(acc.x * inv, acc.y * inv);
            }
            if (at == 0 && p.lse != nullptr) p.lse[head_at] = l == 0.0f ? -INFINITY : m * kLn2 + logf(l);
        }
        return;
    }
    // ---- weights
    extern __shared__ float2 head_ml[];  // maximum and reciprocal sum of the query heads that count here
    const uint32_t block = blockIdx.x - join_blocks;
    const uint32_t pair = block / weight_chunks;
    const uint32_t chunk = block - pair * weight_chunks;
    const int32_t b = pair / p.n_weight_heads, wh = pair - b * p.n_weight_heads;
    const Span span = SpanOf(p, b);
    const int32_t from = span.first + static_cast<int32_t>(chunk) * kWeightThreads;
    if (from >= span.len) return;
    const int32_t n_heads = p.n_weight_heads == 1 ? p.n_q_heads : p.group;
    const int32_t head0 = p.n_weight_heads == 1 ? 0 : wh * p.group;
    const int64_t before = p.steps_before[b];
    for (int32_t i = tid >> 5; i < n_heads; i += kWeightThreads / 32) {
        const int32_t head = head0 + i;
        const int32_t kv = head / p.group, in_group = head - kv * p.group;
        const Shares sh = SharesOf(p, before, span.steps, per, kv * p.row_tiles + in_group / kRows);
        float m, l = 0.0f;
        if (sh.first == sh.last) {
            const float2 ml = p.whole_ml[static_cast<int64_t>(b) * p.n_q_heads + head];
            m = ml.x;
            l = ml.y;
        } else {
            m = -INFINITY;
            for (int32_t w = sh.first + (tid & 31); w <= sh.last; w += 32) {
                const float2 ml = p.part_ml[sh.Slot(w) * kRows + in_group % kRows];
                const float grown = fmaxf(m, ml.x);
                const float use = grown == -INFINITY ? 0.0f : grown;
                l = l * exp2f(m - use) + ml.y * exp2f(ml.x - use);
                m = grown;
            }
#pragma unroll
            for (int d = 16; d > 0; d /= 2) {
                const float m2 = __shfl_xor_sync(0xffffffffu, m, d), l2 = __shfl_xor_sync(0xffffffffu, l, d);
                const float grown = fmaxf(m, m2);
                const float use = grown == -INFINITY ? 0.0f : grown;
                l = l * exp2f(m - use) + l2 * exp2f(m2 - use);
                m = grown;
            }
        }
        if ((tid & 31) == 0) head_ml[i] = make_float2(m == -INFINITY ? 0.0f : m, l == 0.0f ? 0.0f : 1.0f / l);
    }
    __syncthreads();
    const int32_t t = from + static_cast<int32_t>(tid);
    if (t >= span.len) return;
    // a token on a page outside the pool was masked like any other: its score is negative infinity
    const float *scores = p.scores + (static_cast<int64_t>(b) * p.n_q_heads + head0) * p.score_stride + (t - span.first);
    float received = 0.0f;
#pragma unroll 4
    for (int32_t i = 0; i < n_heads; ++i) {
        const float2 ml = head_ml[i];
        received += exp2f(scores[i * p.score_stride] - ml.x) * ml.y;
    }
    p.weights_out[b * p.wo_batch + wh * p.wo_head + t] = p.weights[b * p.w_batch + wh * p.w_head + t] + received;
}

int64_t Aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }

struct AttendWorkspace {
    int64_t steps_before, part_o, part_ml, whole_ml, scores, total;
    int64_t score_stride;
};

AttendWorkspace LayOut(int32_t batch, int32_t n_q_heads, int32_t group, int32_t head_dim, int64_t table_tokens, bool with_weights) {
    const int rows = group <= 8 ? 8 : 16;
    const int dim = head_dim <= 64 ? 64 : (head_dim <= 128 ? 128 : 256);
    AttendWorkspace w;
    w.steps_before = 0;
    w.part_o = Aligned((static_cast<int64_t>(batch) + 1) * 8);
    w.part_ml = w.part_o + Aligned(int64_t{kMaxWorkers} * 2 * rows * dim * 4);
    w.whole_ml = w.part_ml + Aligned(int64_t{kMaxWorkers} * 2 * rows * 8);
    w.scores = w.whole_ml + (with_weights ? Aligned(static_cast<int64_t>(batch) * n_q_heads * 8) : 0);
    w.score_stride = (table_tokens + kStep - 1) / kStep * kStep;
    w.total = w.scores + (with_weights ? Aligned(static_cast<int64_t>(batch) * n_q_heads * w.score_stride * 4) : 0);
    return w;
}

template <typename T, int kDim, int kRows, bool kScores>
void LaunchAttend(AttendParams p, cudaStream_t stream) {
    using Shape = AttendShape<kDim, kRows>;
    auto *main_kernel = AttendPagesKernel<T, kDim, kRows, kScores>;
    auto *join_kernel = JoinSharesKernel<T, kDim, kRows>;
    EnsureDynamicSmem(main_kernel, Shape::kSmemBytes);
    p.workers = std::min(kMaxWorkers, GetDeviceInfo().sm_count * Shape::kCtasPerSm);
    main_kernel<<<p.workers, kAttendThreads, Shape::kSmemBytes, stream>>>(p);

    const uint32_t join_blocks = static_cast<uint32_t>(p.batch) * p.n_q_heads;
    const int64_t most = p.window > 0 ? std::min(p.window, p.table_tokens) : p.table_tokens;
    const uint32_t weight_chunks = kScores ? static_cast<uint32_t>((most + kWeightThreads - 1) / kWeightThreads) : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(join_blocks + weight_chunks * static_cast<uint32_t>(p.batch) * p.n_weight_heads);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = kScores ? static_cast<size_t>(p.n_weight_heads == 1 ? p.n_q_heads : p.group) * 8 : 0;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, join_kernel, p, join_blocks, std::max(weight_chunks, 1u));
}

template <typename T, int kDim>
void DispatchAttend(const AttendParams &p, cudaStream_t stream) {
    if (p.group <= 8) {
        p.scores != nullptr ? LaunchAttend<T, kDim, 8, true>(p, stream) : LaunchAttend<T, kDim, 8, false>(p, stream);
    } else {
        p.scores != nullptr ? LaunchAttend<T, kDim, 16, true>(p, stream) : LaunchAttend<T, kDim, 16, false>(p, stream);
    }
}

template <typename T>
void DispatchAttend(const AttendParams &p, cudaStream_t stream) {
    if (p.pools.head_dim <= 64) {
        DispatchAttend<T, 64>(p, stream);
    } else if (p.pools.head_dim <= 128) {
        DispatchAttend<T, 128>(p, stream);
    } else {
        DispatchAttend<T, 256>(p, stream);
    }
}

}  // namespace
}  // namespace kvcm

extern "C" {

int64_t kvcm_b200_attend_workspace_bytes(int32_t batch, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                         int64_t table_tokens, int32_t with_weights) {
    if (batch < 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0 || head_dim <= 0 ||
        head_dim > kvcm::kMaxAttendHeadDim || table_tokens < 0 || table_tokens > kvcm::kMaxTableTokens) {
        return -1;
    }
    return kvcm::LayOut(batch, n_q_heads, n_q_heads / n_kv_heads, head_dim, table_tokens, with_weights != 0).total;
}

int32_t kvcm_b200_attend_pages(const kvcm_b200_kv_pools_t *pools, const void *d_query, int64_t q_batch_stride,
                               int64_t q_head_stride, int32_t batch, int32_t n_q_heads, const int32_t *d_block_table,
                               int64_t table_stride, int32_t table_width, const int32_t *d_context_lens, float scale,
                               int32_t window, void *d_out, float *d_lse, const float *d_weights,
                               int64_t w_batch_stride, int64_t w_head_stride, float *d_weights_out,
                               int64_t wo_batch_stride, int64_t wo_head_stride, int32_t n_weight_heads,
                               void *d_workspace, int64_t workspace_bytes, uint32_t *d_status, kvcm_stream_t stream) {
    using namespace kvcm;
    const int32_t rc = CheckPools(pools, kMaxAttendHeadDim);
    if (rc != KVCM_OK) return rc;
    const bool with_weights = d_weights != nullptr;
    const int64_t table_tokens = static_cast<int64_t>(table_width) * pools->page_tokens;
    if (batch < 0 || n_q_heads <= 0 || n_q_heads % pools->n_kv_heads != 0 || table_width < 0 || window < 0 ||
        with_weights != (d_weights_out != nullptr) ||
        (with_weights && n_weight_heads != 1 && n_weight_heads != pools->n_kv_heads) ||
        (with_weights && d_weights == d_weights_out && (w_batch_stride != wo_batch_stride || w_head_stride != wo_head_stride))) {
        return KVCM_ER_INVALID_PARAMS;
    }
    const int64_t weight_blocks = with_weights ? (table_tokens / kWeightThreads + 1) * batch * n_weight_heads : 0;
    if (batch > 65536 || n_q_heads > 4096 || table_tokens > kMaxTableTokens || weight_blocks > (int64_t{1} << 30)) {
        return KVCM_EC_OUT_OF_LIMIT;
    }
    if ((batch > 0 && (d_query == nullptr || (d_block_table == nullptr && table_width > 0) || d_context_lens == nullptr ||
                       d_out == nullptr || d_workspace == nullptr)) ||
        !RowsAre16ByteAligned(*pools) || (reinterpret_cast<uintptr_t>(d_workspace) & 15u) != 0 ||
        (reinterpret_cast<uintptr_t>(d_query) & 3u) != 0 || (reinterpret_cast<uintptr_t>(d_out) & 3u) != 0 ||
        ((q_batch_stride | q_head_stride) & 1) != 0) {
        return KVCM_ER_INVALID_ADDRESS;
    }
    const int32_t group = n_q_heads / pools->n_kv_heads;
    const AttendWorkspace w = LayOut(batch, n_q_heads, group, pools->head_dim, table_tokens, with_weights);
    if (batch > 0 && workspace_bytes < w.total) return KVCM_ER_INVALID_PARAMS;
    if (!HaveDevice()) return KVCM_ER_NO_DEVICE;
    if (batch == 0) return KVCM_OK;
    uint8_t *ws = static_cast<uint8_t *>(d_workspace);
    AttendParams p = {};
    p.pools = AsPagedPools(*pools);
    p.query = static_cast<const uint8_t *>(d_query);
    p.q_batch = q_batch_stride;
    p.q_head = q_head_stride;
    p.table = d_block_table;
    p.table_stride = table_stride;
    p.lens = d_context_lens;
    p.out = static_cast<uint8_t *>(d_out);
    p.lse = d_lse;
    p.status = d_status;
    p.weights = d_weights;
    p.weights_out = d_weights_out;
    p.w_batch = w_batch_stride;
    p.w_head = w_head_stride;
    p.wo_batch = wo_batch_stride;
    p.wo_head = wo_head_stride;
    p.n_weight_heads = with_weights ? n_weight_heads : 0;
    p.steps_before = reinterpret_cast<int64_t *>(ws + w.steps_before);
    p.part_o = reinterpret_cast<float *>(ws + w.part_o);
    p.part_ml = reinterpret_cast<float2 *>(ws + w.part_ml);
    p.whole_ml = reinterpret_cast<float2 *>(ws + w.whole_ml);
    p.scores = with_weights ? reinterpret_cast<float *>(ws + w.scores) : nullptr;
    p.score_stride = w.score_stride;
    p.batch = batch;
    p.n_q_heads = n_q_heads;
    p.group = group;
    const int rows = group <= 8 ? 8 : 16;
    p.row_tiles = (group + rows - 1) / rows;
    p.units = pools->n_kv_heads * p.row_tiles;
    p.table_tokens = static_cast<int32_t>(table_tokens);
    p.window = window;
    p.scale_log2 = scale * kLog2e;
    if (pools->dtype == KVCM_DTYPE_BF16) {
        DispatchAttend<__nv_bfloat16>(p, AsStream(stream));
    } else {
        DispatchAttend<__half>(p, AsStream(stream));
    }
    return LaunchStatus();
}

}  // extern "C"
