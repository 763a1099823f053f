// Attention of one new token per sequence over its paged keys and values, with the attention weights accumulated per
// cached token on request.
//
//   o_h = sum_t p_t V[t],  p = softmax_t(scale * q_h . K[t]),  t over the sequence's last `window` tokens or all.
//
// Bound by HBM: every K and V row is read once (512 bytes per token and KV head of 128) and used by the query heads that
// share the KV head, 2 to 32 multiplications per byte.  One pass with a running maximum and sum.  A group of more than
// sixteen query heads is cut into row tiles of sixteen, each of which reads the rows again (groups of 17 and of 32 take
// 2.2 and 2.3 times the time of one pass over the bytes, of 64 4.6 times).
//
// Four warps to a CTA, each with a ring of its own: tiles of 16 tokens of one KV head come from HBM by 16-byte asynchronous
// copies, issued by the warp one to three tiles ahead, the table entry of the one after those already on its way; then
// ldmatrix, 16x8x16 matrix instructions whose 16 rows are the group's query heads, softmax in registers, and the product
// with V.  No warp waits for another until a head is complete.  (TMA tile loads were measured in three forms and left:
// with producer warps, 65 cycles to issue each box set the pace, 1050 to 1700 for a step of four tiles; with every warp
// loading its own tile, the four barrier operations a tile needs, about 100 cycles each, did.)  A group is far too
// small for the 128 rows of the tcgen05 instructions, and the tensor pipe is idle most of the time as it is.
//
// Probabilities enter the second product as two 16-bit halves, p = hi + lo, whose sum carries 16 (bf16) or 22 (fp16) bits,
// so the output is rounded once.  fp16 has nothing between 0 and 2^-24, so there the product takes p times 2^15, and the sums
// are brought back where a share is written: all 22 bits are kept down to 2^-28 of the largest probability and errors
// stay below 2^-40 of it, where without the factor a token 18 nats below an attention sink was lost whole.  With a group of
// at most eight the halves cost nothing: hi takes rows 0-7 of the matrix instruction, lo the rows 8-15 that the group
// leaves free.
//
// The work is cut by tokens, not by sequences: the steps (four tiles of one sequence) of the whole batch are numbered
// through, and each of the persistent CTAs takes an equal run of them, found from the lengths on the device.  Finishing a
// head costs about as much as two steps, so two are added to each that no one has to do: without them the CTAs that took
// many short sequences finished last (37 sequences of 1 to 5000 tokens: 33 us instead of 27).  A head that lies within
// one run is finished there; the runs of a head that is cut leave their unnormalised sums and statistics in the
// workspace, and the second kernel joins them, in order, so results do not depend on timing.  A third adds up the
// weights, which need every head's final statistics.
//
// 64 sequences of 512 to 8192 tokens, 32 query and 8 KV heads of 128, bf16: 175 us, 6.5 TB/s read, as fast as a plain copy
// reads and writes together.  One sequence of 131,072 tokens on one KV head, fp16: 22.5 us, of which 10.3 are its bytes; 16
// of 2000 to 6001 tokens with weights: 55 us, of which 41.
#include "paged_kv.cuh"

namespace kvcm {
namespace {

constexpr int kAttendWarps = 4;
constexpr int kAttendThreads = kAttendWarps * 32;
constexpr int kTile = 16;                                  // tokens of a tile
constexpr int kUnitCost = 2;                               // steps that finishing a unit takes about as long as
constexpr int kUncutSteps = 4;                             // of a unit that stays whole whatever the batch
constexpr int kMaxWorkers = 512;
constexpr int kMaxAttendHeadDim = 256;
constexpr int kJoinThreads = 128;
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
    float *part_o;          // [step_heads * kRows][dim / 16][2 * workers][16]: a join reads many shares of a few elements
    float2 *part_ml;        // [step_heads * kRows][2 * workers] maximum and sum of a share, the maximum in units of log2
    float2 *whole_ml;       // [batch][n_q_heads] maximum and sum of whole heads; with weights only
    float *scores;          // [batch][n_q_heads][score_stride], in units of log2; null without weights
    int64_t score_stride;
    int32_t batch, n_q_heads, group;
    int32_t row_tiles;   // tiles of kRows query heads per KV head
    int32_t step_heads;  // KV heads of a step, 1, 2 or 4: its four tiles are step_heads heads by step_tokens tokens
    int32_t step_tokens;
    int32_t uncut;       // every unit is a run
    int32_t kv_groups;   // KV heads / step_heads
    int32_t units;       // kv_groups * row_tiles
    int32_t k_steps;     // 16-element pieces of a row that are not padding
    int64_t v_minus_k;   // bytes from a row of K to the same of V
    int64_t copy_stride; // bytes between the rows that one copy instruction after another takes
    int32_t table_tokens;
    int32_t window;
    int32_t whole_tiles;  // page_tokens is a multiple of kTile: a tile lies in one page
    int32_t page_shift;   // log2 of page_tokens, or -1
    float scale_log2;
    int32_t workers;
};

struct Span {
    int32_t first, len;  // attended tokens [first, len)
    int32_t base;        // first rounded down to a tile
    int32_t real;        // steps with tokens
    int32_t steps;       // and those that stand for the cost of finishing a unit, when there are any tokens
};

__device__ __forceinline__ Span SpanOf(const AttendParams &p, int32_t b) {
    Span s;
    s.len = max(0, min(__ldg(p.lens + b), p.table_tokens));
    s.first = p.window > 0 ? max(0, s.len - p.window) : 0;
    s.base = s.first & ~(kTile - 1);
    s.real = (s.len - s.base + p.step_tokens - 1) / p.step_tokens;
    s.steps = s.real > 0 ? s.real + kUnitCost : 0;
    return s;
}

// a / b, in 32 bits where they do: a 64-bit division takes several times as long.
__device__ __forceinline__ int64_t Divide(int64_t a, int64_t b) {
    return (a | b) <= 0xffffffffll ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}

// Where a share's entry of a line of entries lies, one per slot.
__device__ __forceinline__ int64_t PartAt(int32_t line, int32_t slot, int32_t workers) {
    return static_cast<int64_t>(line) * (2 * workers) + slot;
}

// Steps per run, the same in the kernels that compute shares and join them.
__device__ __forceinline__ int64_t StepsPerRun(int64_t all, int32_t workers) {
    const int64_t per = Divide(all + workers - 1, workers);
    return per > 1 ? per : 1;
}

// The steps of all sequences numbered through, each sequence's `times` over.
struct StepScan {
    int64_t mine, before, all;  // of this thread's sequences, of those before them, of the batch; once over
    int32_t b_first, b_last;
};

// Every thread of the block takes part; `warp_sums` has a word per warp.
template <int kThreads>
__device__ __forceinline__ StepScan ScanSteps(const AttendParams &p, int64_t *warp_sums) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t chunk = (p.batch + kThreads - 1) / kThreads;
    StepScan s;
    s.b_first = min(p.batch, static_cast<int32_t>(tid) * chunk);
    s.b_last = min(p.batch, s.b_first + chunk);
    s.mine = 0;
    for (int32_t b = s.b_first; b < s.b_last; ++b) s.mine += SpanOf(p, b).steps;
    int64_t inclusive = s.mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int64_t up = __shfl_up_sync(0xffffffffu, inclusive, d);
        if (lane >= d) inclusive += up;
    }
    if (lane == 31) warp_sums[warp] = inclusive;
    __syncthreads();
    s.before = inclusive - s.mine;
    s.all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < static_cast<int>(warp)) s.before += warp_sums[w];
        s.all += warp_sums[w];
    }
    return s;
}

struct Place64 {
    int64_t before;  // steps of the sequences before b, `times` over
    int32_t b;
};

// Where step x, which has to exist, lies.  Ends with a barrier.
__device__ __forceinline__ void FindStep(const AttendParams &p, const StepScan &s, int64_t times, int64_t x, Place64 *found) {
    if (s.before * times <= x && x < (s.before + s.mine) * times) {
        int64_t at = s.before;
        int32_t b = s.b_first;
        for (;; ++b) {
            const int32_t steps = SpanOf(p, b).steps;
            if (x < (at + steps) * times) break;
            at += steps;
        }
        found->b = b;
        found->before = at * times;
    }
    __syncthreads();
}

__device__ __forceinline__ float Exp2(float x) {  // results below 2^-126 are zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float Log2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// K and V rows are read once: they may leave L2 before what the kernels after this one read.
__device__ __forceinline__ uint64_t ReadOncePolicy() {
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;\n" : "=l"(policy));
    return policy;
}
// 16 bytes, of which the first `bytes` come from src and the rest are zeros.
__device__ __forceinline__ void CopyAsync16(uint32_t dst, const void *src, uint32_t bytes, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;\n" ::"r"(dst), "l"(src), "r"(bytes), "l"(policy)
                 : "memory");
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

// What probabilities are multiplied by before they are split, and its inverse.  bf16 has the exponents of a float.
template <typename T>
struct SplitScale {
    static constexpr float kUp = 1.0f, kDown = 1.0f;
};
template <>
struct SplitScale<__half> {
    static constexpr float kUp = 32768.0f, kDown = 1.0f / 32768.0f;  // the largest stays finite
};

// p0, p1 as 16-bit halves: hi is p (scaled) rounded, lo what the rounding left over, rounded again.
template <typename T>
__device__ __forceinline__ void SplitPair(float p0, float p1, uint32_t &hi, uint32_t &lo) {
    p0 *= SplitScale<T>::kUp;
    p1 *= SplitScale<T>::kUp;
    const auto h = Half16<T>::FromFloat2(p0, p1);
    const float2 back = Half16<T>::ToFloat2(h);
    const auto l = Half16<T>::FromFloat2(p0 - back.x, p1 - back.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

// Shapes of the main kernel: kDim (64, 128, 256) is head_dim rounded up.
template <int kDim, bool kScores>
struct AttendShape {
    static constexpr int kRowBytes = kDim * 2;
    static constexpr int kTileBytes = kTile * kRowBytes;  // of K, and again of V
    static constexpr int kStageBytes = kAttendWarps * 2 * kTileBytes;
    // Warps hide one another's latencies better than deeper rings do: three CTAs of two stages against two of three
    // measured 181 against 185 us on the ragged batch, 138 against 161 with a head_dim of 80 - where registers allow.
    static constexpr int kCtasPerSm = kDim == 256 ? 1 : (kDim == 64 || !kScores ? 3 : 2);
    static constexpr int kStages = kDim == 64 ? 4 : (kDim == 128 && !kScores ? 2 : 3);
    static constexpr int kAhead = kDim == 64 || kCtasPerSm == 2 ? 8 : 4;              // K operands fetched together
    static constexpr int kVAhead = kDim == 64 ? 4 : (kCtasPerSm == 2 ? kDim / 16 : 2);  // and V operands
    static constexpr int kRingBytes = kStages * kStageBytes;
};

template <typename T, int kDim, int kRows, bool kScores>
__global__ void __launch_bounds__(kAttendThreads, AttendShape<kDim, kScores>::kCtasPerSm)
    AttendPagesKernel(const __grid_constant__ AttendParams p) {
    using Shape = AttendShape<kDim, kScores>;
    constexpr int kStages = Shape::kStages;
    constexpr int kPieces = kDim / 8;              // 16-byte pieces of a row
    constexpr int kCopyRows = 32 / kPieces;        // rows one copy instruction of a warp covers
    constexpr int kCopies = kTile / kCopyRows;     // copy instructions per tile of K
    extern __shared__ __align__(128) uint8_t ring_bytes[];
    __shared__ float2 join_ml[kAttendWarps][kRows];
    __shared__ uint32_t valid_masks[kAttendWarps][kStages];
    __shared__ int64_t scan_warp[kAttendWarps];
    __shared__ Place64 found;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t ring = SmemAddr(ring_bytes);

    if (blockIdx.x == 0 && p.status != nullptr) {
        for (int32_t b = tid; b < p.batch; b += kAttendThreads) {
            if (__ldg(p.lens + b) > p.table_tokens) CountSkipped(p.status, b, 1u);
        }
    }
    // Sequences without tokens belong to no run: zeros, here.
    for (int32_t b = blockIdx.x; b < p.batch; b += gridDim.x) {
        if (SpanOf(p, b).steps != 0) continue;
        T *out = reinterpret_cast<T *>(p.out) + static_cast<int64_t>(b) * p.n_q_heads * p.pools.head_dim;
        for (int32_t i = tid; i < p.n_q_heads * p.pools.head_dim; i += kAttendThreads) out[i] = Half16<T>::FromFloat(0.0f);
        if (p.lse != nullptr) {
            for (int32_t i = tid; i < p.n_q_heads; i += kAttendThreads) p.lse[static_cast<int64_t>(b) * p.n_q_heads + i] = -INFINITY;
        }
    }
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    // ---- the run of this CTA: `left` steps from a step of a unit on.  A unit, when units are short enough to stay whole;
    // else an equal part of all steps, found by a scan over the sequences.
    int32_t b, unit, step = 0;
    int32_t left;
    Span span;
    if (p.uncut) {
        b = blockIdx.x / p.units;
        unit = blockIdx.x - b * p.units;
        span = SpanOf(p, b);
        left = span.steps;
        if (left == 0) return;
    } else {
        const StepScan scan = ScanSteps<kAttendThreads>(p, scan_warp);
        const int64_t total = scan.all * p.units;
        const int64_t per = StepsPerRun(total, p.workers);
        const int64_t begin = blockIdx.x * per;
        if (begin >= total) return;
        FindStep(p, scan, p.units, begin, &found);
        b = found.b;
        span = SpanOf(p, b);
        const int64_t inside = begin - found.before;
        unit = static_cast<int32_t>(Divide(inside, span.steps));
        step = static_cast<int32_t>(inside - static_cast<int64_t>(unit) * span.steps);
        left = static_cast<int32_t>(min(per, total - begin));
    }
    const int32_t token_tiles = p.step_tokens / kTile;  // of a step: 4, 2, 1
    const int32_t my_head = static_cast<int32_t>(warp) / token_tiles;
    const int32_t my_t = (static_cast<int32_t>(warp) - my_head * token_tiles) * kTile;  // from the step's first token

    // A place in the run: a step with tokens, and the steps that are left from there, none or fewer at the run's end.  The
    // place that loads also keeps which tokens its sequence attends; the one that computes is told by masks.
    struct Place {
        int32_t b, kvg, row_tile, step, real, left;
        __device__ __forceinline__ bool UnitEnds() const { return step + 1 == real; }
        __device__ __forceinline__ int32_t LeftAfter() const { return left - (UnitEnds() ? 1 + kUnitCost : 1); }
        // True when it has come to another sequence.
        __device__ __forceinline__ bool Next(const AttendParams &p) {
            left = LeftAfter();
            if (++step < real || left <= 0) return false;
            step = 0;
            if (++row_tile < p.row_tiles) return false;
            row_tile = 0;
            if (++kvg < p.kv_groups) return false;
            kvg = 0;
            do {
                real = SpanOf(p, ++b).real;
            } while (real == 0);
            return true;
        }
    };
    Place now;
    now.b = b;
    now.kvg = unit / p.row_tiles;
    now.row_tile = unit - now.kvg * p.row_tiles;
    now.step = step;
    now.real = span.real;
    now.left = left;
    bool begins_run = true;  // the share at hand begins where the run does
    if (step >= span.real) {  // among the steps that no one has to do
        begins_run = false;
        now.left += step - (span.real - 1);
        now.step = span.real - 1;
        if (now.Next(p)) span = SpanOf(p, now.b);
        if (now.left <= 0) return;
    }
    Place ask = now;  // of the next tile to load
    int32_t ask_first = span.first, ask_len = span.len, ask_base = span.base;

    // The table entry of the next tile to load: of the whole tile, or of token lane % 16 where tiles cross pages.
    int32_t ask_page = 0, ask_token = 0;
    auto look_up = [&]() {
        const int32_t t0 = ask_base + ask.step * p.step_tokens + my_t;
        const int32_t t = p.whole_tiles ? t0 : t0 + static_cast<int32_t>(lane & (kTile - 1));
        ask_page = -1;
        if (t < ask_len && (p.whole_tiles ? t + kTile : t + 1) > ask_first) {
            const int32_t page_i = p.page_shift >= 0 ? t >> p.page_shift : t / p.pools.page_tokens;
            ask_token = t - page_i * p.pools.page_tokens;
            ask_page = __ldg(p.table + ask.b * p.table_stride + page_i);
        }
    };

    // A page outside the pool is counted once: at its first token, or at the first that is attended.
    auto report_page = [&](int32_t t0, int32_t begins) {
        const int32_t t = p.whole_tiles ? t0 + begins : t0 + static_cast<int32_t>(lane & (kTile - 1));
        const bool mine = p.whole_tiles ? lane == 0 : lane < kTile && t >= ask_first && t < ask_len;
        if (mine && my_head == 0 && ask.kvg == 0 && ask.row_tile == 0 && (ask_token == 0 || t == ask_first)) {
            CountSkipped(p.status, static_cast<uint32_t>(ask.b), 1u);
        }
    };

    const uint32_t tiles_at = ring + warp * 2 * Shape::kTileBytes;
    const uint32_t copy_piece = lane % kPieces, copy_row = lane / kPieces;
    const uint32_t copy_to = copy_row * Shape::kRowBytes + ((copy_piece ^ copy_row) * 16);  // of the first copy
    const int64_t copy_from = static_cast<int64_t>(copy_row) * p.pools.token_stride +
                              (copy_piece * 8 < static_cast<uint32_t>(p.pools.head_dim) ? copy_piece * 16 : 0);
    // Starts the copies of this warp's tile of the next step; rows that take no part become zeros, so that whatever lies
    // there cannot reach a product.
    auto load_tile = [&](int to_stage) {
        const int32_t t0 = ask_base + ask.step * p.step_tokens + my_t;
        const int32_t begins = max(ask_first - t0, 0), ends = min(ask_len - t0, kTile);
        uint32_t valid = ends > begins ? ((1u << ends) - 1u) & ~((1u << begins) - 1u) : 0u;
        const bool page_ok = ask_page >= 0 && ask_page < p.pools.pool_pages;
        if (!page_ok && valid != 0) report_page(t0, begins);
        const int64_t head_off = static_cast<int64_t>(ask.kvg * p.step_heads + my_head) * p.pools.head_stride;
        const uint32_t to = tiles_at + to_stage * Shape::kStageBytes + copy_to;
        const uint64_t policy = ReadOncePolicy();
        const uint32_t copy_bytes = copy_piece * 8 < static_cast<uint32_t>(p.pools.head_dim) ? 16u : 0u;
        if (p.whole_tiles) {
            if (!page_ok) valid = 0;
            if (valid != 0) {
                const uint8_t *from = p.pools.k + ask_page * p.pools.page_stride + ask_token * p.pools.token_stride + head_off + copy_from;
#pragma unroll
                for (int i = 0; i < kCopies; ++i) {
                    const uint32_t row = i * kCopyRows + copy_row;
                    const uint32_t bytes = (valid >> row) & 1u ? copy_bytes : 0u;
                    const uint32_t at = (to ^ (((i * kCopyRows) & 7) * 16)) + i * kCopyRows * Shape::kRowBytes;
                    CopyAsync16(at, from, bytes, policy);
                    CopyAsync16(at + Shape::kTileBytes, from + p.v_minus_k, bytes, policy);
                    from += p.copy_stride;
                }
            }
        } else {
            valid &= __ballot_sync(0xffffffffu, page_ok);
            const int64_t off = ask_page * p.pools.page_stride + ask_token * p.pools.token_stride + head_off;
            if (valid != 0) {
#pragma unroll
                for (int i = 0; i < kCopies; ++i) {
                    const uint32_t row = i * kCopyRows + copy_row;
                    const int64_t row_off = __shfl_sync(0xffffffffu, off, row);
                    const uint32_t bytes = (valid >> row) & 1u ? copy_bytes : 0u;
                    const uint8_t *from = p.pools.k + (bytes != 0 ? row_off + copy_piece * 16 : 0);
                    const uint32_t at = (to ^ (((i * kCopyRows) & 7) * 16)) + i * kCopyRows * Shape::kRowBytes;
                    CopyAsync16(at, from, bytes, policy);
                    CopyAsync16(at + Shape::kTileBytes, from + p.v_minus_k, bytes, policy);
                }
            }
        }
        if (lane == 0) valid_masks[warp][to_stage] = valid;
    };

    constexpr int kOut = kDim / 8;
    float o[kOut][4];
    uint32_t qa[kDim / 16][kRows == 8 ? 2 : 4];
    float top[2], sum[2];  // of rows lane / 4 and lane / 4 + 8
    auto load_queries = [&](int32_t of_b, int32_t head0, int32_t rows) {
        const T *q = reinterpret_cast<const T *>(p.query) + of_b * p.q_batch + (head0 + my_head * p.group) * p.q_head;
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
    };
    auto clear = [&]() {
#pragma unroll
        for (int j = 0; j < kOut; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        top[0] = top[1] = -INFINITY;
        sum[0] = sum[1] = 0.0f;
    };

    // lane's row and 16-byte column in the swizzled tiles, for the K and the V product
    const uint32_t k_row = (lane & 7) + ((lane >> 4) << 3), v_row = lane & 15;
    const uint32_t k_lane = k_row * Shape::kRowBytes + ((((lane >> 3) & 1) ^ (k_row & 7)) * 16);
    const uint32_t v_lane = Shape::kTileBytes + v_row * Shape::kRowBytes + (((lane >> 4) ^ (v_row & 7)) * 16);
    int32_t head0 = 0, rows = 0;
    bool from_first = now.step == 0;  // the share at hand has its unit's first step
    bool fresh = true;
    int stage = 0, to_stage = 0;
    // Iteration s works on the run's step s, loads step s + kStages - 1 and looks up the one after that; the first kStages
    // iterations only fill the ring.  (One copy of the code: a run is short, and instructions that are met for the
    // first time come from L2.)
    for (int32_t s = -kStages;; ++s) {
        CopyWait<kStages - 2>();
        __syncwarp();
        if (s > -kStages) {
            if (ask.left > 0) {
                load_tile(to_stage);
                if (ask.Next(p)) {
                    const Span next = SpanOf(p, ask.b);
                    ask_first = next.first;
                    ask_len = next.len;
                    ask_base = next.base;
                }
            }
            CopyCommit();
            to_stage = to_stage + 1 == kStages ? 0 : to_stage + 1;
        }
        if (ask.left > 0) look_up();
        if (s < 0) continue;
        if (fresh) {
            fresh = false;
            head0 = now.kvg * p.step_heads * p.group + now.row_tile * kRows;  // the step's first query head
            rows = min(kRows, p.group - now.row_tile * kRows);                // and those of a row tile
            load_queries(now.b, head0, rows);
            clear();
        }
        const uint32_t valid = valid_masks[warp][stage];
        const uint32_t tile = tiles_at + stage * Shape::kStageBytes;
        int64_t score_at = 0;  // where this thread's scores of row lane / 4 go: two pairs of tokens, eight apart
        if (kScores) {
            score_at = (static_cast<int64_t>(now.b) * p.n_q_heads + head0 + my_head * p.group + (lane >> 2)) * p.score_stride +
                       static_cast<int64_t>(now.step) * p.step_tokens + my_t + (lane & 3) * 2;
            if (valid == 0) {
#pragma unroll
                for (int r = 0; r < kRows / 8; ++r) {
                    if (static_cast<int>(lane >> 2) + r * 8 < rows) {
                        float *to = p.scores + score_at + r * 8 * p.score_stride;
                        *reinterpret_cast<float2 *>(to) = make_float2(-INFINITY, -INFINITY);
                        *reinterpret_cast<float2 *>(to + 8) = make_float2(-INFINITY, -INFINITY);
                    }
                }
            }
        }
        if (valid != 0) {
            // ---- scores of 16 tokens: two 16x8 products over the head dimension, operands fetched ahead in groups
            constexpr int kAhead = Shape::kAhead;
            float c[2][2][4] = {};
#pragma unroll
            for (int k0 = 0; k0 < kDim / 16; k0 += kAhead) {
                uint32_t kb[kAhead][4];
#pragma unroll
                for (int i = 0; i < kAhead && k0 + i < kDim / 16; ++i) {
                    const int ks = k0 + i;
                    LoadMatrix(kb[i], ((tile + k_lane) ^ ((ks & 3) * 32)) + (ks >> 2) * 128);
                }
#pragma unroll
                for (int i = 0; i < kAhead && k0 + i < kDim / 16; ++i) {
                    const int ks = k0 + i;
                    if (kDim == 64 || ks < kDim / 32 || ks < p.k_steps) {
                        if constexpr (kRows == 8) {
                            MatrixMultiply<T>(c[ks & 1][0], qa[ks][0], 0u, qa[ks][1], 0u, kb[i][0], kb[i][1]);
                            MatrixMultiply<T>(c[ks & 1][1], qa[ks][0], 0u, qa[ks][1], 0u, kb[i][2], kb[i][3]);
                        } else {
                            MatrixMultiply<T>(c[ks & 1][0], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], kb[i][0], kb[i][1]);
                            MatrixMultiply<T>(c[ks & 1][1], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], kb[i][2], kb[i][3]);
                        }
                    }
                }
            }
            // the first of V's operands, on their way during the softmax
            constexpr int kVAhead = Shape::kVAhead;
            uint32_t vb[kVAhead][4];
            auto load_v = [&](int j) {
                LoadMatrixTransposed(vb[j % kVAhead], ((tile + v_lane) ^ ((j & 3) * 32)) + (j >> 2) * 128);
            };
#pragma unroll
            for (int j = 0; j < kVAhead; ++j) load_v(j);
            float x[2][4];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[nt][e] = (c[0][nt][e] + c[1][nt][e]) * p.scale_log2;
            }
            if (valid != 0xffffu) {
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t col = nt * 8 + (lane & 3) * 2 + (e & 1);
                        if (((valid >> col) & 1u) == 0) x[nt][e] = -INFINITY;
                    }
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
                scale_o[r] = Exp2(top[r] - use);
                top[r] = m;
                float e[2][2];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    e[nt][0] = Exp2(x[nt][r * 2] - use);
                    e[nt][1] = Exp2(x[nt][r * 2 + 1] - use);
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
#pragma unroll
            for (int j = 0; j < kDim / 16; ++j) {
                if (kDim == 64 || j < kDim / 32 || j < p.k_steps) {
                    const uint32_t(&v)[4] = vb[j % kVAhead];
                    MatrixMultiply<T>(o[2 * j], pa[0], pa[1], pa[2], pa[3], v[0], v[1]);
                    MatrixMultiply<T>(o[2 * j + 1], pa[0], pa[1], pa[2], pa[3], v[2], v[3]);
                    if constexpr (kRows == 16) {
                        MatrixMultiply<T>(o[2 * j], pl[0], pl[1], pl[2], pl[3], v[0], v[1]);
                        MatrixMultiply<T>(o[2 * j + 1], pl[0], pl[1], pl[2], pl[3], v[2], v[3]);
                    }
                }
                if (j + kVAhead < kDim / 16) load_v(j + kVAhead);
            }
        }

        __syncwarp();  // the stage may be filled again

        const bool unit_ends = now.UnitEnds();
        const bool more = now.LeftAfter() > 0;
        if (unit_ends || !more) {
            // ---- the share is complete: the sums of the warps with the same KV head are joined, in the tiles that this
            // step has used up
            const bool whole = from_first && unit_ends;
#pragma unroll
            for (int r = 0; r < kRows / 8; ++r) {
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
                if ((lane & 3) == 0) join_ml[warp][(lane >> 2) + r * 8] = make_float2(top[r], sum[r]);
            }
            uint8_t *sums = ring_bytes + stage * Shape::kStageBytes;  // warp w's at w * 2 * kTileBytes, [kRows][kDim]
            float *mine_o = reinterpret_cast<float *>(sums + warp * 2 * Shape::kTileBytes) + (lane >> 2) * kDim + (lane & 3) * 2;
#pragma unroll
            for (int j = 0; j < kOut; ++j) {
                constexpr float kDown = SplitScale<T>::kDown;
                if constexpr (kRows == 8) {
                    *reinterpret_cast<float2 *>(mine_o + j * 8) = make_float2((o[j][0] + o[j][2]) * kDown, (o[j][1] + o[j][3]) * kDown);
                } else {
                    *reinterpret_cast<float2 *>(mine_o + j * 8) = make_float2(o[j][0] * kDown, o[j][1] * kDown);
                    *reinterpret_cast<float2 *>(mine_o + 8 * kDim + j * 8) = make_float2(o[j][2] * kDown, o[j][3] * kDown);
                }
            }
            __syncthreads();
            const int32_t slot = blockIdx.x + (begins_run ? 0 : p.workers);
#pragma unroll 1  // few rounds, and registers are short
            for (int32_t i = tid; i < p.step_heads * rows * (kDim / 2); i += kAttendThreads) {
                const int32_t head_row = i / (kDim / 2), kv_i = head_row / rows, row = head_row - kv_i * rows;
                const int32_t d = (i - head_row * (kDim / 2)) * 2;
                float m = -INFINITY;
#pragma unroll 1
                for (int32_t w = kv_i * token_tiles; w < (kv_i + 1) * token_tiles; ++w) m = fmaxf(m, join_ml[w][row].x);
                const float use = m == -INFINITY ? 0.0f : m;
                float l = 0.0f;
                float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll 1
                for (int32_t w = kv_i * token_tiles; w < (kv_i + 1) * token_tiles; ++w) {
                    const float2 ml = join_ml[w][row];
                    const float f = Exp2(ml.x - use);
                    const float2 part = *reinterpret_cast<const float2 *>(
                        reinterpret_cast<const float *>(sums + w * 2 * Shape::kTileBytes) + row * kDim + d);
                    l += ml.y * f;
                    acc.x += part.x * f;
                    acc.y += part.y * f;
                }
                if (whole) {
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    const int64_t head_at = static_cast<int64_t>(now.b) * p.n_q_heads + head0 + kv_i * p.group + row;
                    if (d < p.pools.head_dim) {
                        T *to = reinterpret_cast<T *>(p.out) + head_at * p.pools.head_dim + d;
                        *reinterpret_cast<typename Half16<T>::Pair *>(to) = Half16<T>::FromFloat2(acc.x * inv, acc.y * inv);
                    }
                    if (d == 0) {
                        if (kScores) p.whole_ml[head_at] = make_float2(m, l);
                        if (p.lse != nullptr) p.lse[head_at] = l == 0.0f ? -INFINITY : (m + Log2(l)) * kLn2;
                    }
                } else {
                    const int32_t part_row = kv_i * kRows + row;
                    *reinterpret_cast<float2 *>(p.part_o + PartAt(part_row * (kDim / 16) + d / 16, slot, p.workers) * 16 + d % 16) = acc;
                    if (d == 0) p.part_ml[PartAt(part_row, slot, p.workers)] = make_float2(m, l);
                }
            }
            __syncthreads();  // the sums may be overwritten
            fresh = from_first = true;
            begins_run = false;
        }
        if (!more) break;
        now.Next(p);
        stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    CopyWait<0>();
}

// Where the shares of a unit lie: runs [first, last]; the share of run w is in slot w, or workers + w where the unit begins
// within the run: consecutive runs in consecutive slots.
struct Shares {
    int64_t t0, per;
    int32_t first, last;
    __device__ __forceinline__ int32_t Slot(int32_t w, int32_t workers) const { return w + (t0 > w * per ? workers : 0); }
};

__device__ __forceinline__ Shares SharesAt(int64_t t0, int64_t steps, int64_t per) {
    Shares s;
    s.t0 = t0;
    s.per = per;
    s.first = static_cast<int32_t>(Divide(t0, per));
    s.last = static_cast<int32_t>(Divide(t0 + steps - 1, per));
    return s;
}

// A sum in progress: maximum (log2 units), sum of exponentials, four output elements.
struct Partial {
    float m, l;
    float4 o;
    __device__ __forceinline__ void Add(float m2, float l2, float4 o2) {
        const float grown = fmaxf(m, m2);
        const float use = grown == -INFINITY ? 0.0f : grown;
        const float f = Exp2(m - use), f2 = Exp2(m2 - use);
        l = l * f + l2 * f2;
        o.x = o.x * f + o2.x * f2;
        o.y = o.y * f + o2.y * f2;
        o.z = o.z * f + o2.z * f2;
        o.w = o.w * f + o2.w * f2;
        m = grown;
    }
};

// Joins the shares of heads that were cut.  It starts when the first kernel's last CTA ends, so what counts is the chain of
// dependent loads after that: small blocks, all resident at once, find their work from the lengths while the first
// kernel still runs, and load all they need of its results together.  Block w looks at the point where run w begins.
// When that lies within a unit, the unit's shares are joined by the blocks of all such points together: with c cuts
// each block takes a c-th of the unit's output elements, four to a thread group, over all shares, so that one long head
// is joined by as many blocks as computed it.
template <typename T, int kDim, int kRows, bool kScores>
__global__ void __launch_bounds__(kJoinThreads, 8) JoinSharesKernel(const __grid_constant__ AttendParams p) {
    __shared__ Partial partials[kJoinThreads / 32];
    __shared__ int64_t scan_warp[kJoinThreads / 32];
    __shared__ Place64 found;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const StepScan scan = ScanSteps<kJoinThreads>(p, scan_warp);
    const int64_t per = StepsPerRun(scan.all * p.units, p.workers);
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int32_t w = blockIdx.x;
    // Every block waits for the first kernel, also one without work: the kernel after this one relies on it.
    if (w * per >= scan.all * p.units) {
        asm volatile("griddepcontrol.wait;\n" ::: "memory");
        return;
    }
    FindStep(p, scan, p.units, w * per, &found);
    const int32_t b = found.b;
    const Span span = SpanOf(p, b);
    const int64_t inside = w * per - found.before;
    const int32_t unit = static_cast<int32_t>(Divide(inside, span.steps));
    const int64_t into = inside - static_cast<int64_t>(unit) * span.steps;
    if (into == 0 || into >= span.real) {  // nothing is cut here
        asm volatile("griddepcontrol.wait;\n" ::: "memory");
        return;
    }
    const Shares sh = SharesAt(w * per - into, span.real, per);
    const int32_t cuts = sh.last - sh.first, cut = w - sh.first - 1;
    const int32_t kvg = unit / p.row_tiles, row_tile = unit - kvg * p.row_tiles;
    const int32_t rows = min(kRows, p.group - row_tile * kRows);
    const int64_t head0 = static_cast<int64_t>(b) * p.n_q_heads + kvg * p.step_heads * p.group + row_tile * kRows;
    const int32_t fours = p.step_heads * rows * (kDim / 4);    // groups of four output elements
    const int32_t mine = (fours + cuts - 1) / cuts;            // this block's
    int32_t lanes = 1;                                         // thread groups per pass, a power of two
    while (lanes < mine && lanes < kJoinThreads) lanes *= 2;
    const int32_t parts = kJoinThreads / lanes;                // threads that share a group's shares
    const int32_t at = tid / parts, part = tid % parts;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    for (int32_t base = 0; base < mine; base += lanes) {
        const int32_t four = cut * mine + base + at;
        const bool live = base + at < mine && four < fours;
        const int32_t head_row = live ? four / (kDim / 4) : 0, d = live ? (four - head_row * (kDim / 4)) * 4 : 0;
        const int32_t kv_i = head_row / rows, row = head_row - kv_i * rows;
        const int64_t head_at = head0 + kv_i * p.group + row;
        Partial acc = {-INFINITY, 0.0f, make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
        constexpr int kTogether = 4;
        for (int32_t i0 = sh.first + part; live && i0 <= sh.last; i0 += kTogether * parts) {
            Partial got[kTogether];
#pragma unroll
            for (int j = 0; j < kTogether; ++j) {
                const int32_t i = i0 + j * parts;
                got[j] = {-INFINITY, 0.0f, make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
                if (i <= sh.last) {
                    const int32_t slot = sh.Slot(i, p.workers), part_row = kv_i * kRows + row;
                    const float2 ml = __ldcg(p.part_ml + PartAt(part_row, slot, p.workers));
                    const float *from = p.part_o + PartAt(part_row * (kDim / 16) + d / 16, slot, p.workers) * 16 + d % 16;
                    got[j] = {ml.x, ml.y, __ldcg(reinterpret_cast<const float4 *>(from))};
                }
            }
#pragma unroll
            for (int j = 0; j < kTogether; ++j) acc.Add(got[j].m, got[j].l, got[j].o);
        }
        for (int32_t i = 1; i < min(parts, 32); i *= 2) {
            Partial other;
            other.m = __shfl_xor_sync(0xffffffffu, acc.m, i);
            other.l = __shfl_xor_sync(0xffffffffu, acc.l, i);
            other.o.x = __shfl_xor_sync(0xffffffffu, acc.o.x, i);
            other.o.y = __shfl_xor_sync(0xffffffffu, acc.o.y, i);
            other.o.z = __shfl_xor_sync(0xffffffffu, acc.o.z, i);
            other.o.w = __shfl_xor_sync(0xffffffffu, acc.o.w, i);
            acc.Add(other.m, other.l, other.o);
        }
        if (parts > 32) {
            __syncthreads();
            if (lane == 0) partials[warp] = acc;
            __syncthreads();
            if (part == 0) {
                for (int32_t i = 1; i < parts / 32; ++i) {
                    const Partial other = partials[warp + i];
                    acc.Add(other.m, other.l, other.o);
                }
            }
        }
        if (live && part == 0) {
            const float inv = acc.l == 0.0f ? 0.0f : 1.0f / acc.l;
            if (d < p.pools.head_dim) {  // head_dim is a multiple of eight
                auto *to = reinterpret_cast<typename Half16<T>::Pair *>(reinterpret_cast<T *>(p.out) + head_at * p.pools.head_dim + d);
                to[0] = Half16<T>::FromFloat2(acc.o.x * inv, acc.o.y * inv);
                to[1] = Half16<T>::FromFloat2(acc.o.z * inv, acc.o.w * inv);
            }
            if (kScores && d == 0) p.whole_ml[head_at] = make_float2(acc.m, acc.l);
            if (d == 0 && p.lse != nullptr) p.lse[head_at] = acc.l == 0.0f ? -INFINITY : (acc.m + Log2(acc.l)) * kLn2;
        }
    }
}

// Adds the attention every token received to its weight.  The steps of all sequences and weight heads are cut into equal
// runs, one to a block; like the second kernel this one finds its work before it waits for the results.
// kAtOnce tokens and kHeads heads of a thread have their loads in flight together.
template <int kThreads, int kAtOnce, int kHeads>
__global__ void __launch_bounds__(kThreads, 8) AddWeightsKernel(const __grid_constant__ AttendParams p) {
    __shared__ int64_t scan_warp[kThreads / 32];
    __shared__ Place64 found;
    const uint32_t tid = threadIdx.x;
    const StepScan scan = ScanSteps<kThreads>(p, scan_warp);
    const int64_t total = scan.all * p.n_weight_heads;
    const int64_t share = Divide(total + gridDim.x - 1, gridDim.x);
    int64_t at = blockIdx.x * share;
    const int64_t end = min(total, at + share);
    if (at >= end) {  // what follows in the stream relies on every block having waited
        asm volatile("griddepcontrol.wait;\n" ::: "memory");
        return;
    }
    FindStep(p, scan, p.n_weight_heads, at, &found);
    int32_t b = found.b;
    Span span = SpanOf(p, b);
    int32_t wh = static_cast<int32_t>(Divide(at - found.before, span.steps));
    int32_t step0 = static_cast<int32_t>(at - found.before - static_cast<int64_t>(wh) * span.steps);
    const int32_t n_heads = p.n_weight_heads == 1 ? p.n_q_heads : p.group;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    while (at < end) {
        const int32_t steps = static_cast<int32_t>(min(static_cast<int64_t>(span.steps - step0), end - at));
        const int64_t head_at = static_cast<int64_t>(b) * p.n_q_heads + (p.n_weight_heads == 1 ? 0 : wh * p.group);
        const float2 *stats = p.whole_ml + head_at;
        // a token on a page outside the pool was masked like any other: its score is negative infinity
        const float *scores = p.scores + head_at * p.score_stride;
        const float *w_in = p.weights + b * p.w_batch + wh * p.w_head + span.base;
        float *w_out = p.weights_out + b * p.wo_batch + wh * p.wo_head + span.base;
        const int32_t skip = span.first - span.base;  // tokens of the first tile that lie before the window
        const int32_t last = min((step0 + steps) * p.step_tokens, span.len - span.base);
        for (int32_t t0 = step0 * p.step_tokens + static_cast<int32_t>(tid); t0 < last; t0 += kAtOnce * kThreads) {
            float received[kAtOnce] = {}, old[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const int32_t t = t0 + j * kThreads;
                old[j] = t < last && t >= skip ? w_in[t] : 0.0f;
            }
#pragma unroll kHeads
            for (int32_t i = 0; i < n_heads; ++i) {
                const float2 ml = __ldcg(stats + i);
                const float *row = scores + i * p.score_stride + t0;
                float score[kAtOnce];
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) score[j] = t0 + j * kThreads < last ? __ldcg(row + j * kThreads) : -INFINITY;
                const float top = ml.x == -INFINITY ? 0.0f : ml.x, inv = ml.y == 0.0f ? 0.0f : 1.0f / ml.y;
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) received[j] += Exp2(score[j] - top) * inv;
            }
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const int32_t t = t0 + j * kThreads;
                if (t < last && t >= skip) w_out[t] = old[j] + received[j];
            }
        }
        at += steps;
        step0 = 0;
        if (++wh == p.n_weight_heads && at < end) {
            wh = 0;
            do {
                span = SpanOf(p, ++b);
            } while (span.steps == 0);
        }
    }
}

int64_t Aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }

struct AttendWorkspace {
    int64_t part_o, part_ml, whole_ml, scores, total;
    int64_t score_stride;
};

AttendWorkspace LayOut(int32_t batch, int32_t n_q_heads, int32_t group, int32_t head_dim, int64_t table_tokens, bool with_weights) {
    const int rows = group <= 8 ? 8 : 16;
    const int dim = head_dim <= 64 ? 64 : (head_dim <= 128 ? 128 : 256);
    AttendWorkspace w;
    w.part_o = 0;
    w.part_ml = w.part_o + Aligned(int64_t{kMaxWorkers} * 2 * kAttendWarps * rows * dim * 4);
    w.whole_ml = w.part_ml + Aligned(int64_t{kMaxWorkers} * 2 * kAttendWarps * rows * 8);
    w.scores = w.whole_ml + (with_weights ? Aligned(static_cast<int64_t>(batch) * n_q_heads * 8) : 0);
    // whole steps from a base that may lie up to 15 tokens before the first
    w.score_stride = (table_tokens + kTile * kAttendWarps - 1) / (kTile * kAttendWarps) * (kTile * kAttendWarps) + kTile * kAttendWarps;
    w.total = w.scores + (with_weights ? Aligned(static_cast<int64_t>(batch) * n_q_heads * w.score_stride * 4) : 0);
    return w;
}

template <typename T, int kDim, int kRows, bool kScores>
int32_t LaunchAttend(AttendParams p, cudaStream_t stream) {
    using Shape = AttendShape<kDim, kScores>;
    static_assert((Shape::kRingBytes + 2048) * Shape::kCtasPerSm <= 228 * 1024, "CTAs per SM");
    auto *main_kernel = AttendPagesKernel<T, kDim, kRows, kScores>;
    const int32_t sm_count = GetDeviceInfo().sm_count;
    p.copy_stride = (32 / (kDim / 8)) * p.pools.token_stride;
    p.workers = std::min(kMaxWorkers, sm_count * Shape::kCtasPerSm);
    Requests requests;
    requests.Make([&] { return EnsureDynamicSmem(main_kernel, Shape::kRingBytes); });
    requests.Make([&] {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<uint32_t>(p.uncut ? p.batch * p.units : p.workers));
        cfg.blockDim = dim3(kAttendThreads);
        cfg.dynamicSmemBytes = Shape::kRingBytes;
        cfg.stream = stream;
        return cudaLaunchKernelEx(&cfg, main_kernel, p);
    });

    // The kernels that follow wait on the device for the one before them; their launch overlaps it.
    auto launch_after = [&](auto kernel, int32_t blocks) {
        requests.Make([&] {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(static_cast<uint32_t>(blocks));
            cfg.blockDim = dim3(kJoinThreads);
            cfg.stream = stream;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[0].val.programmaticStreamSerializationAllowed = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            return cudaLaunchKernelEx(&cfg, kernel, p);
        });
    };
    if (!p.uncut) launch_after(JoinSharesKernel<T, kDim, kRows, kScores>, p.workers);
    if (kScores) {
        // loads in flight over tokens, or over heads where all query heads count for one weight
        const bool many_heads = p.n_weight_heads == 1 && p.n_q_heads >= 8;
        launch_after(many_heads ? AddWeightsKernel<kJoinThreads, 1, 8> : AddWeightsKernel<kJoinThreads, 4, 4>, 8 * sm_count);
    }
    return requests.Status();
}

template <typename T, int kDim>
int32_t DispatchAttend(const AttendParams &p, cudaStream_t stream) {
    if (p.group <= 8) {
        return p.scores != nullptr ? LaunchAttend<T, kDim, 8, true>(p, stream) : LaunchAttend<T, kDim, 8, false>(p, stream);
    }
    return p.scores != nullptr ? LaunchAttend<T, kDim, 16, true>(p, stream) : LaunchAttend<T, kDim, 16, false>(p, stream);
}

template <typename T>
int32_t DispatchAttend(const AttendParams &p, cudaStream_t stream) {
    if (p.pools.head_dim <= 64) return DispatchAttend<T, 64>(p, stream);
    if (p.pools.head_dim <= 128) return DispatchAttend<T, 128>(p, stream);
    return DispatchAttend<T, 256>(p, stream);
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
    // Steps are counted in 64 bits over the batch and in 32 within a CTA's run.
    const double most_steps = static_cast<double>(batch) * n_q_heads * (static_cast<double>(table_tokens) / kTile + 1 + kUnitCost);
    if (batch > 65536 || n_q_heads > 4096 || table_tokens > kMaxTableTokens || most_steps > 1e11) return KVCM_EC_OUT_OF_LIMIT;
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
    // HBM and L2 move 64 to 256 bytes at a time.  Where a head's row is no multiple of 256 bytes and the next head's follows
    // it, a step takes rows of two or four heads instead of more tokens of one, so that what is fetched with a row is
    // used: 177 -> 138 us for heads of 80 elements, 217 -> 198 us for 64, 181 -> 152 us for 96; rows of 256 bytes take 174 us
    // one head at a time and 175 to 177 us otherwise, as do pages that keep a head's tokens together.
    p.step_heads = 1;
    const int32_t row_bytes = pools->head_dim * 2;
    if (pools->head_stride == pools->head_dim) {
        while (p.step_heads < kAttendWarps && pools->n_kv_heads % (p.step_heads * 2) == 0 && p.step_heads * row_bytes % 256 != 0) {
            p.step_heads *= 2;
        }
    }
    p.step_tokens = kTile * kAttendWarps / p.step_heads;
    p.kv_groups = pools->n_kv_heads / p.step_heads;
    p.units = p.kv_groups * p.row_tiles;
    p.k_steps = (pools->head_dim + 15) / 16;
    p.v_minus_k = p.pools.v - p.pools.k;
    // A few steps are done sooner in one CTA than in several whose shares a second kernel joins: a table of
    // kUncutSteps steps or less leaves every unit whole (one sequence of 100 tokens: 5.6 us instead of 7.3 us).
    p.uncut = table_tokens <= kUncutSteps * p.step_tokens;
    p.table_tokens = static_cast<int32_t>(table_tokens);
    p.window = window;
    p.scale_log2 = scale * kLog2e;
    p.whole_tiles = pools->page_tokens % kTile == 0;
    p.page_shift = -1;
    for (int32_t i = 0; i < 31; ++i) {
        if (pools->page_tokens == 1 << i) p.page_shift = i;
    }
    return pools->dtype == KVCM_DTYPE_BF16 ? DispatchAttend<__nv_bfloat16>(p, AsStream(stream))
                                           : DispatchAttend<__half>(p, AsStream(stream));
}

}  // extern "C"
