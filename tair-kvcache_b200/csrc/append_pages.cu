// Rotary positions and append: new tokens' queries and keys rotated, keys and values written into their pool slots.
//
// For token t and pair j < rotary_dim / 2 with angle a = positions[t] * inv_freq[j]:
//   (x, y) -> f * (x cos a - y sin a, y cos a + x sin a)
// the pair being elements (j, j + rotary_dim / 2) of a head, or (2j, 2j + 1).
//
// Bound by HBM: every query element is read and written once, every key and value element read once and written once,
// 24.6 KB per token at 32 query and 8 KV heads of 128.  The angles of a token are shared by all its heads, so a CTA takes
// whole tokens, forms their sine-cosine pairs once into shared memory, and its threads walk the tokens' heads in
// 16-byte pieces, a piece or a pair of pieces in flight each.  The first are loaded before the angles are formed, so the
// latencies of the two overlap.  With one token to a CTA the angles' chain of 64-bit operations, not HBM, set the
// pace (138 us for 16,384 tokens); with four it is met once for four.  An angle is formed and reduced to one
// turn in 64 bits: at position 10^6 a 32-bit product would be off by 0.06 rad.
//
// 16,384 tokens of 32 + 8 heads of 128: 70 us, 5.75 TB/s, 88 % of a plain copy.  Two items in flight per thread and four
// CTAs per SM took 105 us, six or eight CTAs 79 and 109 us (registers), two tokens to a CTA 81 us (all four with plain
// stores, which took 76 us otherwise).
#include "paged_kv.cuh"

namespace kvcm {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendItems = 1;  // items a thread has in flight
constexpr int kMaxAppendHeadDim = 1024;
constexpr int kMaxAppendTokens = 4;  // of a CTA

struct HeadRows {
    const void *src;
    void *dst;
    int64_t src_token, src_head, dst_token, dst_head;  // in elements; dst_* of keys and values come from the pools
};

struct AppendParams {
    PagedPools pools;
    HeadRows query, key, value;
    const void *positions;
    const void *slots;
    const float *inv_freq;
    uint32_t *status;
    int32_t positions64, slots64;
    int32_t n_q_heads;
    int32_t rotary_half;
    float factor;
    uint32_t rot_items;      // per head: items of 2 x V elements that are rotated
    FastDivide head_items;   // rot_items + items of V elements that pass through
    FastDivide value_items;  // per value head
    FastDivide token_items;
    uint32_t qk_items;       // per token: of queries and keys
    int32_t n_tokens;
    int32_t tokens;  // of a CTA
};

__device__ __forceinline__ int64_t LoadIndex(const void *p, int32_t is64, int64_t i) {
    return is64 ? __ldg(static_cast<const long long *>(p) + i) : static_cast<int64_t>(__ldg(static_cast<const int *>(p) + i));
}

// Where the angle of pair j lies among a token's: an item of V pairs reads them two at a time, and the lanes of a warp, which
// have consecutive items, find each two side by side (one after the other they would meet in the same banks).
template <int V>
__device__ __forceinline__ uint32_t AngleAt(uint32_t j, uint32_t rot_items) {
    if (V == 1) return j;
    return (j % V / 2 * rot_items + j / V) * 2 + j % 2;
}

template <typename T, int V>
struct alignas(2 * V) Vec {
    T x[V];
};

// A piece as the plain word that the streaming accesses take.
template <int V>
struct RawOf;
template <>
struct RawOf<8> {
    using Type = uint4;
};
template <>
struct RawOf<4> {
    using Type = uint2;
};
template <>
struct RawOf<2> {
    using Type = uint32_t;
};
template <>
struct RawOf<1> {
    using Type = unsigned short;
};
// Nothing here is read or written twice: stores that leave L2 first took a prompt from 76 to 70 us.
template <typename T, int V>
__device__ __forceinline__ void StorePiece(void *to, const Vec<T, V> &piece) {
    using Raw = typename RawOf<V>::Type;
    __stcs(reinterpret_cast<Raw *>(to), *reinterpret_cast<const Raw *>(&piece));
}

template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kAppendThreads, 5) AppendPagesKernel(const __grid_constant__ AppendParams p) {
    extern __shared__ __align__(16) float2 cs[];  // [tokens][rotary_half]
    __shared__ int64_t rows[kMaxAppendTokens];  // byte offset of each token's row in the pools, -1 for none
    using Piece = Vec<T, V>;
    const int64_t token0 = static_cast<int64_t>(blockIdx.x) * p.tokens;
    const int32_t here = static_cast<int32_t>(min(static_cast<int64_t>(p.tokens), p.n_tokens - token0));
    if (static_cast<int32_t>(threadIdx.x) < here) {
        const int64_t slot = LoadIndex(p.slots, p.slots64, token0 + threadIdx.x);
        const int64_t page = slot >= 0 ? slot / p.pools.page_tokens : -1;
        const bool write = page >= 0 && page < p.pools.pool_pages;
        rows[threadIdx.x] = write ? page * p.pools.page_stride + (slot - page * p.pools.page_tokens) * p.pools.token_stride : -1;
        if (!write && slot != -1 && blockIdx.y == 0) CountSkipped(p.status, static_cast<uint32_t>(token0 + threadIdx.x), 1u);
    }
    const uint32_t n_items = static_cast<uint32_t>(here) * p.token_items.d;
    const uint32_t stride = kAppendThreads * kAppendItems * gridDim.y;
    bool ready = false;
    for (uint32_t base = blockIdx.y * kAppendThreads * kAppendItems; base < n_items; base += stride) {
        Piece a[kAppendItems], b[kAppendItems];
        T *to_a[kAppendItems], *to_b[kAppendItems];
        int32_t freq[kAppendItems], pool_token[kAppendItems];
#pragma unroll
        for (int i = 0; i < kAppendItems; ++i) {
            const uint32_t item = base + i * kAppendThreads + threadIdx.x;
            to_a[i] = to_b[i] = nullptr;
            freq[i] = -1;
            pool_token[i] = -1;
            if (item >= n_items) continue;
            const uint32_t in_block = p.token_items(item);
            const uint32_t of_token = item - in_block * p.token_items.d;
            const int64_t token = token0 + in_block;
            const T *from;
            T *to;
            uint32_t within;
            if (of_token < p.qk_items) {
                const uint32_t head = p.head_items(of_token);
                within = of_token - head * p.head_items.d;
                if (head < static_cast<uint32_t>(p.n_q_heads)) {
                    from = static_cast<const T *>(p.query.src) + token * p.query.src_token + head * p.query.src_head;
                    to = static_cast<T *>(p.query.dst) + token * p.query.dst_token + head * p.query.dst_head;
                } else {
                    const uint32_t kv = head - p.n_q_heads;
                    from = static_cast<const T *>(p.key.src) + token * p.key.src_token + kv * p.key.src_head;
                    to = reinterpret_cast<T *>(p.pools.k + kv * p.pools.head_stride);
                    pool_token[i] = static_cast<int32_t>(in_block);
                }
                if (within < p.rot_items) {
                    const uint32_t first = kInterleaved ? within * 2 * V : within * V;
                    const uint32_t second = kInterleaved ? first + V : first + p.rotary_half;
                    freq[i] = static_cast<int32_t>(in_block * p.rotary_half + within * (V == 1 ? 1 : 2));
                    a[i] = *reinterpret_cast<const Piece *>(from + first);
                    b[i] = *reinterpret_cast<const Piece *>(from + second);
                    to_a[i] = to + first;
                    to_b[i] = to + second;
                    continue;
                }
                within = 2 * p.rotary_half + (within - p.rot_items) * V;
            } else {
                const uint32_t v = of_token - p.qk_items;
                const uint32_t kv = p.value_items(v);
                within = (v - kv * p.value_items.d) * V;
                from = static_cast<const T *>(p.value.src) + token * p.value.src_token + kv * p.value.src_head;
                to = reinterpret_cast<T *>(p.pools.v + kv * p.pools.head_stride);
                pool_token[i] = static_cast<int32_t>(in_block);
            }
            a[i] = *reinterpret_cast<const Piece *>(from + within);
            to_a[i] = to + within;
        }
        if (!ready) {
            const int32_t pairs = here * p.rotary_half;
            for (int32_t j = threadIdx.x; j < pairs; j += kAppendThreads) {
                const int32_t in_block = j / p.rotary_half;
                const double position = static_cast<double>(LoadIndex(p.positions, p.positions64, token0 + in_block));
                const double angle = position * static_cast<double>(__ldg(p.inv_freq + (j - in_block * p.rotary_half)));
                double turns = angle * 0.15915494309189533577;  // 1 / (2 pi)
                turns -= rint(turns);
                float s, c;
                sincospif(static_cast<float>(2.0 * turns), &s, &c);
                const uint32_t pair = j - in_block * p.rotary_half;
                cs[in_block * p.rotary_half + AngleAt<V>(pair, p.rot_items)] = make_float2(c * p.factor, s * p.factor);
            }
            __syncthreads();
            ready = true;
        }
#pragma unroll
        for (int i = 0; i < kAppendItems; ++i) {
            if (freq[i] >= 0) {
                float2 r[V];
                if constexpr (V == 1) {
                    r[0] = cs[freq[i]];
                } else {
#pragma unroll
                    for (int e = 0; e < V; e += 2) {
                        const float4 two = *reinterpret_cast<const float4 *>(cs + freq[i] + e * p.rot_items);
                        r[e] = make_float2(two.x, two.y);
                        r[e + 1] = make_float2(two.z, two.w);
                    }
                }
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    // interleaved: pair e of the 2 V consecutive elements held by a and b together
                    T &x = kInterleaved ? (2 * e < V ? a[i].x[2 * e] : b[i].x[2 * e - V]) : a[i].x[e];
                    T &y = kInterleaved ? (2 * e + 1 < V ? a[i].x[2 * e + 1] : b[i].x[2 * e + 1 - V]) : b[i].x[e];
                    const float xf = Half16<T>::ToFloat(x), yf = Half16<T>::ToFloat(y);
                    x = Half16<T>::FromFloat(xf * r[e].x - yf * r[e].y);
                    y = Half16<T>::FromFloat(yf * r[e].x + xf * r[e].y);
                }
            }
            if (to_a[i] == nullptr) continue;
            int64_t row = 0;
            if (pool_token[i] >= 0) {
                row = rows[pool_token[i]];
                if (row < 0) continue;  // padding, or no such slot
            }
            StorePiece(reinterpret_cast<uint8_t *>(to_a[i]) + row, a[i]);
            if (to_b[i] != nullptr) StorePiece(reinterpret_cast<uint8_t *>(to_b[i]) + row, b[i]);
        }
    }
}

template <typename T, int V>
void LaunchAppend(AppendParams p, bool interleaved, cudaStream_t stream) {
    // Few tokens: several CTAs share a token's heads, each forming the angles for itself.  Many: several tokens to a CTA,
    // as long as every SM still gets a few CTAs.
    const int32_t sm_count = GetDeviceInfo().sm_count;
    const uint32_t rounds = (p.token_items.d + kAppendThreads * kAppendItems - 1) / (kAppendThreads * kAppendItems);
    const uint32_t split = p.n_tokens >= sm_count ? 1u : rounds;
    p.tokens = 1;
    while (p.tokens < kMaxAppendTokens && p.n_tokens / (p.tokens * 2) >= 8 * sm_count) p.tokens *= 2;
    const dim3 grid(static_cast<uint32_t>((p.n_tokens + p.tokens - 1) / p.tokens), std::min(std::max(split, 1u), 65535u));
    const size_t smem = static_cast<size_t>(p.tokens) * p.rotary_half * sizeof(float2);
    if (interleaved) {
        AppendPagesKernel<T, V, true><<<grid, kAppendThreads, smem, stream>>>(p);
    } else {
        AppendPagesKernel<T, V, false><<<grid, kAppendThreads, smem, stream>>>(p);
    }
}

template <typename T>
void DispatchAppend(AppendParams p, int v, bool interleaved, cudaStream_t stream) {
    p.rot_items = static_cast<uint32_t>(p.rotary_half / v);
    p.head_items = FastDivide(p.rot_items + static_cast<uint32_t>((p.pools.head_dim - 2 * p.rotary_half) / v));
    p.value_items = FastDivide(static_cast<uint32_t>(p.pools.head_dim / v));
    p.qk_items = (static_cast<uint32_t>(p.n_q_heads) + p.pools.n_kv_heads) * p.head_items.d;
    p.token_items = FastDivide(p.qk_items + static_cast<uint32_t>(p.pools.n_kv_heads) * p.value_items.d);
    switch (v) {
        case 8: LaunchAppend<T, 8>(p, interleaved, stream); break;
        case 4: LaunchAppend<T, 4>(p, interleaved, stream); break;
        case 2: LaunchAppend<T, 2>(p, interleaved, stream); break;
        default: LaunchAppend<T, 1>(p, interleaved, stream); break;
    }
}

}  // namespace
}  // namespace kvcm

extern "C" {

int32_t kvcm_b200_append_pages(const kvcm_b200_kv_pools_t *pools, const void *d_query, int64_t q_token_stride,
                               int64_t q_head_stride, int32_t n_q_heads, void *d_query_out, int64_t qo_token_stride,
                               int64_t qo_head_stride, const void *d_key, int64_t k_token_stride,
                               int64_t k_head_stride, const void *d_value, int64_t v_token_stride,
                               int64_t v_head_stride, const void *d_positions, int32_t position_bytes,
                               const void *d_slot_idx, int32_t slot_bytes, int32_t n_tokens, const float *d_inv_freq,
                               int32_t rotary_dim, int32_t interleaved, float attention_factor, uint32_t *d_status,
                               kvcm_stream_t stream) {
    using namespace kvcm;
    const int32_t rc = CheckPools(pools, kMaxAppendHeadDim);
    if (rc != KVCM_OK) return rc;
    if (n_tokens < 0 || n_q_heads < 0 || n_q_heads > 65536 || pools->n_kv_heads > 65536 || rotary_dim < 0 ||
        rotary_dim % 2 != 0 || rotary_dim > pools->head_dim || (position_bytes != 4 && position_bytes != 8) ||
        (slot_bytes != 4 && slot_bytes != 8)) {
        return KVCM_ER_INVALID_PARAMS;
    }
    if (n_tokens > 0 && (d_key == nullptr || d_value == nullptr || d_positions == nullptr || d_slot_idx == nullptr ||
        (rotary_dim > 0 && d_inv_freq == nullptr) || (n_q_heads > 0 && (d_query == nullptr || d_query_out == nullptr)))) {
        return KVCM_ER_INVALID_ADDRESS;
    }
    AppendParams p{};
    p.pools = AsPagedPools(*pools);
    p.query = {d_query, d_query_out, q_token_stride, q_head_stride, qo_token_stride, qo_head_stride};
    p.key = {d_key, nullptr, k_token_stride, k_head_stride, 0, 0};
    p.value = {d_value, nullptr, v_token_stride, v_head_stride, 0, 0};
    p.positions = d_positions;
    p.slots = d_slot_idx;
    p.positions64 = position_bytes == 8;
    p.slots64 = slot_bytes == 8;
    p.inv_freq = d_inv_freq;
    p.status = d_status;
    p.n_q_heads = n_q_heads;
    p.rotary_half = rotary_dim / 2;
    p.factor = attention_factor;
    // The widest piece that every address, stride and the rotary split allow, in elements of two bytes.
    uint64_t bits = static_cast<uint64_t>(pools->page_stride) | static_cast<uint64_t>(pools->token_stride) |
                    static_cast<uint64_t>(pools->head_stride) | static_cast<uint64_t>(k_token_stride) |
                    static_cast<uint64_t>(k_head_stride) | static_cast<uint64_t>(v_token_stride) |
                    static_cast<uint64_t>(v_head_stride) | static_cast<uint64_t>(pools->head_dim) |
                    static_cast<uint64_t>(p.rotary_half) | static_cast<uint64_t>(pools->head_dim - rotary_dim);
    uintptr_t addresses = reinterpret_cast<uintptr_t>(pools->k_pool) | reinterpret_cast<uintptr_t>(pools->v_pool) |
                          reinterpret_cast<uintptr_t>(d_key) | reinterpret_cast<uintptr_t>(d_value);
    if (n_q_heads > 0) {
        bits |= static_cast<uint64_t>(q_token_stride) | static_cast<uint64_t>(q_head_stride) |
                static_cast<uint64_t>(qo_token_stride) | static_cast<uint64_t>(qo_head_stride);
        addresses |= reinterpret_cast<uintptr_t>(d_query) | reinterpret_cast<uintptr_t>(d_query_out);
    }
    if (addresses & 1u) return KVCM_ER_INVALID_ADDRESS;
    // A query that is rotated in place is read and written piece by piece, each by one thread.
    if (n_q_heads > 0 && d_query == d_query_out && ((n_tokens > 1 && q_token_stride != qo_token_stride) ||
                                                    (n_q_heads > 1 && q_head_stride != qo_head_stride))) {
        return KVCM_ER_INVALID_PARAMS;
    }
    if (!HaveDevice()) return KVCM_ER_NO_DEVICE;
    if (n_tokens == 0) return KVCM_OK;
    int v = 8;
    while (v > 1 && ((bits & (v - 1)) != 0 || (addresses & (2 * v - 1)) != 0)) v /= 2;
    p.n_tokens = n_tokens;
    if (pools->dtype == KVCM_DTYPE_BF16) {
        DispatchAppend<__nv_bfloat16>(p, v, interleaved != 0, AsStream(stream));
    } else {
        DispatchAppend<__half>(p, v, interleaved != 0, AsStream(stream));
    }
    return LaunchStatus();
}

}  // extern "C"
