// Rotary positions and append: new tokens' queries and keys rotated, keys and values written into their pool slots.
//
// For token t and pair j < rotary_dim / 2 with angle a = positions[t] * inv_freq[j]:
//   (x, y) -> f * (x cos a - y sin a, y cos a + x sin a)
// the pair being elements (j, j + rotary_dim / 2) of a head, or (2j, 2j + 1).
//
// Bound by HBM: every query element is read and written once, every key and value element read once and written once,
// 24.6 KB per token at 32 query and 8 KV heads of 128.  The angles of a token are shared by all its heads, so one CTA
// takes one token, forms rotary_dim / 2 sine-cosine pairs once into shared memory, and its threads walk the token's
// heads in 16-byte pieces.  The first pieces are loaded before the angles are formed, so the latency of the two
// overlaps.  An angle is formed and reduced to one turn in 64 bits: at position 10^6 a 32-bit product would be off by
// 0.06 rad.
#include "paged_kv.cuh"

namespace kvcm {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendItems = 2;  // items a thread loads before it stores the first
constexpr int kMaxAppendHeadDim = 1024;

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
    uint32_t rot_items;   // per head: items of 2 x V elements that are rotated
    uint32_t head_items;  // rot_items + items of V elements that pass through
    uint32_t value_items;
    uint32_t n_items;  // per token
};

__device__ __forceinline__ int64_t LoadIndex(const void *p, int32_t is64, int64_t i) {
    return is64 ? __ldg(static_cast<const long long *>(p) + i) : static_cast<int64_t>(__ldg(static_cast<const int *>(p) + i));
}

template <typename T, int V>
struct alignas(2 * V) Vec {
    T x[V];
};

template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kAppendThreads) AppendPagesKernel(const AppendParams p) {
    __shared__ float2 cs[kMaxAppendHeadDim / 2];
    using Piece = Vec<T, V>;
    const int64_t token = blockIdx.x;
    const int64_t slot = LoadIndex(p.slots, p.slots64, token);
    const int64_t page = slot >= 0 ? slot / p.pools.page_tokens : -1;
    const bool write = page >= 0 && page < p.pools.pool_pages;
    const int64_t row = write ? page * p.pools.page_stride + (slot - page * p.pools.page_tokens) * p.pools.token_stride : 0;
    if (!write && slot != -1 && threadIdx.x == 0 && blockIdx.y == 0) {
        CountSkipped(p.status, static_cast<uint32_t>(token), 1u);
    }
    const uint32_t qk_items = (static_cast<uint32_t>(p.n_q_heads) + p.pools.n_kv_heads) * p.head_items;
    const uint32_t stride = kAppendThreads * kAppendItems * gridDim.y;
    bool have_angles = false;
    for (uint32_t base = blockIdx.y * kAppendThreads * kAppendItems; base < p.n_items; base += stride) {
        Piece a[kAppendItems], b[kAppendItems];
        T *to_a[kAppendItems], *to_b[kAppendItems];
        int32_t freq[kAppendItems];
#pragma unroll
        for (int i = 0; i < kAppendItems; ++i) {
            const uint32_t item = base + i * kAppendThreads + threadIdx.x;
            to_a[i] = to_b[i] = nullptr;
            freq[i] = -1;
            if (item >= p.n_items) continue;
            const T *from;
            T *to;
            uint32_t within;
            if (item < qk_items) {
                const uint32_t head = item / p.head_items;
                within = item - head * p.head_items;
                if (head < static_cast<uint32_t>(p.n_q_heads)) {
                    from = static_cast<const T *>(p.query.src) + token * p.query.src_token + head * p.query.src_head;
                    to = static_cast<T *>(p.query.dst) + token * p.query.dst_token + head * p.query.dst_head;
                } else {
                    if (!write) continue;
                    const uint32_t kv = head - p.n_q_heads;
                    from = static_cast<const T *>(p.key.src) + token * p.key.src_token + kv * p.key.src_head;
                    to = reinterpret_cast<T *>(p.pools.k + row + kv * p.pools.head_stride);
                }
                if (within < p.rot_items) {
                    const uint32_t first = kInterleaved ? within * 2 * V : within * V;
                    const uint32_t second = kInterleaved ? first + V : first + p.rotary_half;
                    freq[i] = static_cast<int32_t>(within * V);
                    a[i] = *reinterpret_cast<const Piece *>(from + first);
                    b[i] = *reinterpret_cast<const Piece *>(from + second);
                    to_a[i] = to + first;
                    to_b[i] = to + second;
                    continue;
                }
                within = 2 * p.rotary_half + (within - p.rot_items) * V;
            } else {
                if (!write) continue;
                const uint32_t v = item - qk_items;
                const uint32_t kv = v / p.value_items;
                within = (v - kv * p.value_items) * V;
                from = static_cast<const T *>(p.value.src) + token * p.value.src_token + kv * p.value.src_head;
                to = reinterpret_cast<T *>(p.pools.v + row + kv * p.pools.head_stride);
            }
            a[i] = *reinterpret_cast<const Piece *>(from + within);
            to_a[i] = to + within;
        }
        if (!have_angles) {
            const double position = static_cast<double>(LoadIndex(p.positions, p.positions64, token));
            for (int32_t j = threadIdx.x; j < p.rotary_half; j += kAppendThreads) {
                const double angle = position * static_cast<double>(__ldg(p.inv_freq + j));
                double turns = angle * 0.15915494309189533577;  // 1 / (2 pi)
                turns -= rint(turns);
                float s, c;
                sincospif(static_cast<float>(2.0 * turns), &s, &c);
                cs[j] = make_float2(c * p.factor, s * p.factor);
            }
            __syncthreads();
            have_angles = true;
        }
#pragma unroll
        for (int i = 0; i < kAppendItems; ++i) {
            if (freq[i] >= 0) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float2 r = cs[freq[i] + e];
                    // interleaved: pair e of the 2 V consecutive elements held by a and b together
                    T &x = kInterleaved ? (2 * e < V ? a[i].x[2 * e] : b[i].x[2 * e - V]) : a[i].x[e];
                    T &y = kInterleaved ? (2 * e + 1 < V ? a[i].x[2 * e + 1] : b[i].x[2 * e + 1 - V]) : b[i].x[e];
                    const float xf = Half16<T>::ToFloat(x), yf = Half16<T>::ToFloat(y);
                    x = Half16<T>::FromFloat(xf * r.x - yf * r.y);
                    y = Half16<T>::FromFloat(yf * r.x + xf * r.y);
                }
            }
            if (to_a[i] != nullptr) *reinterpret_cast<Piece *>(to_a[i]) = a[i];
            if (to_b[i] != nullptr) *reinterpret_cast<Piece *>(to_b[i]) = b[i];
        }
    }
}

template <typename T, int V>
void LaunchAppend(const AppendParams &p, int32_t n_tokens, bool interleaved, cudaStream_t stream) {
    // One or a few tokens: several CTAs share a token's heads, each forming the angles for itself.
    const uint32_t rounds = (p.n_items + kAppendThreads * kAppendItems - 1) / (kAppendThreads * kAppendItems);
    const uint32_t wanted = n_tokens >= GetDeviceInfo().sm_count ? 1u : rounds;
    const dim3 grid(static_cast<uint32_t>(n_tokens), std::min(std::max(wanted, 1u), 65535u));
    if (interleaved) {
        AppendPagesKernel<T, V, true><<<grid, kAppendThreads, 0, stream>>>(p);
    } else {
        AppendPagesKernel<T, V, false><<<grid, kAppendThreads, 0, stream>>>(p);
    }
}

template <typename T>
void DispatchAppend(AppendParams p, int v, int32_t n_tokens, bool interleaved, cudaStream_t stream) {
    p.rot_items = static_cast<uint32_t>(p.rotary_half / v);
    p.head_items = p.rot_items + static_cast<uint32_t>((p.pools.head_dim - 2 * p.rotary_half) / v);
    p.value_items = static_cast<uint32_t>(p.pools.head_dim / v);
    p.n_items = (static_cast<uint32_t>(p.n_q_heads) + p.pools.n_kv_heads) * p.head_items +
                static_cast<uint32_t>(p.pools.n_kv_heads) * p.value_items;
    switch (v) {
        case 8: LaunchAppend<T, 8>(p, n_tokens, interleaved, stream); break;
        case 4: LaunchAppend<T, 4>(p, n_tokens, interleaved, stream); break;
        case 2: LaunchAppend<T, 2>(p, n_tokens, interleaved, stream); break;
        default: LaunchAppend<T, 1>(p, n_tokens, interleaved, stream); break;
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
    AppendParams p = {};
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
    if (!HaveDevice()) return KVCM_ER_NO_DEVICE;
    if (n_tokens == 0) return KVCM_OK;
    int v = 8;
    while (v > 1 && ((bits & (v - 1)) != 0 || (addresses & (2 * v - 1)) != 0)) v /= 2;
    if (pools->dtype == KVCM_DTYPE_BF16) {
        DispatchAppend<__nv_bfloat16>(p, v, n_tokens, interleaved != 0, AsStream(stream));
    } else {
        DispatchAppend<__half>(p, v, n_tokens, interleaved != 0, AsStream(stream));
    }
    return LaunchStatus();
}

}  // extern "C"
