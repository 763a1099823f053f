// What the decode-step kernels (append, attend, evict) share: the description of a layer's two pools and the checks
// every entry point makes on it.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kvcm_common.cuh"

namespace kvcm {

// A layer's pools as the kernels address them: byte strides, row (page, token, head) at
// pool + page * page_stride + token * token_stride + head * head_stride.
struct PagedPools {
    uint8_t *k;
    uint8_t *v;
    int64_t page_stride;
    int64_t token_stride;
    int64_t head_stride;
    int64_t pool_pages;
    int32_t page_tokens;
    int32_t n_kv_heads;
    int32_t head_dim;
};

constexpr int64_t kMaxTableTokens = int64_t{1} << 30;

inline PagedPools AsPagedPools(const kvcm_b200_kv_pools_t &p) {
    PagedPools q;
    q.k = static_cast<uint8_t *>(p.k_pool);
    q.v = static_cast<uint8_t *>(p.v_pool);
    q.page_stride = p.page_stride * 2;
    q.token_stride = p.token_stride * 2;
    q.head_stride = p.head_stride * 2;
    q.pool_pages = p.pool_pages;
    q.page_tokens = p.page_tokens;
    q.n_kv_heads = p.n_kv_heads;
    q.head_dim = p.head_dim;
    return q;
}

inline int32_t CheckPools(const kvcm_b200_kv_pools_t *p, int32_t max_head_dim) {
    if (p == nullptr) return KVCM_ER_INVALID_ADDRESS;
    if (p->page_tokens <= 0 || p->n_kv_heads <= 0 || p->head_dim <= 0 || p->head_dim > max_head_dim ||
        p->pool_pages < 0 || p->pool_pages > INT32_MAX || p->page_stride < 0 || p->token_stride < 0 ||
        p->head_stride < 0 || static_cast<int64_t>(p->n_kv_heads) * p->head_dim > (1 << 24) || (p->dtype != KVCM_DTYPE_BF16 && p->dtype != KVCM_DTYPE_FP16)) {
        return KVCM_ER_INVALID_PARAMS;
    }
    if (p->k_pool == nullptr || p->v_pool == nullptr) return KVCM_ER_INVALID_ADDRESS;
    return KVCM_OK;
}

// Rows that are read or written in 16-byte pieces.
inline bool RowsAre16ByteAligned(const kvcm_b200_kv_pools_t &p) {
    return ((reinterpret_cast<uintptr_t>(p.k_pool) | reinterpret_cast<uintptr_t>(p.v_pool)) & 15u) == 0 &&
           ((p.page_stride | p.token_stride | p.head_stride | p.head_dim) & 7) == 0;
}

// What a call asks of the CUDA runtime, in order, and nothing after the first request that is refused: the kernels that
// follow another take their work from the workspace, and without it would run on whatever lies there.
class Requests {
public:
    template <typename Request>
    void Make(Request request) {
        if (error_ == cudaSuccess) error_ = request();
    }
    int32_t Status() const {
        if (error_ == cudaSuccess) return LaunchStatus();
        cudaGetLastError();  // what is reported here is not reported again
        return KVCM_ER_CUDAMEMCPY_ERROR;
    }

private:
    cudaError_t error_ = cudaSuccess;
};

// n / d for 32-bit numbers by one wide multiplication: magic = floor(2^64 / d) + 1 (0 for d = 1) is exact for all of them.
struct FastDivide {
    uint64_t magic;
    uint32_t d;
    FastDivide(uint32_t by = 1) : magic(by <= 1 ? 0 : ~uint64_t{0} / by + 1), d(by < 1 ? 1 : by) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
        return magic == 0 ? n : static_cast<uint32_t>(__umul64hi(n, magic));
    }
};

// status[0] += count, status[1] = max(status[1], 1 + number of the offending token or sequence).
__device__ __forceinline__ void CountSkipped(uint32_t *status, uint32_t number, uint32_t count) {
    if (status != nullptr) {
        atomicAdd(&status[0], count);
        atomicMax(&status[1], number + 1u);
    }
}

template <typename T>
struct Half16;
template <>
struct Half16<__nv_bfloat16> {
    using Pair = __nv_bfloat162;
    static __device__ __forceinline__ float ToFloat(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 FromFloat(float x) { return __float2bfloat16_rn(x); }
    static __device__ __forceinline__ float2 ToFloat2(Pair x) { return __bfloat1622float2(x); }
    static __device__ __forceinline__ Pair FromFloat2(float a, float b) { return __floats2bfloat162_rn(a, b); }
};
template <>
struct Half16<__half> {
    using Pair = __half2;
    static __device__ __forceinline__ float ToFloat(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half FromFloat(float x) { return __float2half_rn(x); }
    static __device__ __forceinline__ float2 ToFloat2(Pair x) { return __half22float2(x); }
    static __device__ __forceinline__ Pair FromFloat2(float a, float b) { return __floats2half2_rn(a, b); }
};

}  // namespace kvcm
