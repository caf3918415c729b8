// What the attention kernels share: 16-bit types, the view of a paged cache, and the way from a row of packed tokens to its
// sequence and position.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "dmm_common.cuh"

namespace dmm {

// two floats rounded to one word of two 16-bit values, a in the low half
template <class T>
__device__ __forceinline__ uint32_t pack16(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <class T>
__device__ __forceinline__ float2 unpack16(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack16<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <>
__device__ __forceinline__ float2 unpack16<__nv_bfloat16>(uint32_t w) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w));
}

// Weights of a softmax, which the tensor cores take in the type of the values: 2^(x - m + kRaise<T>) against a running maximum m
// that is 8 too low at most.  fp16 ends at 2^-25: against a heaviest weight of 1, many light ones beside one heavy key lose their
// bits or vanish, while the sum of weights has them.  Raised by 7, the heaviest has 2^7 to 2^15, and what vanishes is 2^-32 of it.  (2048 keys
// beside one that is e^16 times as heavy and has a value of 0: off by 0.48 % on average and 2.3 % at worst without it, 0.017 % and 0.056 % with it.)  The
// factor is in the sums too, and cancels.  bf16 has the range of fp32.
template <class T>
constexpr float kRaise = 0.0f;
template <>
constexpr float kRaise<__half> = 7.0f;
// Two of them rounded to one word.  Scores beyond 2^24, where their products with the scale are rounded to more than 1, can come out above
// 2^16: not infinite.
template <class T>
__device__ __forceinline__ uint32_t pack_weights(float a, float b) {
    return pack16<T>(a, b);
}
template <>
__device__ __forceinline__ uint32_t pack_weights<__half>(float a, float b) {
    uint32_t w;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    return w;
}

// 2^x, off by 2^-22 at most
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void load_floats(const float *p, float (&x)[4]) {
    const float4 f = *reinterpret_cast<const float4 *>(p);
    x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
}
__device__ __forceinline__ void load_floats(const float *p, float (&x)[2]) {
    const float2 f = *reinterpret_cast<const float2 *>(p);
    x[0] = f.x, x[1] = f.y;
}

// Lets a kernel have more than 48 KB of dynamic shared memory, once per device.
struct SmemAllowance {
    std::atomic<bool> given[64];
    int get(const void *kernel, unsigned bytes) {
        int dev = 0;
        cudaError_t err = cudaGetDevice(&dev);
        if (err != cudaSuccess) return err;
        if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
        if (given[dev].load(std::memory_order_relaxed)) return 0;
        err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
        if (err == cudaSuccess) given[dev].store(true, std::memory_order_relaxed);
        return err;
    }
};

// The cache as the kernels see it (dmm_paged_cache).
struct CacheView {
    void *k, *v;
    const int32_t *page_table;
    const int32_t *seq_lens;
    long long page_stride, head_stride, row_stride, table_stride;
    int num_pages, kv_heads, page_shift, num_seqs, max_pages;
};

// Length of sequence b, within what its row of the page table can hold.
__device__ __forceinline__ int cache_len(const CacheView &c, int b) {
    const int len = c.seq_lens[b];
    const long long most = static_cast<long long>(c.max_pages) << c.page_shift;
    if (len >= 0 && len <= most) return len;
    raise_status(DMM_STATUS_BAD_PAGE);
    return len < 0 ? 0 : static_cast<int>(most);
}

// Offset (in elements) of the row of token `pos` of sequence b, head h; -1 when the table names a page that the cache does not have.
__device__ __forceinline__ long long cache_row(const CacheView &c, int b, int pos, int h) {
    const int page = c.page_table[b * c.table_stride + (pos >> c.page_shift)];
    if (page < 0 || page >= c.num_pages) {
        raise_status(DMM_STATUS_BAD_PAGE);
        return -1;
    }
    return page * c.page_stride + h * c.head_stride + (pos & ((1 << c.page_shift) - 1)) * c.row_stride;
}

// The rows of sequence b among the packed tokens: [begin, begin + n).
struct TokenSpan {
    int begin, n;
};
__device__ __forceinline__ TokenSpan token_span(const int32_t *cu, int b, int tokens) {
    if (cu == nullptr) return {b, b < tokens ? 1 : 0};
    const int c0 = cu[b], c1 = cu[b + 1];
    if (c0 < 0 || c1 < c0 || c1 > tokens) {
        raise_status(DMM_STATUS_BAD_PAGE);
        return {0, 0};
    }
    return {c0, c1 - c0};
}

// The sequence that row t of the packed tokens belongs to, -1 behind the last one.  Called by every thread of a block of NT
// threads; *found is a word of shared memory.
template <int NT>
__device__ __forceinline__ int token_sequence(const int32_t *cu, int num_seqs, int tokens, int t, int *found) {
    if (cu == nullptr) return t < num_seqs ? t : -1;
    if (threadIdx.x == 0) *found = -1;
    __syncthreads();
    for (int b = threadIdx.x; b < num_seqs; b += NT) {
        const TokenSpan s = token_span(cu, b, tokens);
        if (s.begin <= t && t - s.begin < s.n) *found = b;
    }
    __syncthreads();
    return *found;
}

}  // namespace dmm
