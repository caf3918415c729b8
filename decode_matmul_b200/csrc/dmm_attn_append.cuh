// From the result of a qkv product to rotated queries and new rows of a paged key-value cache, in one pass.
//
// Token at position p, pair i of a query or key head: angle w = p * freqs[i], (a, b) -> (a cos w - b sin w, a sin w + b cos w).
// Positions go to 10^5 and beyond, where a 32-bit angle is off by 10^-2: the angle is taken in turns in 64 bits, its whole
// turns go, and the sine and cosine of what is left are 32-bit ones.
//
// A block has one token and some of its heads.  The D / 2 sines and cosines of the token are worked out once per block
// into shared memory; then a thread takes 16 values of a head at a time, as two runs of 8 (the two halves of 8 pairs, or 8
// neighbouring pairs), so that every load and store is 16 bytes wide, and asks for its next 16 before it works on these.
//
// Bound: bytes, 4 (fp32) or 2 read and 2 written for each value.  B200, graph: 2048 tokens of 64 + 16 heads of 128, fp32 in,
// 22.0 us (5.7 TB/s, 88 % of what a copy reaches); 8164 tokens of prompts of many lengths 81 us (6.2 TB/s, 94 %).  One token
// takes 2.9 us (2.3 when all of it is in L2), a launch and three dependent loads: its sequence's length and page and the row itself.
#pragma once

#include "dmm_attn_common.cuh"

namespace dmm {

constexpr int kAppendThreads = 128;

struct AppendParams {
    const void *qkv;
    const double *freqs;
    void *q_out;
    const int32_t *cu;
    long long qkv_ld, q_ld;
    CacheView cache;
    int tokens, heads, interleaved;
};

// 8 consecutive values as floats
__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <class T>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack16<T>(ws[i]);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}
template <class T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(p) =
        make_uint4(pack16<T>(x[0], x[1]), pack16<T>(x[2], x[3]), pack16<T>(x[4], x[5]), pack16<T>(x[6], x[7]));
}

template <class TIn, class T, int D>
__global__ void __launch_bounds__(kAppendThreads) append_kv_kernel(const AppendParams p) {
    __shared__ int s_seq;
    __shared__ float s_cos[D / 2], s_sin[D / 2];
    grid_dep_wait();
    const int t = blockIdx.x;
    constexpr int kRuns = D / 16;
    const int units = (p.heads + 2 * p.cache.kv_heads) * kRuns;
    const TIn *src = static_cast<const TIn *>(p.qkv) + t * p.qkv_ld;
    // The first values are asked for before it is known where they go, and then always the next ones ahead.
    float a[8], bb[8];
    const auto load = [&](int u, float (&lo)[8], float (&hi)[8]) {
        const int c = u % kRuns;
        const TIn *from = src + u / kRuns * D;
        load8(from + (p.interleaved ? 16 * c : 8 * c), lo);
        load8(from + (p.interleaved ? 16 * c + 8 : D / 2 + 8 * c), hi);
    };
    int u = blockIdx.y * kAppendThreads + threadIdx.x;
    if (u < units) load(u, a, bb);
    const int b = token_sequence<kAppendThreads>(p.cu, p.cache.num_seqs, p.tokens, t, &s_seq);
    if (b < 0) return;
    const TokenSpan span = token_span(p.cu, b, p.tokens);
    const int pos = cache_len(p.cache, b) - span.n + (t - span.begin);
    if (pos < 0) {  // (without cu: a sequence that has no tokens, whose place in the batch is idle)
        if (p.cu != nullptr) raise_status(DMM_STATUS_BAD_PAGE);
        return;
    }
    if (p.freqs != nullptr && threadIdx.x < D / 2) {
        const double turns = static_cast<double>(pos) * p.freqs[threadIdx.x] * 0.15915494309189533577;  // 1 / (2 pi)
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s_sin[threadIdx.x], &s_cos[threadIdx.x]);
    }
    __syncthreads();
    const long long row = cache_row(p.cache, b, pos, 0);
    while (u < units) {
        const int head = u / kRuns, c = u % kRuns;
        const int lo = p.interleaved ? 16 * c : 8 * c, hi = p.interleaved ? 16 * c + 8 : D / 2 + 8 * c;
        u += gridDim.y * kAppendThreads;
        float next_a[8], next_bb[8];
        if (u < units) load(u, next_a, next_bb);
        if (p.freqs != nullptr && head < p.heads + p.cache.kv_heads) {
            const float *cs = s_cos + 8 * c, *sn = s_sin + 8 * c;
            if (p.interleaved) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x0 = a[2 * i], y0 = a[2 * i + 1], x1 = bb[2 * i], y1 = bb[2 * i + 1];
                    a[2 * i] = x0 * cs[i] - y0 * sn[i];
                    a[2 * i + 1] = x0 * sn[i] + y0 * cs[i];
                    bb[2 * i] = x1 * cs[i + 4] - y1 * sn[i + 4];
                    bb[2 * i + 1] = x1 * sn[i + 4] + y1 * cs[i + 4];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = a[i], y = bb[i];
                    a[i] = x * cs[i] - y * sn[i];
                    bb[i] = x * sn[i] + y * cs[i];
                }
            }
        }
        T *dst = static_cast<T *>(p.q_out) + t * p.q_ld + head * D;
        if (head >= p.heads) {
            const int h = head - p.heads;
            dst = h < p.cache.kv_heads ? static_cast<T *>(p.cache.k) + row + h * p.cache.head_stride
                                       : static_cast<T *>(p.cache.v) + row + (h - p.cache.kv_heads) * p.cache.head_stride;
        }
        if (head < p.heads || row >= 0) {
            store8(dst + lo, a);
            store8(dst + hi, bb);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a[i] = next_a[i];
            bb[i] = next_bb[i];
        }
    }
}

template <class TIn, class T, int D>
inline int launch_append_typed(const AppendParams &p, int num_sms, bool pdl, cudaStream_t stream) {
    const int units = (p.heads + 2 * p.cache.kv_heads) * (D / 16);
    // Few tokens: a thread takes one unit, so that all of the GPU loads at once (with all of it in L2 one token of 80 heads 2.1 us
    // against 3.6 with one block for the token, 32 tokens of 96 heads 2.6 against 4.3); many: a block keeps its token, whose sines and cosines it works out
    // once (8164 tokens 81 us against 92).
    int parts = (units + kAppendThreads - 1) / kAppendThreads;
    if (static_cast<long long>(parts) * p.tokens > 16ll * num_sms) parts = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.tokens), static_cast<unsigned>(parts));
    cfg.blockDim = dim3(kAppendThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, append_kv_kernel<TIn, T, D>, p);
}

template <class T, int D>
inline int launch_append(const AppendParams &p, int qkv_type, int num_sms, bool pdl, cudaStream_t stream) {
    switch (qkv_type) {
        case DMM_T_F32: return launch_append_typed<float, T, D>(p, num_sms, pdl, stream);
        case DMM_T_F16: return launch_append_typed<__half, T, D>(p, num_sms, pdl, stream);
        default: return launch_append_typed<__nv_bfloat16, T, D>(p, num_sms, pdl, stream);
    }
}

}  // namespace dmm
