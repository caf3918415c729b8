// Attention over a paged cache, the simplest form: a block has one query row, its four warps take keys in turn, each
// with a running maximum m, sum l = sum exp(x - m) and weighted sum of values, and the four are joined at the end.
#pragma once

#include "dmm_attn_common.cuh"

namespace dmm {

struct AttnParams {
    const void *q;
    void *out;
    const int32_t *cu;
    long long q_ld, out_ld;
    CacheView cache;
    int tokens, heads, group;
    float scale;
};

template <class T, int D>
__global__ void __launch_bounds__(128) attention_simple_kernel(const AttnParams p) {
    constexpr int kV = D / 32;  // values per lane
    __shared__ int s_seq;
    __shared__ float s_m[4], s_l[4], s_o[4][D];
    grid_dep_wait();
    const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int b = token_sequence<128>(p.cu, p.cache.num_seqs, p.tokens, t, &s_seq);
    if (b < 0) return;
    const TokenSpan span = token_span(p.cu, b, p.tokens);
    const int keys = cache_len(p.cache, b) - span.n + (t - span.begin) + 1;
    const T *qp = static_cast<const T *>(p.q) + t * p.q_ld + h * D + lane * kV;
    float q[kV], o[kV] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kV; ++i) q[i] = static_cast<float>(qp[i]) * p.scale;
    for (int j = warp; j < keys; j += 4) {
        const long long row = cache_row(p.cache, b, j, h / p.group);
        float x = 0.0f, v[kV] = {};
        if (row >= 0) {
            const T *kp = static_cast<const T *>(p.cache.k) + row + lane * kV, *vp = static_cast<const T *>(p.cache.v) + row + lane * kV;
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                x += q[i] * static_cast<float>(kp[i]);
                v[i] = static_cast<float>(vp[i]);
            }
        }
        for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
        const float mn = fmaxf(m, x), f = m == -INFINITY ? 0.0f : expf(m - mn), e = expf(x - mn);
        l = l * f + e;
#pragma unroll
        for (int i = 0; i < kV; ++i) o[i] = o[i] * f + e * v[i];
        m = mn;
    }
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
    for (int i = 0; i < kV; ++i) s_o[warp][lane * kV + i] = o[i];
    __syncthreads();
    if (threadIdx.x < D) {
        float mm = -INFINITY, sum = 0.0f, acc = 0.0f;
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, s_m[w]);
        for (int w = 0; w < 4; ++w) {
            const float f = s_l[w] == 0.0f ? 0.0f : expf(s_m[w] - mm);
            sum += f * s_l[w];
            acc += f * s_o[w][threadIdx.x];
        }
        T *op = static_cast<T *>(p.out) + t * p.out_ld + h * D;
        op[threadIdx.x] = static_cast<T>(keys > 0 ? acc / sum : 0.0f);
    }
}

template <class T, int D>
inline int launch_attention(const AttnParams &p, bool pdl, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.tokens), static_cast<unsigned>(p.heads));
    cfg.blockDim = dim3(128);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, attention_simple_kernel<T, D>, p);
}

}  // namespace dmm
