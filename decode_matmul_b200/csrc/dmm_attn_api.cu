// C ABI of the attention operators (declared in include/dmm.h): argument validation and launches.
#include <atomic>

#include "dmm_attn_append.cuh"
#include "dmm_attn_common.cuh"
#include "dmm_attn_decode.cuh"
#include "dmm_attn_prompt.cuh"
#include "dmm_launch.h"

namespace dmm {

static bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int take_attention_status(unsigned *v) { return take_status(v); }

static int device_sms(int *sms) {
    static std::atomic<int> known[64];  // zero: not asked yet
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    int n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        err = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        if (err != cudaSuccess) return err;
        known[dev].store(n, std::memory_order_relaxed);
    }
    *sms = n;
    return 0;
}

// Checks a cache description and turns it into what the kernels take.
static int cache_view(const dmm_paged_cache *c, CacheView *view) {
    if (!c || !c->k || !c->v || !c->page_table || !c->seq_lens) return DMM_ERR_NULL;
    if (c->type != DMM_T_F16 && c->type != DMM_T_BF16) return DMM_ERR_ARG;
    if (c->head_dim != 64 && c->head_dim != 128) return DMM_ERR_UNSUPPORTED;
    if (c->page_size < 16 || (c->page_size & (c->page_size - 1)) != 0) return DMM_ERR_UNSUPPORTED;
    if (c->kv_heads < 1 || c->kv_heads > 65535 || c->num_seqs < 1 || c->num_seqs > (1 << 20) || c->max_pages < 1 || c->num_pages < 1 ||
        c->num_pages > 0x7fffffff || c->table_stride < c->max_pages)
        return DMM_ERR_SHAPE;
    // positions are 32-bit numbers
    if (static_cast<long long>(c->max_pages) * c->page_size > (1ll << 30)) return DMM_ERR_SHAPE;
    if (!aligned16(c->k) || !aligned16(c->v)) return DMM_ERR_ALIGN;
    // no two rows overlap: from the smallest stride on, each holds all of the one before
    struct {
        long long n, stride;
    } dim[3] = {{c->num_pages, c->page_stride}, {c->kv_heads, c->head_stride}, {c->page_size, c->row_stride}};
    for (auto &d : dim) {
        if (d.n == 1) d.stride = 0;  // never multiplied by anything but 0
        if (d.stride < 0 || d.stride >= (1ll << 38)) return DMM_ERR_SHAPE;
        if (d.stride % 8 != 0) return DMM_ERR_ALIGN;
    }
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (dim[j].stride < dim[i].stride) {
                const auto t = dim[i];
                dim[i] = dim[j];
                dim[j] = t;
            }
    long long span = c->head_dim;
    for (const auto &d : dim) {
        if (d.n == 1) continue;
        if (d.stride < span) return DMM_ERR_SHAPE;
        if (d.n > (1ll << 60) / d.stride) return DMM_ERR_SHAPE;
        span = d.stride * (d.n - 1) + span;
    }
    view->k = c->k;
    view->v = c->v;
    view->page_table = c->page_table;
    view->seq_lens = c->seq_lens;
    view->page_stride = c->page_stride;
    view->head_stride = c->head_stride;
    view->row_stride = c->row_stride;
    view->table_stride = c->table_stride;
    view->num_pages = static_cast<int>(c->num_pages);
    view->kv_heads = c->kv_heads;
    view->page_shift = __builtin_ctz(static_cast<unsigned>(c->page_size));
    view->num_seqs = c->num_seqs;
    view->max_pages = c->max_pages;
    return 0;
}

static int check_rows(const void *p, long long ld, long long width) {
    if (!p) return DMM_ERR_NULL;
    if (!aligned16(p)) return DMM_ERR_ALIGN;
    if (ld < width || ld >= (1ll << 38)) return DMM_ERR_SHAPE;
    return ld % 8 != 0 ? DMM_ERR_ALIGN : 0;
}

// What both attention entries check.
static int check_attention(const void *q, int64_t q_ld, int64_t tokens, int heads, const void *out, int64_t out_ld,
                           const dmm_paged_cache *cache, CacheView *view, const void *workspace, size_t workspace_bytes, unsigned flags) {
    int rc = cache_view(cache, view);
    if (rc) return rc;
    if (heads < 1 || heads % cache->kv_heads != 0 || heads / cache->kv_heads > 128) return DMM_ERR_SHAPE;
    if (tokens < 1 || tokens > 0x7fffffff || heads > 65535) return DMM_ERR_SHAPE;
    const long long width = static_cast<long long>(heads) * cache->head_dim;
    rc = check_rows(q, q_ld, width);
    if (rc) return rc;
    rc = check_rows(out, out_ld, width);
    if (rc) return rc;
    if (flags & ~DMM_FLAG_PDL) return DMM_ERR_ARG;
    const size_t need = dmm_attention_workspace_bytes(tokens, cache->num_seqs, heads, cache->kv_heads, cache->head_dim);
    if (workspace == nullptr || workspace_bytes < need) return DMM_ERR_WORKSPACE;
    return reinterpret_cast<uintptr_t>(workspace) % 256 != 0 ? DMM_ERR_ALIGN : 0;
}

}  // namespace dmm

using namespace dmm;

extern "C" {

int dmm_append_kv(const void *qkv, int qkv_type, int64_t qkv_ld, int64_t tokens, int heads, const double *freqs,
                  int interleaved, void *q_out, int64_t q_ld, const dmm_paged_cache *cache, const int32_t *cu_seqlens,
                  unsigned flags, void *stream) {
    AppendParams p = {};
    int rc = cache_view(cache, &p.cache);
    if (rc) return rc;
    if (qkv_type != DMM_T_F32 && qkv_type != DMM_T_F16 && qkv_type != DMM_T_BF16) return DMM_ERR_ARG;
    if (flags & ~DMM_FLAG_PDL) return DMM_ERR_ARG;
    if (heads < 1 || heads > 65535 || tokens < 1 || tokens > 0x7fffffff) return DMM_ERR_SHAPE;
    if (!cu_seqlens && tokens != cache->num_seqs) return DMM_ERR_SHAPE;
    rc = check_rows(qkv, qkv_ld, (heads + 2ll * cache->kv_heads) * cache->head_dim);
    if (rc) return rc;
    rc = check_rows(q_out, q_ld, static_cast<long long>(heads) * cache->head_dim);
    if (rc) return rc;
    int sms = 0;
    rc = device_sms(&sms);
    if (rc) return rc;
    p.qkv = qkv;
    p.freqs = freqs;
    p.q_out = q_out;
    p.cu = cu_seqlens;
    p.qkv_ld = qkv_ld;
    p.q_ld = q_ld;
    p.tokens = static_cast<int>(tokens);
    p.heads = heads;
    p.interleaved = interleaved ? 1 : 0;
    const bool pdl = (flags & DMM_FLAG_PDL) != 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    g_launches.fetch_add(1, std::memory_order_relaxed);
    if (cache->type == DMM_T_F16)
        return cache->head_dim == 64 ? launch_append<__half, 64>(p, qkv_type, sms, pdl, st) : launch_append<__half, 128>(p, qkv_type, sms, pdl, st);
    return cache->head_dim == 64 ? launch_append<__nv_bfloat16, 64>(p, qkv_type, sms, pdl, st)
                                 : launch_append<__nv_bfloat16, 128>(p, qkv_type, sms, pdl, st);
}

size_t dmm_attention_workspace_bytes(int64_t tokens, int num_seqs, int heads, int kv_heads, int head_dim) {
    (void)tokens, (void)num_seqs, (void)heads, (void)kv_heads;
    int sms = 0;
    if (device_sms(&sms) != 0 || sms < 1) sms = 256;
    const size_t decode = decode_workspace(head_dim, sms), prompt = prompt_workspace(head_dim, sms);
    return decode > prompt ? decode : prompt;
}

int dmm_paged_attention(const void *q, int64_t q_ld, int heads, float scale, void *out, int64_t out_ld,
                        const dmm_paged_cache *cache, void *workspace, size_t workspace_bytes, unsigned flags, void *stream) {
    if (!cache) return DMM_ERR_NULL;
    DecodeParams p = {};
    int rc = check_attention(q, q_ld, cache->num_seqs, heads, out, out_ld, cache, &p.cache, workspace, workspace_bytes, flags);
    if (rc) return rc;
    int sms = 0;
    rc = device_sms(&sms);
    if (rc) return rc;
    p.q = q;
    p.out = out;
    p.partial = static_cast<float *>(workspace);
    p.q_ld = q_ld;
    p.out_ld = out_ld;
    p.group = heads / cache->kv_heads;
    p.scale = scale;
    const bool pdl = (flags & DMM_FLAG_PDL) != 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    g_launches.fetch_add(2, std::memory_order_relaxed);
    if (cache->type == DMM_T_F16)
        return cache->head_dim == 64 ? launch_decode<__half, 64>(p, sms, pdl, st) : launch_decode<__half, 128>(p, sms, pdl, st);
    return cache->head_dim == 64 ? launch_decode<__nv_bfloat16, 64>(p, sms, pdl, st) : launch_decode<__nv_bfloat16, 128>(p, sms, pdl, st);
}

int dmm_prompt_attention(const void *q, int64_t q_ld, int64_t tokens, int heads, float scale, void *out, int64_t out_ld,
                         const dmm_paged_cache *cache, const int32_t *cu_seqlens, void *workspace,
                         size_t workspace_bytes, unsigned flags, void *stream) {
    if (!cu_seqlens) return DMM_ERR_NULL;
    PromptParams p = {};
    int rc = check_attention(q, q_ld, tokens, heads, out, out_ld, cache, &p.cache, workspace, workspace_bytes, flags);
    if (rc) return rc;
    rc = device_sms(&p.ctas);
    if (rc) return rc;
    p.workspace = static_cast<uint8_t *>(workspace);
    p.q = q;
    p.out = out;
    p.cu = cu_seqlens;
    p.q_ld = q_ld;
    p.out_ld = out_ld;
    p.tokens = static_cast<int>(tokens);
    p.heads = heads;
    p.group = heads / cache->kv_heads;
    p.scale = scale;
    g_launches.fetch_add(2, std::memory_order_relaxed);
    return launch_prompt(p, cache->type, cache->head_dim, (flags & DMM_FLAG_PDL) != 0, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
