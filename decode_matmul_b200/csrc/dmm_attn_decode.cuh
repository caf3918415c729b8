// Attention of one new token per sequence over a paged cache.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = exp2(c q . k_j - m), c = scale log2(e): every key and value is read once and used
// for the few query heads that share it, so the cache's bytes are the bound.
//
// The work is cut into units of 16 keys of one (sequence, key head), a segment being all units of one; the units of all
// segments in one line are divided evenly, first among the CTAs, one per SM, then among a CTA's eight warps.  A
// warp streams its units through a ring of its own in shared memory (cp.async, a page never ends inside a unit), and works
// on warp-level tensor cores: S[16 queries, 16 keys] = Q K^T, P V with the fragments of S as operands.  With
// group <= 8 half of the 16 rows is idle, which costs nothing: the multiplications take a fifth of the time of the bytes.
// No barrier until a warp has finished.  A segment that a warp has whole is written out by it.  What several warps have of
// one segment is joined through shared memory, what several CTAs have through the workspace by a second kernel: always in the
// order of the keys, so that results do not depend on who comes first.
// The running maximum only moves when it has risen by more than 8 (weights then stay below 2^8).
#pragma once

#include "dmm_attn_common.cuh"
#include "dmm_tmem.cuh"

namespace dmm {

constexpr int kDecodeWarps = 8;
constexpr int kUnitKeys = 16;

struct DecodeParams {
    const void *q;
    void *out;
    float *partial;  // [2 * CTAs][16][D], then [2 * CTAs][16][2]: maximum and sum
    long long q_ld, out_ld;
    CacheView cache;
    int group, q_tiles;  // q_tiles: of 16 query heads that share a key head
    float scale;
};

// A part of a segment: weighted sums of values (rows padded against bank conflicts), then maximum and sum of each row.
template <int D, int kRows>
struct DecodePlan {
    static constexpr int kStages = (D == 128 ? 3 : 6) - (kRows == 2 ? D == 128 ? 1 : 2 : 0);
    static constexpr uint32_t kRowBytes = 2 * D;
    static constexpr uint32_t kUnitBytes = kUnitKeys * kRowBytes;  // of K, and again of V
    static constexpr uint32_t kWarpBytes = kStages * 2 * kUnitBytes;
    static constexpr int kPad = D + 4;
    static constexpr int kPartFloats = 8 * kRows * (kPad + 2);
    // the rings, and a part per warp beside them; a warp's last part takes the place of its ring
    static constexpr uint32_t kParts = kDecodeWarps * kWarpBytes;
    static constexpr uint32_t kBytes = kParts + kDecodeWarps * kPartFloats * 4;
    static_assert(kPartFloats * 4 <= kWarpBytes, "a part fits into a ring");
    static_assert(kBytes <= 227 * 1024 - 1024, "shared memory");
};

inline size_t decode_workspace(int head_dim, int ctas) { return static_cast<size_t>(ctas) * 2 * 16 * (head_dim + 2) * sizeof(float); }

// Where a unit lies: segment (seq, head, with head counting the tiles of 16 queries too), unit within it, and the segment's
// length.  A sequence without keys has one unit, without keys.
struct DecodeAt {
    long long start;  // unit number of the segment's first
    int seq, head, unit, units, len;
};
__device__ __forceinline__ int units_of(int len) { return len > 0 ? (len + kUnitKeys - 1) / kUnitKeys : 1; }

// Units of all sequences, and the place of unit `u` of them.  By the lanes of a warp.
__device__ __forceinline__ long long decode_units(const CacheView &c, int heads) {
    const int lane = threadIdx.x & 31;
    long long sum = 0;
    for (int b = lane; b < c.num_seqs; b += 32) sum += units_of(cache_len(c, b));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum * heads;
}
__device__ __forceinline__ DecodeAt decode_at(const CacheView &c, int heads, long long u) {
    const int lane = threadIdx.x & 31;
    DecodeAt at = {0, 0, 0, 0, 1, 0};
    long long before = 0;
    for (int b0 = 0; b0 < c.num_seqs; b0 += 32) {
        const int b = b0 + lane, len = b < c.num_seqs ? cache_len(c, b) : 0;
        const long long mine = b < c.num_seqs ? static_cast<long long>(units_of(len)) * heads : 0;
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned after = __ballot_sync(0xffffffffu, before + upto > u);
        if (after != 0) {
            const int who = __ffs(after) - 1;
            at.seq = b0 + who;
            at.len = __shfl_sync(0xffffffffu, len, who);
            at.units = units_of(at.len);
            const long long first = before + __shfl_sync(0xffffffffu, upto - mine, who);
            at.head = static_cast<int>((u - first) / at.units);
            at.start = first + static_cast<long long>(at.head) * at.units;
            at.unit = static_cast<int>(u - at.start);
            return at;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return at;
}
__device__ __forceinline__ void decode_next(const CacheView &c, int heads, DecodeAt &at) {
    if (++at.unit < at.units) return;
    at.start += at.units;
    at.unit = 0;
    if (++at.head < heads) return;
    at.head = 0;
    if (++at.seq < c.num_seqs) {
        at.len = cache_len(c, at.seq);
        at.units = units_of(at.len);
    }
}

__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void *src, bool have) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(have ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <class T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_f16(c, a[0], a[1], a[2], a[3], b0, b1);
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// What a warp has of one segment when it could not write it out.
struct DecodePart {
    long long start;
    int seq, head, units, have;  // have: units of it that this part covers, 0 = no part
};

// kRows: 1 for groups of up to 8 query heads, 2 for up to 16 (rows lane / 4 and lane / 4 + 8 of a fragment)
template <class T, int D, int kRows>
__global__ void __launch_bounds__(32 * kDecodeWarps, 1) paged_attention_kernel(const DecodeParams p) {
    using Plan = DecodePlan<D, kRows>;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    __shared__ DecodePart s_part[2 * kDecodeWarps];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, quad = lane / 4, pair = lane % 4;
    const uint32_t smem = smem_u32(smem_raw);
    grid_dep_wait();
    grid_dep_launch();  // the kernel that joins the CTAs' parts may take its place; it waits for this one's end
    const int heads = p.cache.kv_heads * p.q_tiles;
    const long long all = decode_units(p.cache, heads);
    const long long c0 = part_begin(all, gridDim.x, blockIdx.x), c1 = part_begin(all, gridDim.x, blockIdx.x + 1);
    const long long u0 = c0 + (c1 - c0) * warp / kDecodeWarps, u1 = c0 + (c1 - c0) * (warp + 1) / kDecodeWarps;
    if (lane < 2) s_part[2 * warp + lane].have = 0;
    __syncwarp();

    const uint32_t ring = smem + warp * Plan::kWarpBytes;
    // pieces of 16 bytes: a row has D / 8 of them, piece c of row r lies at c ^ (r % 8), so that eight rows' same piece is conflict free
    constexpr int kPieces = D / 8, kRowsAtOnce = 32 / kPieces;
    const int piece = lane % kPieces, row0 = lane / kPieces;

    float o[D / 8][4], m[2], l[2];
    uint32_t qf[D / 16][4];
    const float c = p.scale * 1.4426950408889634f;
    float *const first_part = reinterpret_cast<float *>(smem_raw + Plan::kParts) + warp * Plan::kPartFloats;
    float *const last_part = reinterpret_cast<float *>(smem_raw + warp * Plan::kWarpBytes);

    DecodeAt load = {}, at = {};
    int page = 0;
    const auto fetch_page = [&](const DecodeAt &w) {
        return w.len > 0 ? p.cache.page_table[w.seq * p.cache.table_stride + ((w.unit * kUnitKeys) >> p.cache.page_shift)] : -1;
    };
    const auto issue = [&](int stage) {
        const int pos = load.unit * kUnitKeys, keys = load.len - pos;
        bool there = keys > 0;
        if (there && (page < 0 || page >= p.cache.num_pages)) {
            raise_status(DMM_STATUS_BAD_PAGE);
            there = false;
        }
        const long long base = there ? page * p.cache.page_stride + (load.head / p.q_tiles) * p.cache.head_stride +
                                           (pos & ((1 << p.cache.page_shift) - 1)) * p.cache.row_stride
                                     : 0;
        const T *k = static_cast<const T *>(p.cache.k) + base + piece * 8, *v = static_cast<const T *>(p.cache.v) + base + piece * 8;
        const uint32_t dst = ring + stage * 2 * Plan::kUnitBytes;
#pragma unroll
        for (int r = row0; r < kUnitKeys; r += kRowsAtOnce) {
            const bool have = there && r < keys;
            const uint32_t d = dst + r * Plan::kRowBytes + ((piece ^ (r & 7)) << 4);
            const long long off = have ? r * p.cache.row_stride : 0;
            cp_async16_or_zero(d, k + off, have);
            cp_async16_or_zero(d + Plan::kUnitBytes, v + off, have);
        }
    };

    if (u0 < u1) {
        at = decode_at(p.cache, heads, u0);
        load = at;
        long long ahead = u0;  // the next unit to load
        page = fetch_page(load);
#pragma unroll
        for (int s = 0; s < Plan::kStages - 1; ++s) {
            if (ahead < u1) {
                issue(s);
                if (++ahead < u1) {
                    decode_next(p.cache, heads, load);
                    page = fetch_page(load);
                }
            }
            cp_async_commit();
        }
        int stage = 0;
        bool fresh = true;
        int have = 0;
        for (long long u = u0; u < u1; ++u) {
            if (fresh) {
                const T *q = static_cast<const T *>(p.q) + at.seq * p.q_ld + static_cast<long long>(at.head / p.q_tiles) * p.group * D;
                const int r0 = (at.head % p.q_tiles) * 16 + quad;
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        qf[k][2 * h] = r0 < p.group ? *reinterpret_cast<const uint32_t *>(q + r0 * D + 16 * k + 8 * h + 2 * pair) : 0u;
                        qf[k][2 * h + 1] = kRows == 2 && r0 + 8 < p.group ? *reinterpret_cast<const uint32_t *>(q + (r0 + 8) * D + 16 * k + 8 * h + 2 * pair) : 0u;
                    }
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[n][x] = 0.0f;
                m[0] = m[1] = -INFINITY;
                l[0] = l[1] = 0.0f;
                fresh = false;
                have = 0;
            }
            cp_async_wait<Plan::kStages - 2>();
            __syncwarp();  // all lanes' pieces of this unit are there, and all have read the unit before
            if (ahead < u1) {
                issue(stage == 0 ? Plan::kStages - 1 : stage - 1);
                if (++ahead < u1) {
                    decode_next(p.cache, heads, load);
                    page = fetch_page(load);
                }
            }
            cp_async_commit();

            const uint32_t kb = ring + stage * 2 * Plan::kUnitBytes, vb = kb + Plan::kUnitBytes;
            float s[2][4] = {};
            {
                const int r = (lane / 16) * 8 + lane % 8, half = (lane / 8) % 2;
                const uint32_t row = kb + r * Plan::kRowBytes;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    uint32_t b[4];
                    ldsm4(row + (((2 * k + half) ^ (r & 7)) << 4), b);
                    mma16<T>(s[0], qf[k], b[0], b[1]);
                    mma16<T>(s[1], qf[k], b[2], b[3]);
                }
            }
            const int keys = at.len - at.unit * kUnitKeys;
            uint32_t pf[4] = {};
            float top[kRows];
#pragma unroll
            for (int h = 0; h < kRows; ++h) {
                top[h] = -INFINITY;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float &v = s[n][2 * h + x];
                        v = 8 * n + 2 * pair + x < keys ? v * c : -INFINITY;
                        top[h] = fmaxf(top[h], v);
                    }
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
            }
            bool rise = false;
#pragma unroll
            for (int h = 0; h < kRows; ++h) rise |= top[h] > m[h] + 8.0f;
            if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
                for (int h = 0; h < kRows; ++h) {
                    const float to = fmaxf(m[h], top[h]), f = m[h] == -INFINITY ? 0.0f : exp2_fast(m[h] - to);
                    m[h] = to;
                    l[h] *= f;
#pragma unroll
                    for (int n = 0; n < D / 8; ++n) {
                        o[n][2 * h] *= f;
                        o[n][2 * h + 1] *= f;
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < kRows; ++h) {
                const float mm = m[h] == -INFINITY ? 0.0f : m[h];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float a = exp2_fast(s[n][2 * h] - mm), b = exp2_fast(s[n][2 * h + 1] - mm);
                    l[h] += a + b;
                    pf[2 * n + h] = pack16<T>(a, b);
                }
            }
            {
                const int r = ((lane / 8) % 2) * 8 + lane % 8, half = lane / 16;
                const uint32_t row = vb + r * Plan::kRowBytes;
#pragma unroll
                for (int n = 0; n < D / 16; ++n) {
                    uint32_t b[4];
                    ldsm4_trans(row + (((2 * n + half) ^ (r & 7)) << 4), b);
                    mma16<T>(o[2 * n], pf, b[0], b[1]);
                    mma16<T>(o[2 * n + 1], pf, b[2], b[3]);
                }
            }
            if (++stage == Plan::kStages) stage = 0;
            ++have;

            if (at.unit + 1 == at.units || u + 1 == u1) {  // the end of the segment or of this warp's share
#pragma unroll
                for (int h = 0; h < kRows; ++h) {
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                }
                const int r0 = (at.head % p.q_tiles) * 16 + quad;
                if (have == at.units) {
                    T *out = static_cast<T *>(p.out) + at.seq * p.out_ld + static_cast<long long>(at.head / p.q_tiles) * p.group * D;
#pragma unroll
                    for (int h = 0; h < kRows; ++h) {
                        if (r0 + 8 * h >= p.group) continue;
                        const float inv = at.len > 0 ? 1.0f / l[h] : 0.0f;
#pragma unroll
                        for (int n = 0; n < D / 8; ++n)
                            *reinterpret_cast<uint32_t *>(out + (r0 + 8 * h) * D + 8 * n + 2 * pair) = pack16<T>(o[n][2 * h] * inv, o[n][2 * h + 1] * inv);
                    }
                } else {
                    const int which = u + 1 < u1 ? 0 : 1;
                    float *part = which == 0 ? first_part : last_part;
                    __syncwarp();  // (the last part lies where all lanes have read the last unit)
#pragma unroll
                    for (int h = 0; h < kRows; ++h) {
                        const int row = quad + 8 * h;
#pragma unroll
                        for (int n = 0; n < D / 8; ++n)
                            *reinterpret_cast<float2 *>(part + row * Plan::kPad + 8 * n + 2 * pair) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
                        if (pair == 0) *reinterpret_cast<float2 *>(part + 8 * kRows * Plan::kPad + 2 * row) = make_float2(m[h], l[h]);
                    }
                    if (lane == 0) s_part[2 * warp + which] = {at.start, at.seq, at.head, at.units, have};
                }
                fresh = true;
            }
            decode_next(p.cache, heads, at);
        }
    }
    cp_async_wait<0>();
    __syncthreads();
    // Parts of one segment lie next to each other in the warps' order: a warp joins the parts of every eighth segment.
    int nth = 0;
    for (int i = 0; i < 2 * kDecodeWarps;) {
        if (s_part[i].have == 0) {
            ++i;
            continue;
        }
        const DecodePart of = s_part[i];
        int end = i + 1, have = of.have;
        while (end < 2 * kDecodeWarps && (s_part[end].have == 0 || s_part[end].start == of.start)) have += s_part[end++].have;
        if (nth++ % kDecodeWarps == warp) {
            constexpr int kC = D / 32;  // columns of a lane
            const auto part_of = [&](int x) {
                return x % 2 == 0 ? reinterpret_cast<const float *>(smem_raw + Plan::kParts) + x / 2 * Plan::kPartFloats
                                  : reinterpret_cast<const float *>(smem_raw + x / 2 * Plan::kWarpBytes);
            };
            for (int row = 0; row < 8 * kRows; ++row) {
                const int r = (of.head % p.q_tiles) * 16 + row;
                if (r >= p.group) break;
                float top = -INFINITY, sum = 0.0f, acc[kC] = {};
                for (int x = i; x < end; ++x)
                    if (s_part[x].have > 0) top = fmaxf(top, part_of(x)[8 * kRows * Plan::kPad + 2 * row]);
                for (int x = i; x < end; ++x) {
                    if (s_part[x].have == 0) continue;
                    const float *part = part_of(x);
                    const float mx = part[8 * kRows * Plan::kPad + 2 * row], w = mx == -INFINITY ? 0.0f : exp2_fast(mx - top);
                    sum += w * part[8 * kRows * Plan::kPad + 2 * row + 1];
#pragma unroll
                    for (int y = 0; y < kC; ++y) acc[y] += w * part[row * Plan::kPad + kC * lane + y];
                }
                if (have == of.units) {
                    T *out = static_cast<T *>(p.out) + of.seq * p.out_ld + (static_cast<long long>(of.head / p.q_tiles) * p.group + r) * D + kC * lane;
                    const float inv = 1.0f / sum;
#pragma unroll
                    for (int y = 0; y < kC; y += 2) *reinterpret_cast<uint32_t *>(out + y) = pack16<T>(acc[y] * inv, acc[y + 1] * inv);
                } else {  // a CTA has at most one segment that began before it, and one that goes on behind it
                    const int slot = 2 * blockIdx.x + (of.start < c0 ? 0 : 1);
                    float *to = p.partial + (static_cast<size_t>(slot) * 16 + row) * D + kC * lane;
#pragma unroll
                    for (int y = 0; y < kC; ++y) to[y] = acc[y];
                    if (lane == 0)
                        *reinterpret_cast<float2 *>(p.partial + static_cast<size_t>(gridDim.x) * 2 * 16 * D + 2 * (slot * 16 + row)) = make_float2(top, sum);
                }
            }
        }
        i = end;
    }
}

// Joins what several CTAs have of one segment.  Block (x, row): the segment that crosses from CTA x to the next, if x is the first
// CTA that has a part of it.  Warps take the parts in turn, in the order of the keys.
template <class T, int D>
__global__ void __launch_bounds__(32 * kDecodeWarps) paged_join_kernel(const DecodeParams p, int ctas) {
    __shared__ float s_w[1024], s_acc[kDecodeWarps][D], s_red[kDecodeWarps];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, row = blockIdx.y;
    const int heads = p.cache.kv_heads * p.q_tiles;
    // (lengths are older than the kernel in front, which has waited for them)
    const long long all = decode_units(p.cache, heads);
    const long long c0 = part_begin(all, ctas, blockIdx.x), c1 = part_begin(all, ctas, blockIdx.x + 1);
    bool work = c0 < c1 && c1 < all;
    DecodeAt at = {};
    int r = 0;
    if (work) {
        at = decode_at(p.cache, heads, c1);
        r = (at.head % p.q_tiles) * 16 + row;
        work = at.unit > 0 && at.start >= c0 && r < p.group;
    }
    grid_dep_wait();
    if (!work) return;
    const int last = static_cast<int>(part_owner(all, ctas, at.start + at.units - 1)), n = last - static_cast<int>(blockIdx.x) + 1;
    const float *ml = p.partial + static_cast<size_t>(ctas) * 2 * 16 * D;
    const auto slot_of = [&](int x) { return 2 * (static_cast<int>(blockIdx.x) + x) + (at.start < part_begin(all, ctas, blockIdx.x + x) ? 0 : 1); };
    const auto empty = [&](int x) { return part_begin(all, ctas, blockIdx.x + x) == part_begin(all, ctas, blockIdx.x + x + 1); };
    float top = -INFINITY;
    for (int x = threadIdx.x; x < n; x += 32 * kDecodeWarps)
        if (!empty(x)) top = fmaxf(top, ml[2 * (slot_of(x) * 16 + row)]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) s_red[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) top = fmaxf(top, s_red[w]);
    __syncthreads();
    float sum = 0.0f;
    for (int x = threadIdx.x; x < n; x += 32 * kDecodeWarps) {
        const float2 v = empty(x) ? make_float2(-INFINITY, 0.0f) : *reinterpret_cast<const float2 *>(ml + 2 * (slot_of(x) * 16 + row));
        const float w = v.x == -INFINITY ? 0.0f : exp2_fast(v.x - top);
        s_w[x] = w;
        sum += w * v.y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_red[warp] = sum;
    __syncthreads();
    constexpr int kC = D / 32;
    float acc[kC] = {};
#pragma unroll 4
    for (int x = warp; x < n; x += kDecodeWarps) {
        const float w = s_w[x];
        if (empty(x)) continue;
        const float *from = p.partial + (static_cast<size_t>(slot_of(x)) * 16 + row) * D + kC * lane;
#pragma unroll
        for (int y = 0; y < kC; ++y) acc[y] += w * from[y];
    }
#pragma unroll
    for (int y = 0; y < kC; ++y) s_acc[warp][kC * lane + y] = acc[y];
    __syncthreads();
    if (threadIdx.x < D / 2) {
        float a = 0.0f, b = 0.0f, all_sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kDecodeWarps; ++w) {
            a += s_acc[w][2 * threadIdx.x];
            b += s_acc[w][2 * threadIdx.x + 1];
            all_sum += s_red[w];
        }
        T *out = static_cast<T *>(p.out) + at.seq * p.out_ld + (static_cast<long long>(at.head / p.q_tiles) * p.group + r) * D;
        *reinterpret_cast<uint32_t *>(out + 2 * threadIdx.x) = pack16<T>(a / all_sum, b / all_sum);
    }
}

template <class T, int D, int kRows>
inline int launch_decode_typed(const DecodeParams &p, int ctas, bool pdl, cudaStream_t stream) {
    using Plan = DecodePlan<D, kRows>;
    const auto kernel = paged_attention_kernel<T, D, kRows>;
    static SmemAllowance allowance;
    const int rc = allowance.get(reinterpret_cast<const void *>(kernel), Plan::kBytes);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(32 * kDecodeWarps);
    cfg.dynamicSmemBytes = Plan::kBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, p);
    if (err != cudaSuccess) return err;
    cfg.gridDim = dim3(static_cast<unsigned>(ctas - 1), static_cast<unsigned>(p.group < 16 ? p.group : 16));
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_join_kernel<T, D>, p, ctas);
}

template <class T, int D>
inline int launch_decode(const DecodeParams &p, int ctas, bool pdl, cudaStream_t stream) {
    return p.group <= 8 ? launch_decode_typed<T, D, 1>(p, ctas, pdl, stream) : launch_decode_typed<T, D, 2>(p, ctas, pdl, stream);
}

}  // namespace dmm
