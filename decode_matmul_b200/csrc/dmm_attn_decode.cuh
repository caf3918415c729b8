// Attention of one new token per sequence over a paged cache.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = 2^(c q . k_j - m), c = scale log2(e): every key and value is read once and used
// for the few query heads that share it, so the cache's bytes are the bound.
//
// The work is cut into units of 16 keys of one (sequence, key head, tile of queries), a segment being all units of one; the
// units of all segments in one line are divided evenly, first among the CTAs, one per SM, then among a CTA's eight
// warps.  A warp streams its units through a ring of its own in shared memory (cp.async; a page never ends inside a unit) and
// works on warp-level tensor cores with the keys as the 16 rows and 8 queries as the columns: S^T[16, 8] = K Q^T and
// O^T[D, 8] += V^T P^T, where P^T is S^T transposed in registers.  (Queries as rows would leave half of them idle
// and take twice the registers.)  Groups of more than 8 query heads have two such column tiles, of more than 16 several tiles
// that read the keys again.
// No barrier until a warp has finished.  A segment that a warp has whole is written out by it.  What several warps have of
// one segment is joined through shared memory, what several CTAs have through the workspace by a second kernel: always in the
// order of the keys, so that results do not depend on who comes first.
// The running maximum only moves when it has risen by more than 8 (weights then stay below 2^8; 2^15 in fp16, see kRaise).  Weights are rounded to
// the type of the values, as the tensor cores take them: half a step each, in no common direction, which the sum over the keys evens out.
// Scores, maxima and sums are fp32, the sum of weights that are not rounded.
//
// Bound: bytes, 4 head_dim for every token and key head.  Two units of 8 KB in flight beside the present one for each of 8 warps keep 128 KB
// under way on every SM, more than HBM's latency asks for.  B200, graph, fp16, heads of 128: 32 sequences with 32 key heads, 405 MB, 72 us (5.6 TB/s,
// 86 % of what a copy reaches); 16 sequences of 64 heads on 8, 84 MB, 24.2 us; one sequence of 4096, 17 MB, 11.6 us (9.8 from L2).  What is not
// bytes is 8 to 10 us a call: lengths, page numbers and keys are dependent loads, the parts are joined twice, and two kernels start.
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
    int group, q_tiles;  // q_tiles: of 8 kN query heads that share a key head
    float scale;
};

// kN: column tiles of 8 queries.
template <int D, int kN>
struct DecodePlan {
    static constexpr int kStages = (D == 128 ? 3 : 5) - (kN == 2 ? 1 : 0);
    static constexpr uint32_t kRowBytes = 2 * D;
    static constexpr uint32_t kUnitBytes = kUnitKeys * kRowBytes;  // of K, and again of V
    static constexpr uint32_t kWarpBytes = kStages * 2 * kUnitBytes;
    // A part of a segment: weighted sums of values (a row per query, padded against bank conflicts), then maximum and sum of each.
    static constexpr int kRows = 8 * kN, kPad = D + 4;
    static constexpr int kPartFloats = kRows * (kPad + 2);
    // The rings, and beside them the queries of the units under way, which may be as many segments (the present one's are in registers); a
    // warp's last part takes the place of its ring.
    static constexpr int kQPlaces = kStages > 2 ? kStages - 1 : 2;
    static constexpr uint32_t kQBytes = kRows * kRowBytes;
    static constexpr uint32_t kQ = kDecodeWarps * kWarpBytes;
    static constexpr uint32_t kBytes = kQ + kDecodeWarps * kQPlaces * kQBytes;
    static_assert(kPartFloats * 4 <= kWarpBytes, "a part fits into a ring");
    static_assert(kBytes <= 227 * 1024 - 1024, "shared memory");
};

// Workspace: what CTAs have of segments that they share, [2 * CTAs][16][D] and [2 * CTAs][16][2] floats, one description of such a
// segment per CTA, and behind it what a warp has of the segment that began before its share, until its CTA joins it.
inline __host__ __device__ size_t decode_shared_floats(int head_dim, int ctas) { return static_cast<size_t>(ctas) * 2 * 16 * (head_dim + 2); }
inline size_t decode_workspace(int head_dim, int ctas) {
    return (decode_shared_floats(head_dim, ctas) + static_cast<size_t>(ctas) * (4 + kDecodeWarps * 16 * (head_dim + 6))) * sizeof(float);
}

__device__ __forceinline__ int units_of(int len) { return len > 0 ? (len + kUnitKeys - 1) / kUnitKeys : 1; }

// `all` units over `ctas` CTAs: CTA x has [begin(x), begin(x + 1)), the first `more` of them one unit more than the others.
struct DecodeShare {
    long long all, each;
    int more;
    __device__ __forceinline__ long long begin(int x) const { return each * x + min(x, more); }
    __device__ __forceinline__ int owner(long long u) const;
};
// a / b for numbers that nearly always fit into 32 bits (a division of 64 bits takes half a microsecond)
__device__ __forceinline__ long long quotient(long long a, long long b) {
    if (((a | b) >> 32) == 0) return static_cast<unsigned>(a) / static_cast<unsigned>(b);
    return a / b;
}
__device__ __forceinline__ int DecodeShare::owner(long long u) const {
    const long long big = (each + 1) * more;
    return static_cast<int>(u < big ? quotient(u, each + 1) : more + quotient(u - big, each));
}
// Where a unit lies: the segment (sequence, key head, tile of its queries), its length, its first unit's number and the unit in it.
struct DecodeAt {
    long long start;
    int seq, head, tile, unit, units, len;
};

// Lengths and units of 32 sequences from b0 on, one per lane, and the running sum of the units.  A sequence without keys has one unit,
// without keys; 32 sequences have less than 2^32.
struct DecodeLens {
    int len;
    unsigned mine, upto;
    __device__ __forceinline__ DecodeLens(const CacheView &c, int b0) {
        const int lane = threadIdx.x & 31, b = b0 + lane;
        len = b < c.num_seqs ? cache_len(c, b) : 0;
        mine = b < c.num_seqs ? static_cast<unsigned>(units_of(len)) : 0u;
        upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
    }
    __device__ __forceinline__ unsigned sum() const { return __shfl_sync(0xffffffffu, upto, 31); }
};
// All by the lanes of a warp; `first` are the lengths from sequence 0 on.
__device__ __forceinline__ DecodeShare decode_share(const CacheView &c, const DecodeLens &first, int heads, int ctas) {
    long long sum = first.sum();
    for (int b0 = 32; b0 < c.num_seqs; b0 += 32) sum += DecodeLens(c, b0).sum();
    DecodeShare s;
    s.all = sum * heads;
    s.each = quotient(s.all, ctas);
    s.more = static_cast<int>(s.all - s.each * ctas);
    return s;
}
// The place of unit u.
__device__ __forceinline__ DecodeAt decode_at(const CacheView &c, DecodeLens lens, int q_tiles, long long u) {
    const int heads = c.kv_heads * q_tiles;
    DecodeAt at = {0, 0, 0, 0, 0, 1, 0};
    long long before = 0;
    for (int b0 = 0;;) {
        const unsigned after = __ballot_sync(0xffffffffu, before + static_cast<long long>(lens.upto) * heads > u);
        if (after != 0) {
            const int who = __ffs(after) - 1;
            at.seq = b0 + who;
            at.len = __shfl_sync(0xffffffffu, lens.len, who);
            at.units = units_of(at.len);
            const long long first = before + static_cast<long long>(__shfl_sync(0xffffffffu, lens.upto - lens.mine, who)) * heads;
            const int segment = static_cast<int>(quotient(u - first, at.units));
            at.head = q_tiles == 1 ? segment : segment / q_tiles;
            at.tile = segment - at.head * q_tiles;
            at.start = first + static_cast<long long>(segment) * at.units;
            at.unit = static_cast<int>(u - at.start);
            return at;
        }
        before += static_cast<long long>(lens.sum()) * heads;
        b0 += 32;
        if (b0 >= c.num_seqs) return at;
        lens = DecodeLens(c, b0);
    }
}
// The next unit; true when it is of another segment.
__device__ __forceinline__ bool decode_next(const CacheView &c, int q_tiles, DecodeAt &at) {
    if (++at.unit < at.units) return false;
    at.start += at.units;
    at.unit = 0;
    if (++at.tile < q_tiles) return true;
    at.tile = 0;
    if (++at.head < c.kv_heads) return true;
    at.head = 0;
    if (++at.seq < c.num_seqs) {
        at.len = cache_len(c, at.seq);
        at.units = units_of(at.len);
    }
    return true;
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
// An 8 x 8 tile of 16-bit values that a warp holds as a fragment, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t w) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
    return r;
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

// Of a sum of weights: 0 where there is none (no keys, or scores that are all -infinity), so that the result is 0.
__device__ __forceinline__ float decode_inverse(float l) { return l > 0.0f || l != l ? 1.0f / l : 0.0f; }

// What a warp has of one segment when it could not write it out.
struct DecodePart {
    long long start;
    int seq, head, tile, units, have;  // have: units of it that this part covers, 0 = no part
};
// The segment that begins in a CTA and goes on in others: what the join needs to know.
struct DecodeCrossing {
    int seq, head, tile, ctas;  // ctas: how many have a part of it, 0 = there is no such segment
};
__device__ __forceinline__ DecodeCrossing *decode_crossings(float *partial, int head_dim, int ctas) {
    return reinterpret_cast<DecodeCrossing *>(partial + decode_shared_floats(head_dim, ctas));
}

template <class T, int D, int kN>
__global__ void __launch_bounds__(32 * kDecodeWarps, 1) paged_attention_kernel(const DecodeParams p) {
    using Plan = DecodePlan<D, kN>;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    __shared__ DecodePart s_part[2 * kDecodeWarps];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, quad = lane / 4, pair = lane % 4;
    grid_dep_wait();
    grid_dep_launch();  // the kernel that joins the CTAs' parts may come in beside this one; it waits for this one's end
    const DecodeLens lens(p.cache, 0);
    const DecodeShare share = decode_share(p.cache, lens, p.cache.kv_heads * p.q_tiles, gridDim.x);
    const long long c0 = share.begin(blockIdx.x);
    const long long mine = share.begin(blockIdx.x + 1) - c0;
    const long long u0 = c0 + mine * warp / kDecodeWarps, u1 = c0 + mine * (warp + 1) / kDecodeWarps;  // (a power of two)
    // what this warp has of a segment that began before its share and ends within it
    float *const first_parts = p.partial + decode_shared_floats(D, gridDim.x) + 4 * gridDim.x + static_cast<size_t>(blockIdx.x) * kDecodeWarps * Plan::kPartFloats;
    if (lane < 2) s_part[2 * warp + lane].have = 0;
    __syncwarp();

    if (u0 < u1) {
        const uint32_t ring = smem_u32(smem_raw) + warp * Plan::kWarpBytes;
        // pieces of 16 bytes: a row has D / 8 of them, piece c of row r lies at c ^ (r % 8), so that eight rows' same piece is conflict free
        constexpr int kPieces = D / 8, kRowsAtOnce = 32 / kPieces;
        const int piece = lane % kPieces, row0 = lane / kPieces;
        const long long my_offset = row0 * p.cache.row_stride + piece * 8, step = kRowsAtOnce * p.cache.row_stride;
        const float c = p.scale * 1.4426950408889634f;

        DecodeAt at = decode_at(p.cache, lens, p.q_tiles, u0), load = at;
        int left = static_cast<int>(u1 - u0);  // units not yet asked for
        bool fresh_load = true;                // the next of them is the first of its segment
        const int32_t *table = p.cache.page_table + load.seq * p.cache.table_stride;
        int page = load.len > 0 ? table[(load.unit * kUnitKeys) >> p.cache.page_shift] : 0;
        // the queries of a segment come with its first unit here, into the places in turn
        const uint32_t q_place = smem_u32(smem_raw) + Plan::kQ + warp * Plan::kQPlaces * Plan::kQBytes;
        int q_load = 0, q_use = 0;
        const auto issue_q = [&]() {
            const int r0 = load.tile * Plan::kRows;
            const T *q = static_cast<const T *>(p.q) + load.seq * p.q_ld + (static_cast<long long>(load.head) * p.group + r0) * D + piece * 8;
            const uint32_t dst = q_place + q_load * Plan::kQBytes;
            if (++q_load == Plan::kQPlaces) q_load = 0;
#pragma unroll
            for (int i = 0; i < Plan::kRows / kRowsAtOnce; ++i) {
                const int row = row0 + i * kRowsAtOnce;
                const bool have = r0 + row < p.group;
                cp_async16_or_zero(dst + row * Plan::kRowBytes + ((piece ^ (row & 7)) << 4), have ? q + row * D : q, have);
            }
        };
        // asks for the unit at `load`, and goes on to the next, whose page number is then under way
        const auto issue = [&](int stage) {
            if (fresh_load) issue_q();
            const int pos = load.unit * kUnitKeys, keys = load.len - pos;
            const bool there = page >= 0 && page < p.cache.num_pages;
            if (!there) raise_status(DMM_STATUS_BAD_PAGE);
            const long long base = there ? page * p.cache.page_stride + load.head * p.cache.head_stride +
                                               (pos & ((1 << p.cache.page_shift) - 1)) * p.cache.row_stride + my_offset
                                         : 0;
            const T *k = static_cast<const T *>(p.cache.k) + base, *v = static_cast<const T *>(p.cache.v) + base;
            const uint32_t dst = ring + stage * 2 * Plan::kUnitBytes + row0 * Plan::kRowBytes;
            const int rows = there ? keys - row0 : 0;  // what is behind the sequence's end becomes zeros
#pragma unroll
            for (int i = 0; i < kUnitKeys / kRowsAtOnce; ++i) {
                const uint32_t d = dst + i * kRowsAtOnce * Plan::kRowBytes + ((piece ^ ((row0 + i * kRowsAtOnce) & 7)) << 4);
                const bool have = i * kRowsAtOnce < rows;
                cp_async16_or_zero(d, have ? k : static_cast<const T *>(p.cache.k), have);
                cp_async16_or_zero(d + Plan::kUnitBytes, have ? v : static_cast<const T *>(p.cache.v), have);
                k += step;
                v += step;
            }
            if (--left > 0) {
                fresh_load = decode_next(p.cache, p.q_tiles, load);
                if (fresh_load) table = p.cache.page_table + load.seq * p.cache.table_stride;
                page = load.len > 0 ? table[(load.unit * kUnitKeys) >> p.cache.page_shift] : 0;
            }
        };
        float o[kN][D / 16][4], m[kN][2], l[kN][2];
        uint32_t qf[kN][D / 16][2];
        int stage = 0, have = 0;
        bool fresh = true;
        const int a_row = ((lane / 8) % 2) * 8 + lane % 8, a_half = lane / 16;   // of K: (keys, 16-byte pieces) of the four tiles of a fragment
        const int v_row = (lane / 16) * 8 + lane % 8, v_half = (lane / 8) % 2;   // of V, which is read transposed
        const int total = static_cast<int>(u1 - u0);
        int fill = 0;
        // (One copy of each step in the code, the first loads' too: a warp has few units, and instructions come from afar the
        // first time.)
        for (int n = 1 - Plan::kStages; n < total; ++n) {
            if (n >= 0) {
                cp_async_wait<Plan::kStages - 2>();
                __syncwarp();  // all lanes' pieces of this unit are there, and all have read the unit before
            }
            if (n >= 0 && fresh) {
                const uint32_t q = q_place + q_use * Plan::kQBytes;
                if (++q_use == Plan::kQPlaces) q_use = 0;
#pragma unroll
                for (int t = 0; t < kN; ++t) {
#pragma unroll
                    for (int k = 0; k < D / 32; ++k) {
                        const int row = 8 * t + lane % 8;
                        uint32_t b[4];
                        ldsm4(q + row * Plan::kRowBytes + (((4 * k + lane / 8) ^ (row & 7)) << 4), b);
                        qf[t][2 * k][0] = b[0], qf[t][2 * k][1] = b[1], qf[t][2 * k + 1][0] = b[2], qf[t][2 * k + 1][1] = b[3];
                    }
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
#pragma unroll
                        for (int x = 0; x < 4; ++x) o[t][k][x] = 0.0f;
                    m[t][0] = m[t][1] = -INFINITY;
                    l[t][0] = l[t][1] = 0.0f;
                }
                fresh = false;
                have = 0;
                __syncwarp();  // (other queries come to this place)
            }
            if (left > 0) issue(fill);
            cp_async_commit();
            if (++fill == Plan::kStages) fill = 0;
            if (n < 0) continue;

            const uint32_t kb = ring + stage * 2 * Plan::kUnitBytes, vb = kb + Plan::kUnitBytes;
            float s[kN][2][4] = {};  // two chains of products, added at the end
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                uint32_t a[4];
                ldsm4(kb + a_row * Plan::kRowBytes + (((2 * k + a_half) ^ (a_row & 7)) << 4), a);
#pragma unroll
                for (int t = 0; t < kN; ++t) mma16<T>(s[t][k & 1], a, qf[t][k][0], qf[t][k][1]);
            }
            const int keys = at.len - at.unit * kUnitKeys;
            float x[kN][4];  // keys quad and quad + 8 of queries 2 pair and 2 pair + 1
            float top[kN][2];
            bool rise = false;
#pragma unroll
            for (int t = 0; t < kN; ++t) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[t][i] = (s[t][0][i] + s[t][1][i]) * c;
                    if (quad + 8 * (i / 2) >= keys) x[t][i] = -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    top[t][i] = fmaxf(x[t][i], x[t][i + 2]);
                    top[t][i] = fmaxf(top[t][i], __shfl_xor_sync(0xffffffffu, top[t][i], 4));
                    top[t][i] = fmaxf(top[t][i], __shfl_xor_sync(0xffffffffu, top[t][i], 8));
                    top[t][i] = fmaxf(top[t][i], __shfl_xor_sync(0xffffffffu, top[t][i], 16));
                    rise |= top[t][i] - m[t][i] > 8.0f;
                }
            }
            if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
                for (int t = 0; t < kN; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float to = fmaxf(m[t][i], top[t][i]), f = m[t][i] == -INFINITY ? 0.0f : exp2_fast(m[t][i] - to);
                        m[t][i] = to;
                        l[t][i] *= f;
#pragma unroll
                        for (int k = 0; k < D / 16; ++k) {
                            o[t][k][i] *= f;
                            o[t][k][i + 2] *= f;
                        }
                    }
            }
            uint32_t pf[kN][2];
#pragma unroll
            for (int t = 0; t < kN; ++t) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[t][i] = exp2_fast(x[t][i] - (m[t][i % 2] == -INFINITY ? 0.0f : m[t][i % 2] - kRaise<T>));
                    l[t][i % 2] += x[t][i];
                }
                pf[t][0] = transposed(pack_weights<T>(x[t][0], x[t][1]));
                pf[t][1] = transposed(pack_weights<T>(x[t][2], x[t][3]));
            }
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                uint32_t a[4];
                ldsm4_trans(vb + v_row * Plan::kRowBytes + (((2 * k + v_half) ^ (v_row & 7)) << 4), a);
#pragma unroll
                for (int t = 0; t < kN; ++t) mma16<T>(o[t][k], a, pf[t][0], pf[t][1]);
            }
            if (++stage == Plan::kStages) stage = 0;
            ++have;

            if (at.unit + 1 == at.units || n + 1 == total) {  // the end of the segment or of this warp's share
                float *part = n + 1 < total ? first_parts + warp * Plan::kPartFloats : reinterpret_cast<float *>(smem_raw + warp * Plan::kWarpBytes);
                __syncwarp();  // (the last part lies where all lanes have read the last unit)
#pragma unroll
                for (int t = 0; t < kN; ++t) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], 4);
                        l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], 8);
                        l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], 16);
                    }
                    if (have == at.units) {
                        const int r = at.tile * Plan::kRows + 8 * t + quad;
                        T *out = static_cast<T *>(p.out) + at.seq * p.out_ld + (static_cast<long long>(at.head) * p.group + r) * D + 2 * pair;
                        const float i0 = decode_inverse(l[t][0]), i1 = decode_inverse(l[t][1]);
#pragma unroll
                        for (int k = 0; k < D / 16; ++k)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t w = transposed(pack16<T>(o[t][k][2 * h] * i0, o[t][k][2 * h + 1] * i1));
                                if (r < p.group) *reinterpret_cast<uint32_t *>(out + 16 * k + 8 * h) = w;
                            }
                    } else {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int row = 8 * t + 2 * pair + i;
#pragma unroll
                            for (int k = 0; k < D / 16; ++k) {
                                part[row * Plan::kPad + 16 * k + quad] = o[t][k][i];
                                part[row * Plan::kPad + 16 * k + quad + 8] = o[t][k][i + 2];
                            }
                            if (quad == 0) *reinterpret_cast<float2 *>(part + Plan::kRows * Plan::kPad + 2 * row) = make_float2(m[t][i], l[t][i]);
                        }
                    }
                }
                if (have != at.units && lane == 0) s_part[2 * warp + (n + 1 < total ? 0 : 1)] = {at.start, at.seq, at.head, at.tile, at.units, have};
                fresh = true;
            }
            decode_next(p.cache, p.q_tiles, at);
        }
        cp_async_wait<0>();
    }
    __syncthreads();
    // Parts of one segment lie next to each other in the warps' order, first parts at even places; lane x looks at part x.  The
    // warps take the rows of what there is to join in turn.
    const int have = lane < 2 * kDecodeWarps ? s_part[lane].have : 0;
    const long long start = lane < 2 * kDecodeWarps ? s_part[lane].start : 0;
    const unsigned valid = __ballot_sync(0xffffffffu, have > 0), below = valid & ((1u << lane) - 1u);
    const long long start_before = __shfl_sync(0xffffffffu, start, below != 0 ? 31 - __clz(below) : 0);
    unsigned leaders = __ballot_sync(0xffffffffu, have > 0 && (below == 0 || start_before != start));
    const float *const my_part = lane % 2 == 0 ? first_parts + lane / 2 * Plan::kPartFloats
                                               : reinterpret_cast<const float *>(smem_raw + (lane / 2 % kDecodeWarps) * Plan::kWarpBytes);
    DecodeCrossing crossing = {0, 0, 0, 0};
    int nth = 0;
    while (leaders != 0) {
        const int i = __ffs(leaders) - 1;
        leaders &= leaders - 1;
        const unsigned members = valid & (~0u << i) & (leaders != 0 ? (1u << (__ffs(leaders) - 1)) - 1u : ~0u);
        const bool member = (members >> lane) & 1u;
        const DecodePart of = s_part[i];
        const bool whole = __reduce_add_sync(0xffffffffu, member ? have : 0) == of.units;
        const int slot = of.start < c0 ? 0 : 1;  // a CTA has at most one segment that began before it, and one that goes on behind it
        if (!whole && slot == 1 && threadIdx.x == 0) crossing = {of.seq, of.head, of.tile, share.owner(of.start + of.units - 1) - static_cast<int>(blockIdx.x) + 1};
        const int rows = min(Plan::kRows, p.group - of.tile * Plan::kRows);
        for (int row = (warp - nth) & (kDecodeWarps - 1); row < rows; row += kDecodeWarps) {
            constexpr int kC = D / 32;  // columns of a lane
            // (of a segment at most the last part is a first part, which lies in the workspace: its row is asked for first)
            const unsigned far = members & 0x55555555u;
            float acc[kC] = {};
            if (far != 0) load_floats(first_parts + (__ffs(far) - 1) / 2 * Plan::kPartFloats + row * Plan::kPad + kC * lane, acc);
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (member) ml = *reinterpret_cast<const float2 *>(my_part + Plan::kRows * Plan::kPad + 2 * row);
            float top = ml.x;
#pragma unroll
            for (int s = 8; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
            top = __shfl_sync(0xffffffffu, top, 0);
            const float w = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - top);
            float sum = w * ml.y;
#pragma unroll
            for (int s = 8; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
            sum = __shfl_sync(0xffffffffu, sum, 0);
            const float w_far = far != 0 ? __shfl_sync(0xffffffffu, w, __ffs(far) - 1) : 0.0f;
#pragma unroll
            for (int y = 0; y < kC; ++y) acc[y] *= w_far;
            const uint32_t near = smem_u32(smem_raw) + 4 * (row * Plan::kPad + kC * lane);
#pragma unroll 2
            for (unsigned todo = members & 0xAAAAAAAAu; todo != 0; todo &= todo - 1) {
                const int x = __ffs(todo) - 1;
                const float wx = __shfl_sync(0xffffffffu, w, x);
                float from[kC];
                if constexpr (kC == 4) {
                    const uint4 f = lds128(near + x / 2 * Plan::kWarpBytes);
                    from[0] = __uint_as_float(f.x), from[1] = __uint_as_float(f.y), from[2] = __uint_as_float(f.z), from[3] = __uint_as_float(f.w);
                } else {
                    const uint2 f = lds64(near + x / 2 * Plan::kWarpBytes);
                    from[0] = __uint_as_float(f.x), from[1] = __uint_as_float(f.y);
                }
#pragma unroll
                for (int y = 0; y < kC; ++y) acc[y] += wx * from[y];
            }
            if (whole) {
                T *out = static_cast<T *>(p.out) + of.seq * p.out_ld + (static_cast<long long>(of.head) * p.group + of.tile * Plan::kRows + row) * D + kC * lane;
                const float inv = decode_inverse(sum);
#pragma unroll
                for (int y = 0; y < kC; y += 2) *reinterpret_cast<uint32_t *>(out + y) = pack16<T>(acc[y] * inv, acc[y + 1] * inv);
            } else {
                const int at = (2 * blockIdx.x + slot) * 16 + row;
                float *to = p.partial + static_cast<size_t>(at) * D + kC * lane;
#pragma unroll
                for (int y = 0; y < kC; ++y) to[y] = acc[y];
                if (lane == 0) *reinterpret_cast<float2 *>(p.partial + static_cast<size_t>(gridDim.x) * 2 * 16 * D + 2 * at) = make_float2(top, sum);
            }
        }
        nth += rows;
    }
    if (threadIdx.x == 0) decode_crossings(p.partial, D, gridDim.x)[blockIdx.x] = crossing;
}

// Joins what several CTAs have of one segment.  Block (x, row): the segment that crosses from CTA x to the next, if x is the first
// CTA that has a part of it.  Warps take the parts in turn, in the order of the keys.
template <class T, int D, int kN>
__global__ void __launch_bounds__(32 * kDecodeWarps) paged_join_kernel(const DecodeParams p, int ctas) {
    constexpr int kC = D / 32, kRows = 8 * kN;
    __shared__ float s_acc[kDecodeWarps][D];
    __shared__ float2 s_ml[kDecodeWarps];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, row = blockIdx.y, x0 = blockIdx.x;
    grid_dep_wait();
    const DecodeCrossing at = decode_crossings(p.partial, D, ctas)[x0];
    const int r = at.tile * kRows + row, n = at.ctas;
    if (n == 0 || r >= p.group) return;
    const float *ml = p.partial + static_cast<size_t>(ctas) * 2 * 16 * D;
    const auto slot_of = [&](int x) { return 2 * (x0 + x) + (x == 0 ? 1 : 0); };  // the segment begins in the first
    // the warp's own parts, eight at a time, with a maximum of its own: the loads wait for nothing but this kernel's start
    constexpr int kAtOnce = 8;
    float top = -INFINITY, sum = 0.0f, acc[kC] = {};
    for (int x = warp; x < n; x += kDecodeWarps * kAtOnce) {
        float2 v[kAtOnce];
        float from[kAtOnce][kC];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int xi = x + i * kDecodeWarps, slot = slot_of(xi);
            v[i] = make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int y = 0; y < kC; ++y) from[i][y] = 0.0f;
            if (xi < n) {
                v[i] = *reinterpret_cast<const float2 *>(ml + 2 * (slot * 16 + row));
                const float *src = p.partial + (static_cast<size_t>(slot) * 16 + row) * D + kC * lane;
                load_floats(src, from[i]);
            }
        }
        float to = top;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) to = fmaxf(to, v[i].x);
        const float f = top == -INFINITY ? 0.0f : exp2_fast(top - to);
        top = to;
        sum *= f;
#pragma unroll
        for (int y = 0; y < kC; ++y) acc[y] *= f;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const float w = v[i].x == -INFINITY ? 0.0f : exp2_fast(v[i].x - top);
            sum += w * v[i].y;
#pragma unroll
            for (int y = 0; y < kC; ++y) acc[y] += w * from[i][y];
        }
    }
#pragma unroll
    for (int y = 0; y < kC; ++y) s_acc[warp][kC * lane + y] = acc[y];
    if (lane == 0) s_ml[warp] = make_float2(top, sum);
    __syncthreads();
    if (threadIdx.x < D / 2) {
        float a = 0.0f, b = 0.0f, all = -INFINITY;
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kDecodeWarps; ++w) all = fmaxf(all, s_ml[w].x);
#pragma unroll
        for (int w = 0; w < kDecodeWarps; ++w) {
            const float2 v = s_ml[w];
            const float f = v.x == -INFINITY ? 0.0f : exp2_fast(v.x - all);
            sum += f * v.y;
            a += f * s_acc[w][2 * threadIdx.x];
            b += f * s_acc[w][2 * threadIdx.x + 1];
        }
        const float inv = decode_inverse(sum);
        T *out = static_cast<T *>(p.out) + at.seq * p.out_ld + (static_cast<long long>(at.head) * p.group + r) * D;
        *reinterpret_cast<uint32_t *>(out + 2 * threadIdx.x) = pack16<T>(a * inv, b * inv);
    }
}

template <class T, int D, int kN>
inline int launch_decode_typed(DecodeParams &p, int ctas, bool pdl, cudaStream_t stream) {
    using Plan = DecodePlan<D, kN>;
    p.q_tiles = (p.group + Plan::kRows - 1) / Plan::kRows;
    const auto kernel = paged_attention_kernel<T, D, kN>;
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
    cfg.gridDim = dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(p.group < Plan::kRows ? p.group : Plan::kRows));
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_join_kernel<T, D, kN>, p, ctas);
}

// Queries in tiles of 8 or of 16: keys are read once for a tile, and 16 columns take twice the instructions of 8.  16 sequences of 2560
// tokens, 8 key heads: groups of 8 take 35.8 us with 8 columns and 36.8 with 16, groups of 16 take 60.8 and 40.4.
template <class T, int D>
inline int launch_decode(DecodeParams &p, int ctas, bool pdl, cudaStream_t stream) {
    return p.group <= 8 ? launch_decode_typed<T, D, 1>(p, ctas, pdl, stream) : launch_decode_typed<T, D, 2>(p, ctas, pdl, stream);
}

}  // namespace dmm
