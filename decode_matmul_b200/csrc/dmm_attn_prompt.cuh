// Causal attention of packed prompts over a paged cache, on the 5th-generation tensor cores.
//
// One pass over the keys with the softmax's running maximum m and sum l: for key tiles j of 128 keys,
//   S = Q K_j^T,  P = exp2(c S - c m),  O += P V_j,  l += rowsum(P),   result O / l,   c = scale log2(e).
//
// A CTA has two tiles of 128 query rows of one key head and one sequence, so that the tensor cores work for one tile while
// the softmax of the other runs.  The rows of a tile are (token, query head of the group): all the heads that share a
// key head read its tile once, and a tile spans few tokens, so little of the causal triangle's edge is computed in vain.
// Tensor memory holds O of both tiles (2 x D columns), P of both in 16 bits (2 x 64) and one S (128), which the tiles use in turn: a tile's
// scores stay there only until its softmax has them in registers, and the next ones are there when it has done with these.
//   warps 0..3, 4..7   softmax of tile 0, 1: a thread has a row
//   warp 8             MMA issue (one elected lane)
//   warp 9             TMA loads: Q, then K_0, V_0, K_1, ...; a tile of keys is one box per page
//   warps 10, 11       guard: rows of V behind the sequence's end become zeros in shared memory (0 * garbage could be NaN), and
//                      values that are not finite too where a row of the tile must not see them; the epilogue then adds
//                      them to the rows that do see them.  Only tiles in which a row ends are looked at.
// O is only brought to a new maximum when that has risen by more than 2^8 (c (max - m) > 8): the weights stay below
// 2^8 (2^15 in fp16, see kRaise), far from overflow, and the quotient O / l is the same.  Weights are rounded to the type of the values, as the tensor
// cores take them: half a step each, in no common direction, which the sum over the keys evens out.  Sums, maxima and O are fp32, l of weights that
// are not rounded.
//
// Bound: 4 D operations for each (row, key) on the tensor cores, 2048 cycles for two tiles of 128 x 128 at D = 128, and as many
// cycles for their 32768 exponentials (16 a cycle).  Neither is reached: a step of a tile's softmax takes some 2000 cycles of a warp (scores
// into registers, the maximum, the exponentials, of which two tiles' share the unit) and waits some 800 for products, and two tiles of
// a CTA are all that tensor memory holds.
// B200, graph, fp16, 64 heads of 128 on 8: 8192 tokens 864 us (1.27 PFLOP/s, 77 % of what a dense product reaches; tensor
// pipe 65 % busy, exponentials 65 %), 2048 tokens 70 us (0.98 PFLOP/s): every item has a beginning (its first keys' way from HBM, the
// guard) and an end (the last P V, O to memory) of 3 to 4 us that only the next item's loads run beside.  Under a load of some seconds
// the power cap takes the clock to 1.53 to 1.73 GHz, and 8192 tokens take 1004 us, 2048 81.  With 64 values a head the exponentials are the bound, at
// twice the products' cycles: 8192 tokens 692 us (477 of exponentials), 2048 65 (30).
#pragma once

#include "dmm_attn_common.cuh"
#include "dmm_attn_item.h"
#include "dmm_tmem.cuh"

namespace dmm {

struct PromptParams {
    const void *q;
    void *out;
    const int32_t *cu;
    long long q_ld, out_ld;
    CacheView cache;
    int tokens, heads, group, tile_tokens;  // tile_tokens = 128 / group: tokens of a tile
    float scale;
    uint8_t *workspace;  // see PromptHead
    int ctas;
};

constexpr int kPromptThreads = 384;
constexpr int kPromptKeys = 128;  // keys of a tile
constexpr long long kPromptTileLimit = 20000;  // cycles that a wait allows for each of many key tiles: they take some 2800

// Key tiles in which rows of a pair of tiles end: they are 256 tokens at most.
constexpr int kMostGuarded = 3;

template <int D>
struct PromptPlan {
    static constexpr int kHalves = D / 64;            // columns of 128 bytes that a tile consists of
    static constexpr uint32_t kHalfBytes = 128 * 128; // 128 rows of 128 bytes
    static constexpr uint32_t kTileBytes = kHalves * kHalfBytes;
    static constexpr int kStages = D == 128 ? 5 : 8;
    static constexpr uint32_t kQ = 0;
    static constexpr uint32_t kRing = 2 * kTileBytes;
    static constexpr uint32_t kBars = kRing + kStages * kTileBytes;
    // Barriers, in the order of their use for an item.  What not every item uses twice in a row has a phase of its own, which its users
    // count; the guard's come in two sets that the items use in turn.
    static constexpr int kBarItem = 0, kBarItemFree = 2, kBarNext = 4, kBarQ = 5, kBarQFree = 7, kBarFull = 9, kBarEmpty = kBarFull + kStages,
                         kBarS = kBarEmpty + kStages, kBarDone = kBarS + 2, kBarSFree = kBarDone + 2, kBarP = kBarSFree + 1, kBarO = kBarP + 2, kBarOFree = kBarO + 2, kBarLook = kBarOFree + 2,
                         kBarGuard = kBarLook + 2 * kMostGuarded, kNumBars = kBarGuard + 2 * kMostGuarded;
    __device__ static constexpr int phase_bit(int item, int tile) { return (item & 1) * kMostGuarded + tile; }
    __device__ static constexpr int look(int item, int tile) { return kBarLook + phase_bit(item, tile); }
    __device__ static constexpr int guard(int item, int tile) { return kBarGuard + phase_bit(item, tile); }
    __device__ static constexpr uint32_t arrivals(int bar) {
        if (bar >= kBarItemFree && bar < kBarNext) return 11;  // every warp but the one that finds the items
        if ((bar >= kBarSFree && bar < kBarO) || (bar >= kBarOFree && bar < kBarLook)) return 4;
        return bar >= kBarGuard ? 2 : 1;
    }
    static constexpr uint32_t kBytes = kBars + 8 * kNumBars + 64 + 1024;  // (the last: alignment)
    // tensor memory columns: P of tile i at 64 i, S of either tile, O of tile i at 256 + D i
    static constexpr uint32_t kP = 0, kS = 128, kO = 256;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void *tmap, int x, int y, int z, int w, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void *tmap, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}

// D[tmem] (+)= A[smem] * B[smem], descriptors as low and high words
__device__ __forceinline__ void mma_ss_f16(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 ad, bd;\nsetp.ne.b32 p, %6, 0;\nmov.b64 ad, {%1, %2};\nmov.b64 bd, {%3, %4};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %5, p;\n}\n" ::"r"(d),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(acc)
        : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_ts_f16_words(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 bd;\nsetp.ne.b32 p, %5, 0;\nmov.b64 bd, {%2, %3};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], bd, %4, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(acc)
        : "memory");
}

// 32 columns of a thread's row, not waited for
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *u) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
          "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]),
          "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]),
          "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(taddr)
        : "memory");
}
// wait::ld that names 32 of the loaded registers, so that no use of them can be moved above it
__device__ __forceinline__ void tmem_wait_ld32(uint32_t *u) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]), "+r"(u[8]), "+r"(u[9]),
                   "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]), "+r"(u[15]), "+r"(u[16]), "+r"(u[17]), "+r"(u[18]),
                   "+r"(u[19]), "+r"(u[20]), "+r"(u[21]), "+r"(u[22]), "+r"(u[23]), "+r"(u[24]), "+r"(u[25]), "+r"(u[26]), "+r"(u[27]),
                   "+r"(u[28]), "+r"(u[29]), "+r"(u[30]), "+r"(u[31])
                 :
                 : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// two fp32 operations at once
__device__ __forceinline__ uint64_t pair32(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair32(uint64_t r) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(r));
    return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

constexpr int kPromptItem = 2;
constexpr float kPromptJoin = 6.0f, kPromptLeast = 0.28f;  // 0.28 = sqrt(0.15 us a part in the join / 1.8 us a key tile)

// The sequences of one lane each, from b0 on; by a warp.
struct PromptSeqs {
    TokenSpan span;
    int len, pairs, first, last;  // first, last: key tiles of the first pair of tiles, and of the last
    __device__ __forceinline__ int units() const { return last + kPromptItem; }
    __device__ __forceinline__ PromptSeqs(const PromptParams &p, int b0) {
        const int b = b0 + static_cast<int>(threadIdx.x & 31);
        span = {0, 0};
        len = 0;
        if (b < p.cache.num_seqs) span = token_span(p.cu, b, p.tokens);
        if (span.n > 0) len = cache_len(p.cache, b);
        pairs = (span.n + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens);
        first = span.n > 0 ? (max(0, len - span.n + min(2 * p.tile_tokens, span.n)) + kPromptKeys - 1) / kPromptKeys : 0;
        last = span.n > 0 ? (len + kPromptKeys - 1) / kPromptKeys : 0;
    }
};
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// How the work is shared out: the same in every CTA, by a warp.
//   each == 0   whole items, which the CTAs take as they come, those with the most keys first.  A prompt from its beginning has items
//               of every length, and the short ones fill up what the long ones leave.
//   otherwise   the key tiles of all items in one line, cut into even shares: CTA x has units [begin(x), begin(x + 1)).  For few
//               items or long ones of one length (the next chunk of a prompt), which would leave CTAs idle.  An item counts as
//               many units as the last of its sequence has key tiles, and kPromptItem more for its beginning and end.  What CTAs
//               have of an item that they share goes through the workspace to a second kernel, which takes as long as
//               kPromptJoin key tiles, and longer the more parts an item has: shares are no smaller than kPromptLeast
//               times the square root of the longest item, and CTAs without one stay idle.
// Which of the two ends sooner is estimated: whole items end with the longest, or half of the shortest of a sequence (on
// average over the work) behind an even share.  B200, whole items against even shares: a prompt of 2048 tokens 76 us against
// 131, of 8192 891 against 1535 (an item counts as the longest of its sequence); on 8 heads and one key head 1024 tokens 22.8 against 25.1, 2048 36.7
// against 33.6, 4096 67 against 71, 8192 126 against 213; four chunks of 33 to 512 tokens behind 511 to 16384 262 against 190; 8 heads behind
// long contexts 16 tokens behind 16384 169 against 36, 512 behind 8192 125 against 40.
struct PromptShare {
    int each, more, all;
    __device__ __forceinline__ int begin(int x) const { return min(each * x + min(x, more), all); }
    __device__ __forceinline__ int owner(int u) const { return u < (each + 1) * more ? u / (each + 1) : more + (u - (each + 1) * more) / each; }
};
// `first`: the sequences from 0 on
__device__ __forceinline__ PromptShare prompt_share(const PromptParams &p, const PromptSeqs &first) {
    float items = 0.0f, tiles = 0.0f, units = 0.0f, least = 0.0f;
    int longest = 0;
    PromptSeqs q = first;
    for (int b0 = 0;;) {
        const float n = static_cast<float>(q.pairs) * static_cast<float>(p.cache.kv_heads), mean = 0.5f * static_cast<float>(q.first + q.last) + kPromptItem;
        items += n;
        tiles += n * mean;
        units += n * static_cast<float>(q.units());
        least += n * mean * static_cast<float>(q.first);
        longest = max(longest, q.last);
        b0 += 32;
        if (b0 >= p.cache.num_seqs) break;
        q = PromptSeqs(p, b0);
    }
    items = warp_sum(items), tiles = warp_sum(tiles), units = warp_sum(units), least = warp_sum(least);
    const float ctas = static_cast<float>(p.ctas), most = static_cast<float>(__reduce_max_sync(0xffffffffu, longest));
    const float whole = items <= ctas ? most : fmaxf(most, tiles / ctas + 0.5f * least / fmaxf(tiles, 1.0f));
    const float least_share = kPromptLeast * sqrtf(most + kPromptItem);
    if (units > 1e9f || whole <= fmaxf(units / ctas, least_share) + kPromptJoin) return {0, 0, 0};
    int all = 0;
    q = first;
    for (int b0 = 0;;) {
        all += q.pairs * p.cache.kv_heads * q.units();
        b0 += 32;
        if (b0 >= p.cache.num_seqs) break;
        q = PromptSeqs(p, b0);
    }
    all = __reduce_add_sync(0xffffffffu, all);
    const int each = all / p.ctas, wanted = static_cast<int>(least_share) + 1;
    if (each < wanted) return {wanted, 0, all};
    return {each, all - each * p.ctas, all};
}

// 32 sequences in the order of the work: those with the longest contexts first, so that what begins late is short.  A lane's sequence
// has `mine` items or units, behind `before` of others.
struct PromptLine {
    PromptSeqs q;
    int size, mine, before;  // size: units of an item
    __device__ __forceinline__ PromptLine(const PromptParams &p, const PromptShare &share, const PromptSeqs &seqs, int b0) : q(seqs) {
        const int lane = threadIdx.x & 31, there = min(32, p.cache.num_seqs - b0);
        size = share.each > 0 ? q.units() : 1;
        mine = q.pairs * p.cache.kv_heads * size;
        before = 0;
        for (int l = 0; l < there; ++l) {
            const int other = __shfl_sync(0xffffffffu, q.last, l), theirs = __shfl_sync(0xffffffffu, mine, l);
            if (other > q.last || (other == q.last && l < lane)) before += theirs;
        }
    }
};

// Item `index`, or the item of unit `index`, of which [index, end) is wanted; the order: 32 sequences at a time, tile pairs from the last
// (which has the most keys) to the first, key heads innermost.  By a warp; seq = -1 when there is no such item.  `first`: the
// sequences from 0 on.  *upto: the first unit behind what the item covers of [index, end).
__device__ __forceinline__ PromptItem prompt_item(const PromptParams &p, const PromptShare &share, const PromptLine &first, int index, int end, int *upto) {
    PromptItem it = {-1, 0, 0, 0, 0, 0, 0, 0, -1, 0};
    int rest = index, b0 = 0;
    PromptLine line = first;
    unsigned here;
    for (;;) {
        here = __ballot_sync(0xffffffffu, rest >= line.before && rest - line.before < line.mine);
        if (here != 0) break;
        rest -= __reduce_add_sync(0xffffffffu, line.mine);
        b0 += 32;
        if (b0 >= p.cache.num_seqs) return it;
        line = PromptLine(p, share, PromptSeqs(p, b0), b0);
    }
    const int who = __ffs(here) - 1, at = __shfl_sync(0xffffffffu, rest - line.before, who);
    it.seq = b0 + who;
    it.begin = __shfl_sync(0xffffffffu, line.q.span.begin, who);
    it.n = __shfl_sync(0xffffffffu, line.q.span.n, who);
    it.len = __shfl_sync(0xffffffffu, line.q.len, who);
    const int pairs = __shfl_sync(0xffffffffu, line.q.pairs, who);
    int item = at, units = 1, unit = 0;
    if (share.each > 0) {
        units = __shfl_sync(0xffffffffu, line.size, who);
        item = at / units;
        unit = at - item * units;
    }
    const int nth = item / p.cache.kv_heads;
    it.head = item - nth * p.cache.kv_heads;
    it.token0 = (pairs - 1 - nth) * 2 * p.tile_tokens;
    it.end = (max(0, it.len - it.n + min(it.token0 + 2 * p.tile_tokens, it.n)) + kPromptKeys - 1) / kPromptKeys;
    if (share.each > 0) {
        const int take = min(units - unit, end - index);
        *upto = index + take;
        if (take < units) {
            const int all = it.end;
            it.first = static_cast<int>(static_cast<long long>(all) * unit / units);
            it.end = static_cast<int>(static_cast<long long>(all) * (unit + take) / units);
            const int x = share.owner(index);
            it.slot = 2 * x + (unit == 0 ? 1 : 0);  // a CTA has at most one item that began before it, and one that goes on behind it
            if (unit == 0) it.ctas = share.owner(index + units - 1) - x + 1;
        }
    }
    return it;
}

// The workspace: whether items are shared; for each CTA the item that begins in it and goes on in others (ctas: how many have a part,
// 0 = there is none); then two slots for each CTA: weighted sums of values [256][D], maxima and sums [256][2].
struct PromptHead {
    int shared, pad[63];
};
__host__ __device__ inline size_t prompt_slots_at(int ctas) { return sizeof(PromptHead) + (static_cast<size_t>(ctas) * sizeof(PromptItem) + 255) / 256 * 256; }
__device__ __forceinline__ PromptItem *prompt_crossings(const PromptParams &p) { return reinterpret_cast<PromptItem *>(p.workspace + sizeof(PromptHead)); }
__device__ __forceinline__ float *prompt_slot(const PromptParams &p, int head_dim, int slot) {
    return reinterpret_cast<float *>(p.workspace + prompt_slots_at(p.ctas)) + static_cast<size_t>(slot) * 256 * (head_dim + 2);
}
inline size_t prompt_workspace(int head_dim, int ctas) { return prompt_slots_at(ctas) + static_cast<size_t>(ctas) * 2 * 256 * (head_dim + 2) * sizeof(float); }

template <class T>
struct F16Kind;  // operand type bits of the instruction descriptor; a word whose 16-bit halves are all exponent
template <>
struct F16Kind<__half> {
    static constexpr uint32_t kType = 0, kExponent = 0x7C00u;
};
template <>
struct F16Kind<__nv_bfloat16> {
    static constexpr uint32_t kType = (1u << 7) | (1u << 10), kExponent = 0x7F80u;
};

// 32 columns of 16 rows, as a warp holds an accumulator of 16 x 8 tiles: u[4 c + x] is row lane / 4 (x < 2) or lane / 4 + 8, column
// 8 c + 2 (lane % 4) + x % 2.
__device__ __forceinline__ void tmem_ld16x32(uint32_t taddr, uint32_t (&u)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
          "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(taddr)
        : "memory");
}

// A thread's row of one tile of scores becomes a row of weights, in tensor memory.  m: the maximum that the weights are taken against,
// l: their sum so far.
template <class T, int D>
struct SoftmaxRow {
    uint32_t s_at, p_at, o_at;  // tensor memory of S, P and O
    float c;               // weights are 2^(c S - c m)
    uint32_t bar, bar_free, bar_done;  // barriers of P, of S when it has been read, and of the products before
    uint32_t done;         // phase of the last
    volatile int *failed;
    int sees;              // keys of the tile that the row sees
    bool begun;            // O has a sum already

    // masked: some row does not see all keys.  (One copy for both, and loops that stay loops all over this kernel: an item runs them a few times
    // only, and with two copies prompts of 1 to 1531 tokens took 10 % longer, of 2048 5 %.)
    __device__ __forceinline__ void step(const bool masked, float &m, float &l) const {
        uint32_t u[128];
        tmem_ld32(s_at, u);
        tmem_ld32(s_at + 32, u + 32);
        tmem_wait_ld32(u);
        tmem_wait_ld32(u + 32);
        tmem_ld32(s_at + 64, u + 64);
        tmem_ld32(s_at + 96, u + 96);
        float tops[8];  // (chains of their own)
        const auto score = [&](int x) { return __uint_as_float(u[x]); };
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (half == 1) {
                tmem_wait_ld32(u + 64);
                tmem_wait_ld32(u + 96);
                tc_fence_before();
                __syncwarp();
                if ((threadIdx.x & 31) == 0) mbar_arrive(bar_free);  // (the other tile's scores come to this place)
            }
            if (masked) {
#pragma unroll
                for (int x = 64 * half; x < 64 * half + 64; ++x) u[x] = x < sees ? u[x] : 0xff800000u;
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                if (half == 0) tops[q] = fmaxf(score(q), score(q + 8));
#pragma unroll
                for (int x = half == 0 ? 16 : 64; x < 64 * half + 64; x += 16) tops[q] = max3(tops[q], score(x + q), score(x + q + 8));
            }
        }
        const float top = max3(max3(tops[0], tops[1], tops[2]), max3(tops[3], tops[4], tops[5]), fmaxf(tops[6], tops[7]));
        if (begun) {  // the products of the tile before have read P and are in O
            mbar_wait(bar_done, done, failed);
            tc_fence_after();
        }
        const bool rise = top > m && (m == -INFINITY || (top - m) * c > 8.0f);
        if (__any_sync(0xffffffffu, rise)) {
            const float to = rise ? top : m, f = m == -INFINITY ? 0.0f : exp2_fast((m - to) * c);
            m = to;
            l *= f;
            if (begun) {
#pragma unroll 1
                for (int q = 0; q < D / 16; ++q) {
                    uint32_t o[16];
                    tmem_ld16(o_at + 16 * q, o);
                    tmem_wait_ld(o);
#pragma unroll
                    for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                    tmem_st16(o_at + 16 * q, o);
                }
            }
        }
        const float mc = m == -INFINITY ? 0.0f : fmaf(-m, c, kRaise<T>);
        const uint64_t c2 = pair32(c, c), mc2 = pair32(mc, mc);
        uint64_t sums[4] = {};
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            uint32_t w[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                float2 y = unpair32(fma2(pair32(score(16 * q + 2 * x), score(16 * q + 2 * x + 1)), c2, mc2));
                y.x = exp2_fast(y.x);
                y.y = exp2_fast(y.y);
                sums[x % 4] = add2(sums[x % 4], pair32(y.x, y.y));
                w[x] = pack_weights<T>(y.x, y.y);
            }
            tmem_st8(p_at + 8 * q, w);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
        const float2 sum = unpair32(add2(add2(sums[0], sums[1]), add2(sums[2], sums[3])));
        l += sum.x + sum.y;
    }
};

// The next block of the grid that has not begun, taken over (cluster launch control): asked for, and the answer, -1 when there is none.
__device__ __forceinline__ void ask_next_block(uint32_t answer, uint32_t bar) {
    fence_async_smem();  // (the answer before has been read)
    mbar_arrive_expect_tx(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ int next_block(uint32_t answer) {
    int x;
    asm volatile(
        "{\n.reg .pred p;\n.reg .b128 r;\nld.shared.b128 r, [%1];\n"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\nmov.b32 %0, -1;\n"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n}\n"
        : "=r"(x)
        : "r"(answer)
        : "memory");
    return x;
}

// What follows from an item: its key tiles for each of its two tiles (from `first` on), how many keys their last rows see, and the first
// key tile in which a row ends (or the sequence).  Row t of the new tokens sees keys below len - n + t + 1; all rows see those below
// `seen`.
struct PromptExtent {
    int tiles[2], most[2], all, seen, guarded;
    __device__ __forceinline__ PromptExtent(const PromptItem &it, int tile_tokens) {
        const int shift = it.len - it.n + 1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t0 = it.token0 + i * tile_tokens, t1 = min(t0 + tile_tokens, it.n);
            most[i] = t1 > t0 ? max(0, shift + t1 - 1) : 0;
            tiles[i] = max(0, min(it.end, (most[i] + kPromptKeys - 1) / kPromptKeys) - it.first);
        }
        all = it.end - it.first;
        seen = max(0, shift + it.token0);
        guarded = seen / kPromptKeys;
    }
};

// A CTA goes from item to item: the loads of the next begin while the tensor cores are still at work on the present one.  The load
// warp finds the items and hands them on in two places in turn.
template <class T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
    prompt_attention_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                            const __grid_constant__ CUtensorMap vmap, const PromptParams p) {
    using Plan = PromptPlan<D>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ PromptItem s_item[2];
    __shared__ __align__(16) uint32_t s_answer[4];
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_failed, s_poison[2];
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) / 32, 0), lane = threadIdx.x % 32, tt = p.tile_tokens;
    const auto bar = [&](int i) { return smem + Plan::kBars + 8u * static_cast<uint32_t>(i); };
    grid_dep_wait();
    if (warp == 8) {
        if (lane == 0) {
            s_failed = 0;
            for (int i = 0; i < Plan::kNumBars; ++i) mbar_init(bar(i), Plan::arrivals(i));
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(smem_u32(&s_tmem), 512);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    grid_dep_launch();  // (the kernel that joins parts waits for this one's end)
    // What other warps may set at any time is read once for a warp: its lanes part nowhere, as what follows wants all of them.
    const auto failed = [&]() { return __any_sync(0xffffffffu, s_failed) != 0; };
    // Most waits are for a step of a key tile; those of a warp that has nothing to do for an item may be as long as the item.
    const auto limit_of = [](int tiles) { return kWaitLimitCycles + kPromptTileLimit * tiles; };
    // The item of turn `k` for every warp but the one that finds them; no more when its sequence is -1.  `before`: key tiles of the item before.
    const auto item_of = [&](int k, int before) {
        mbar_wait(bar(Plan::kBarItem + (k & 1)), static_cast<uint32_t>(k >> 1) & 1u, &s_failed, limit_of(before));
        PromptItem it = s_item[k & 1];
        if (failed()) it.seq = -1;
        return it;
    };
    const auto item_done = [&](int k) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(Plan::kBarItemFree + (k & 1)));
    };

    // Registers: 384 threads are launched with 168 each; the softmax holds a row of 128 scores and wants more, the others need
    // less (256 * 216 + 128 * 72 = 64512).
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 9) {
            // =============================== items and loads ===============================
            const int shift_pg = p.cache.page_shift, page = 1 << shift_pg, box = min(page, kPromptKeys);
            int index = static_cast<int>(blockIdx.x), stage = 0;
            uint32_t parity = 1, q_free = 0, asked = 0;  // q_free: bits, phases
            bool q_used[2] = {false, false};
            const PromptSeqs seqs(p, 0);
            const PromptShare share = prompt_share(p, seqs);
            const PromptLine line(p, share, seqs, 0);
            const bool shared = share.each > 0;
            int unit = 0, unit_end = 0;  // of an even share: what is left of it
            PromptItem crossing = {-1, 0, 0, 0, 0, 0, 0, 0, -1, 0};
            const auto begin_block = [&]() {  // block `index` is this CTA's
                if (index == 0 && lane == 0) reinterpret_cast<PromptHead *>(p.workspace)->shared = shared;
                if (!shared || index < 0 || index >= p.ctas) return;
                unit = share.begin(index);
                unit_end = share.begin(index + 1);
                if (lane == 0) prompt_crossings(p)[index] = crossing;  // (nothing, until the share is done)
            };
            const auto ask = [&]() {
                if (lane == 0) ask_next_block(smem_u32(s_answer), bar(Plan::kBarNext));
                __syncwarp();
            };
            const auto answer = [&]() {
                mbar_wait(bar(Plan::kBarNext), asked & 1u, &s_failed);
                ++asked;
                index = failed() ? -1 : next_block(smem_u32(s_answer));  // (without an answer there is no block)
                __syncwarp();
                begin_block();
            };
            begin_block();
            for (int k = 0;; ++k) {
                PromptItem it = {-1, 0, 0, 0, 0, 0, 0, 0, -1, 0};
                bool more = false;  // of this block's share
                while (index >= 0) {
                    if (!shared || index < p.ctas) it = prompt_item(p, share, line, shared ? unit : index, unit_end, &unit);
                    if (it.seq >= 0 || failed()) break;
                    ask();  // (the grid has some blocks more than there is work for)
                    answer();
                }
                if (shared && it.seq >= 0) {
                    more = unit < unit_end;
                    if (it.ctas > 0) crossing = it;
                    if (!more && lane == 0) prompt_crossings(p)[index] = crossing;
                    if (!more) crossing.ctas = 0;
                }
                if (k >= 2) mbar_wait(bar(Plan::kBarItemFree + (k & 1)), static_cast<uint32_t>((k >> 1) - 1) & 1u, &s_failed);
                if (failed()) it.seq = -1;
                if (lane == 0) {
                    s_item[k & 1] = it;
                    s_poison[k & 1] = 0;
                    mbar_arrive(bar(Plan::kBarItem + (k & 1)));
                }
                if (it.seq < 0) break;
                const PromptExtent ext(it, tt);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (ext.tiles[i] == 0) continue;
                    if (q_used[i]) {  // the products of the item before that used this place are done with it
                        mbar_wait(bar(Plan::kBarQFree + i), (q_free >> i) & 1u, &s_failed);
                        q_free ^= 1u << i;
                    }
                    q_used[i] = true;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(bar(Plan::kBarQ + i), static_cast<uint32_t>(Plan::kHalves * p.group * tt) * 128u);
#pragma unroll
                        for (int hh = 0; hh < Plan::kHalves; ++hh)
                            tma_load_3d(smem + Plan::kQ + i * Plan::kTileBytes + hh * Plan::kHalfBytes, &qmap, 64 * hh, it.head * p.group,
                                        it.begin + it.token0 + i * tt, bar(Plan::kBarQ + i));
                    }
                }
                const int32_t *table = p.cache.page_table + it.seq * p.cache.table_stride;
                if (ext.all == 0 && !more) ask();
                for (int j = 0; j < ext.all; ++j) {
                    if (j + 1 == ext.all && !more) ask();
                    const int tile = it.first + j, pos = tile * kPromptKeys + lane * box;
                    const bool mine = lane * box < kPromptKeys && pos < it.len;
                    int pg = 0;
                    if (mine) {
                        pg = table[pos >> shift_pg];
                        if (pg < 0 || pg >= p.cache.num_pages) {
                            raise_status(DMM_STATUS_BAD_PAGE);
                            pg = -1;  // outside the tensor map: reads as zeros
                        }
                    }
                    const uint32_t bytes = static_cast<uint32_t>(__popc(__ballot_sync(0xffffffffu, mine)) * box) * 128u * Plan::kHalves;
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        mbar_wait(bar(Plan::kBarEmpty + stage), parity, &s_failed);
                        if (failed()) break;
                        // (values that the guard looks at first arrive at barriers of their own)
                        const uint32_t full = bar(kv == 1 && tile >= ext.guarded ? Plan::look(k, tile - ext.guarded) : Plan::kBarFull + stage);
                        if (lane == 0) mbar_arrive_expect_tx(full, bytes);
                        __syncwarp();
                        if (mine) {
                            const uint32_t dst = smem + Plan::kRing + stage * Plan::kTileBytes + static_cast<uint32_t>(lane * box) * 128u;
#pragma unroll
                            for (int hh = 0; hh < Plan::kHalves; ++hh)
                                tma_load_4d(dst + hh * Plan::kHalfBytes, kv == 0 ? &kmap : &vmap, 64 * hh, pos & (page - 1), it.head, pg, full);
                        }
                        if (kv == 1 && tile >= ext.guarded && lane == 0) mbar_arrive(bar(Plan::kBarFull + stage));  // (keeps its phases in step)
                        if (++stage == Plan::kStages) {
                            stage = 0;
                            parity ^= 1u;
                        }
                    }
                }
                if (more) continue;
                answer();
            }
            if (s_failed) {  // a wait gave up: copies in flight land before the CTA goes (they take microseconds)
                const long long t0 = clock64();
                while (clock64() - t0 < 4000000) __nanosleep(1000);
            }
        } else if (warp == 8) {
            // =============================== MMA ===============================
            const bool leader = elect_one();
            // D fp32 (1 at bit 4), the operands' type, N >> 3 at bit 17, M >> 4 at bit 24; V is the operand whose rows run along N (bit 16);
            // -Q for a scale below 0 (bit 13)
            const uint32_t id_s = (p.scale < 0.0f ? 1u << 13 : 0u) | (1u << 4) | F16Kind<T>::kType | ((128u >> 3) << 17) | ((128u >> 4) << 24);
            constexpr uint32_t kIdO = (1u << 4) | F16Kind<T>::kType | (1u << 16) | ((static_cast<uint32_t>(D) >> 3) << 17) | ((128u >> 4) << 24);
            // 128-byte swizzle (2 at bit 61), 8-row groups 1024 bytes apart, version 1 at bit 46; the low word has the address and, for
            // V, the distance from one 64 columns to the next
            constexpr uint32_t kHi = (1024u >> 4) | (1u << 14) | (2u << 29);
            const auto lo = [&](uint32_t addr, uint32_t lbo) { return ((addr >> 4) & 0x3FFFu) | ((lbo >> 4) << 16); };
            const auto place = [&](int s) { return smem + Plan::kRing + static_cast<uint32_t>(s) * Plan::kTileBytes; };
            // A place of the ring: keys and values have every second one.
            struct Ring {
                int stage;
                uint32_t parity;
                __device__ __forceinline__ void step() {
                    stage += 2;
                    if (stage >= Plan::kStages) {
                        stage -= Plan::kStages;
                        parity ^= 1u;
                    }
                }
            };
            Ring keys = {0, 0}, values = {1, 0};
            uint32_t q_full = 0, p_full = 0, o_free = 0, guard = 0, s_count = 0;  // bits: phases
            bool o_used[2] = {false, false};
            for (int k = 0, before = 0;; ++k) {
                const PromptItem it = item_of(k, before);
                if (it.seq < 0) break;
                const PromptExtent ext(it, tt);
                before = ext.all;
                // Scores and products go in the order (tile 0, key tile 0), (tile 1, 0), (0, 1), (1, 1), ...; the scores of two are asked
                // for before the products of the first, and then always the next ones behind those of one more: they are there when
                // a tile's softmax has done with the scores before.
                int si = ext.tiles[0] > 0 ? 0 : 1, sj = 0, pi = si, pj = 0;
                const auto next = [&](int &i, int &j) {  // false: there is no other for this key tile
                    if (i == 0 && j < ext.tiles[1]) {
                        i = 1;
                        return true;
                    }
                    ++j;
                    i = j < ext.tiles[0] ? 0 : 1;
                    return false;
                };
                bool new_keys = true, new_values = true;
                const auto scores = [&]() {
                    if (sj >= ext.all) return;
                    if (new_keys) mbar_wait(bar(Plan::kBarFull + keys.stage), keys.parity, &s_failed);
                    if (sj == 0) {
                        mbar_wait(bar(Plan::kBarQ + si), (q_full >> si) & 1u, &s_failed);
                        q_full ^= 1u << si;
                    }
                    if (s_count > 0) mbar_wait(bar(Plan::kBarSFree), (s_count - 1) & 1u, &s_failed);
                    ++s_count;
                    tc_fence_after();
                    const uint32_t a = lo(smem + Plan::kQ + si * Plan::kTileBytes, 16), b = lo(place(keys.stage), 16);
                    if (leader) {
#pragma unroll
                        for (int d = 0; d < D / 16; ++d) {
                            const uint32_t off = (d / 4) * (Plan::kHalfBytes >> 4) + (d % 4) * 2;
                            mma_ss_f16(tmem + Plan::kS, a + off, kHi, b + off, kHi, id_s, d > 0);
                        }
                        tc_commit(bar(Plan::kBarS + si));
                        if (sj + 1 == (si == 0 ? ext.tiles[0] : ext.tiles[1])) tc_commit(bar(Plan::kBarQFree + si));
                    }
                    __syncwarp();
                    new_keys = !next(si, sj);
                    if (new_keys) {
                        if (leader) tc_commit(bar(Plan::kBarEmpty + keys.stage));
                        __syncwarp();
                        keys.step();
                    }
                };
#pragma unroll 1
                for (int n = ext.tiles[0] > 0 && ext.tiles[1] > 0 ? 3 : 2; n > 0; --n) scores();
                while (pj < ext.all) {
                    if (new_values) {
                        mbar_wait(bar(Plan::kBarFull + values.stage), values.parity, &s_failed);
                        if (it.first + pj >= ext.guarded) {
                            const int g = it.first + pj - ext.guarded, at = Plan::phase_bit(k, g);
                            mbar_wait(bar(Plan::guard(k, g)), (guard >> at) & 1u, &s_failed);
                            guard ^= 1u << at;
                        }
                    }
                    if (pj == 0) {  // the epilogue before has read O
                        if (pi == 0 ? o_used[0] : o_used[1]) {
                            mbar_wait(bar(Plan::kBarOFree + pi), (o_free >> pi) & 1u, &s_failed);
                            o_free ^= 1u << pi;
                        }
                        (pi == 0 ? o_used[0] : o_used[1]) = true;
                    }
                    // (the last tile: only the 16 keys at a time that some row sees)
                    const int steps = min(8, ((pi == 0 ? ext.most[0] : ext.most[1]) - (it.first + pj) * kPromptKeys + 15) / 16);
                    const uint32_t begun = pj > 0 ? 1u : 0u, v = lo(place(values.stage), Plan::kHalfBytes);
                    mbar_wait(bar(Plan::kBarP + pi), (p_full >> pi) & 1u, &s_failed);
                    p_full ^= 1u << pi;
                    tc_fence_after();
                    if (leader) {
#pragma unroll
                        for (int n = 0; n < 8; ++n)
                            if (n < steps) mma_ts_f16_words(tmem + Plan::kO + D * pi, tmem + Plan::kP + 64 * pi + 8 * n, v + n * (2048u >> 4), kHi, kIdO, n > 0 ? 1u : begun);
                    }
                    __syncwarp();
                    if (leader) tc_commit(bar((pj + 1 == (pi == 0 ? ext.tiles[0] : ext.tiles[1]) ? Plan::kBarO : Plan::kBarDone) + pi));
                    new_values = !next(pi, pj);
                    if (new_values) {
                        if (leader) tc_commit(bar(Plan::kBarEmpty + values.stage));
                        values.step();
                    }
                    __syncwarp();
                    scores();
                }
                item_done(k);
            }
        } else if (warp >= 10) {
            // =============================== guard ===============================
            const int t = threadIdx.x - 320;
            constexpr uint32_t kMask = F16Kind<T>::kExponent * 0x10001u;
            int tile0 = 0;        // tiles of the ring that items before had
            uint32_t look = 0;    // bits: phases
            for (int k = 0, before = 0;; ++k) {
                const PromptItem it = item_of(k, before);
                if (it.seq < 0) break;
                const PromptExtent ext(it, tt);
                before = ext.all;
                for (int j = max(0, ext.guarded - it.first); j < ext.all; ++j) {
                    // rows of values behind the first that not every query sees (or all of them, where the sequence ends)
                    const int rows = min(kPromptKeys, it.len - (it.first + j) * kPromptKeys), row0 = max(0, ext.seen - (it.first + j) * kPromptKeys), g = it.first + j - ext.guarded, at = Plan::phase_bit(k, g);
                    mbar_wait(bar(Plan::look(k, g)), (look >> at) & 1u, &s_failed, limit_of(ext.all));
                    look ^= 1u << at;
                    const uint32_t base = smem + Plan::kRing + static_cast<uint32_t>((tile0 + 2 * j + 1) % Plan::kStages) * Plan::kTileBytes;
                    const auto where = [&](int c) { return base + (c / 1024) * Plan::kHalfBytes + (c % 1024) * 16u; };  // piece c: row (c % 1024) / 8
                    // a half is not finite if its exponent is all ones: one more there carries into the sign
                    constexpr uint32_t kOne = (0x8000u - F16Kind<T>::kExponent) * 0x10001u;
                    const auto carries = [&](uint32_t w) { return (w & kMask) + kOne; };
                    uint32_t any = 0;
#pragma unroll 2
                    for (int c = 8 * row0 + t; c < 8 * rows; c += 64)
#pragma unroll
                        for (int hh = 0; hh < Plan::kHalves; ++hh) {
                            const uint4 w = lds128(where(c + 1024 * hh));
                            any |= carries(w.x) | carries(w.y) | carries(w.z) | carries(w.w);
                        }
#pragma unroll 1
                    for (int c = 8 * rows + t; c < 8 * ((rows + 15) & ~15); c += 64)
#pragma unroll
                        for (int hh = 0; hh < Plan::kHalves; ++hh) sts128(where(c + 1024 * hh), make_uint4(0, 0, 0, 0));
                    if (any & 0x80008000u) {
                        s_poison[k & 1] = 1;
#pragma unroll 1
                        for (int c = 8 * row0 + t; c < 8 * rows + 1024 * (Plan::kHalves - 1); c += 64) {
                            if ((c % 1024) / 8 >= rows || (c % 1024) / 8 < row0) continue;
                            const uint4 w = lds128(where(c));
                            uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t bad = carries(x[i]);
                                x[i] &= (bad & 0x8000u ? 0u : 0xFFFFu) | (bad & 0x80000000u ? 0u : 0xFFFF0000u);
                            }
                            sts128(where(c), make_uint4(x[0], x[1], x[2], x[3]));
                        }
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(Plan::guard(k, g)));
                }
                tile0 = (tile0 + 2 * ext.all) % Plan::kStages;
                item_done(k);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // =============================== softmax ===============================
        const int i = warp / 4, r = threadIdx.x % 128, magic = 65536 / p.group + 1, tok = r * magic >> 16;  // (r / group, for r < 128)
        const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * (warp % 4)) << 16);
        const uint32_t s_at = lanes + Plan::kS, p_at = lanes + Plan::kP + 64 * i, o_at = lanes + Plan::kO + D * i;
        // (the products have the sign of the scale; times 2^-149 every finite score is as good as 0, and a hidden one stays -infinity)
        const float c = p.scale == 0.0f ? __uint_as_float(1u) : fabsf(p.scale) * 1.4426950408889634f;
        uint32_t s_full = 0, o_full = 0, done = 0;  // phases
        PromptItem next = item_of(0, 0);
        for (int k = 0;; ++k) {
            const PromptItem it = next;
            if (it.seq < 0) break;
            const PromptExtent ext(it, tt);
            const int tiles = i == 0 ? ext.tiles[0] : ext.tiles[1];
            const int token = it.token0 + i * tt + tok, shift = it.len - it.n + 1;
            const bool mine = tok < tt && token < it.n;
            const int sees = mine ? max(0, shift + token) : 0;
            const int free = max(0, shift + it.token0 + i * tt) / kPromptKeys - it.first;  // key tiles that every row of this tile sees whole
            float m = -INFINITY, l = 0.0f;
            for (int j = 0; j < tiles; ++j) {
                mbar_wait(bar(Plan::kBarS + i), s_full, &s_failed);
                s_full ^= 1u;
                tc_fence_after();
                const SoftmaxRow<T, D> row = {s_at, p_at, o_at, c, bar(Plan::kBarP + i), bar(Plan::kBarSFree), bar(Plan::kBarDone + i), done, &s_failed,
                                              sees - (it.first + j) * kPromptKeys, j > 0};
                if (j > 0) done ^= 1u;
                row.step(j >= free, m, l);
            }
            next = item_of(k + 1, ext.all);  // (known before this item's last products are done: its finding waits for none of them)
            if (tiles > 0) {
                mbar_wait(bar(Plan::kBarO + i), o_full, &s_failed);
                o_full ^= 1u;
                tc_fence_after();
            }
            const bool part = it.slot >= 0;
            const float inv = part ? 1.0f : l > 0.0f || l != l ? 1.0f / l : 0.0f;
            float *const share = part ? prompt_slot(p, D, it.slot) + 128 * D * i : nullptr;
            if (part) *reinterpret_cast<float2 *>(prompt_slot(p, D, it.slot) + 256 * D + 2 * (128 * i + r)) = make_float2(m == -INFINITY ? m : m * c, l);
            T *const out = static_cast<T *>(p.out) + static_cast<long long>(it.begin + it.token0 + i * tt) * p.out_ld + static_cast<long long>(it.head * p.group) * D;
            // (a tile that waits for no products, or not for the later ones of the other tile, may come here while the guard looks: either way
            // is right for it, but the warp's lanes go one way)
            if (__any_sync(0xffffffffu, s_poison[k & 1])) {
                // values that are not finite, which the guard has taken out of the tiles in which rows end: row by row
                T *to = out + static_cast<long long>(tok) * p.out_ld + (r - tok * p.group) * D;
#pragma unroll 1
                for (int q = 0; q < D / 16; ++q) {
                    uint32_t u[16] = {};
                    __syncwarp();  // (rows differ in what they add)
                    if (tiles > 0) {
                        tmem_ld16(o_at + 16 * q, u);
                        tmem_wait_ld(u);
                    }
                    if (!mine) continue;
#pragma unroll 1
                    for (int pos = max(ext.seen, it.first * kPromptKeys); pos < min(sees, it.end * kPromptKeys); ++pos) {
                        const long long row = cache_row(p.cache, it.seq, pos, it.head);
                        if (row < 0) continue;
                        const T *v = static_cast<const T *>(p.cache.v) + row + 16 * q;
#pragma unroll
                        for (int x = 0; x < 16; ++x) {
                            const float f = static_cast<float>(v[x]);
                            if (!isfinite(f)) u[x] = __float_as_uint(__uint_as_float(u[x]) + f);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        if (part)
                            share[r * D + 16 * q + x] = __uint_as_float(u[x]);
                        else
                            to[16 * q + x] = static_cast<T>(__uint_as_float(u[x]) * inv);
                    }
                }
            } else {
                // 8 rows of 32 bytes with each store: a row at a time would touch 32 lines.  (Rows of 16 bytes, which need no exchange, and of 64,
                // which need four, take 2 % longer over prompts of a few hundred tokens.)
                const bool odd = lane & 1;
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {  // 16 rows
                    uint32_t u[D / 32][16] = {};
                    if (tiles > 0) {
#pragma unroll
                        for (int q = 0; q < D / 32; ++q) tmem_ld16x32(o_at + (static_cast<uint32_t>(h) << 20) + 32 * q, u[q]);
#pragma unroll
                        for (int q = 0; q < D / 32; ++q) tmem_wait_ld(u[q]);
                    }
#pragma unroll 1
                    for (int e = 0; e < 2; ++e) {
                        const int in_warp = 16 * h + 8 * e + lane / 4, rr = 32 * (warp % 4) + in_warp, t = rr * magic >> 16;
                        const float f = __shfl_sync(0xffffffffu, inv, in_warp);
                        const bool there = t < tt && it.token0 + i * tt + t < it.n;
                        T *to = out + static_cast<long long>(t) * p.out_ld + (rr - t * p.group) * D + (odd ? 8 : 0) + lane % 4 / 2 * 4;
                        if (part) {
                            if (tiles > 0 && there)
#pragma unroll
                                for (int q = 0; q < D / 32; ++q)
#pragma unroll
                                    for (int x = 0; x < 4; ++x)
                                        *reinterpret_cast<uint2 *>(share + rr * D + 32 * q + 8 * x + 2 * (lane % 4)) = make_uint2(e ? u[q][4 * x + 2] : u[q][4 * x], e ? u[q][4 * x + 3] : u[q][4 * x + 1]);
                            continue;
                        }
#pragma unroll
                        for (int q = 0; q < D / 32; ++q) {
                            uint32_t w[4];
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                const float2 v = unpair32(mul2(pair32(__uint_as_float(e ? u[q][4 * x + 2] : u[q][4 * x]), __uint_as_float(e ? u[q][4 * x + 3] : u[q][4 * x + 1])), pair32(f, f)));
                                w[x] = pack16<T>(v.x, v.y);
                            }
#pragma unroll
                            for (int x = 0; x < 4; x += 2) {  // (neighbouring lanes exchange a word: 4 columns a lane, 16 of a row)
                                const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? w[x] : w[x + 1], 1);
                                if (there) *reinterpret_cast<uint2 *>(to + 32 * q + 8 * x) = make_uint2(odd ? got : w[x], odd ? w[x + 1] : got);
                            }
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && tiles > 0) mbar_arrive(bar(Plan::kBarOFree + i));
            item_done(k);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins what several CTAs have of an item, in the order of the keys.  Blocks (., x) have the item that begins in CTA x, 32 rows each, so
// that one with many parts is read by several SMs (one SM takes 1.1 us a part); eight lanes have a row.  Without any such item
// the kernel takes 1.5 us.
constexpr int kJoinRows = 32;
template <class T, int D>
__global__ void __launch_bounds__(8 * kJoinRows) prompt_join_kernel(const PromptParams p) {
    grid_dep_wait();
    if (reinterpret_cast<const PromptHead *>(p.workspace)->shared == 0) return;
    const PromptItem it = prompt_crossings(p)[blockIdx.y];
    if (!prompt_item_crosses(it, static_cast<int>(blockIdx.y), p.ctas, p.cache.kv_heads, p.tokens)) return;
    const auto slot = [&](int s) { return prompt_slot(p, D, s == 0 ? it.slot : 2 * (static_cast<int>(blockIdx.y) + s)); };
    constexpr int kPieces = D / 32;  // of four columns, 32 columns apart
    const int row = static_cast<int>(blockIdx.x) * kJoinRows + static_cast<int>(threadIdx.x) / 8;
    const int lane = threadIdx.x % 8, tok = row % 128 / p.group, token = it.token0 + row / 128 * p.tile_tokens + tok;
    if (tok >= p.tile_tokens || token >= it.n) return;
    float top = -INFINITY, sum = 0.0f, acc[kPieces][4] = {};
#pragma unroll 4
    for (int s = 0; s < it.ctas; ++s) {
        const float2 ml = *reinterpret_cast<const float2 *>(slot(s) + 256 * D + 2 * row);
        if (ml.x == -INFINITY && ml.y == 0.0f) continue;  // a part whose keys the row does not see: it has no sums
        float f[kPieces][4];
#pragma unroll
        for (int q = 0; q < kPieces; ++q) load_floats(slot(s) + row * D + 32 * q + 4 * lane, f[q]);
        const float to = fmaxf(top, ml.x), old = top == -INFINITY ? 0.0f : exp2_fast(top - to), w = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - to);
        top = to;
        sum = sum * old + w * ml.y;
#pragma unroll
        for (int q = 0; q < kPieces; ++q)
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[q][x] = acc[q][x] * old + w * f[q][x];
    }
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    T *out = static_cast<T *>(p.out) + static_cast<long long>(it.begin + token) * p.out_ld + static_cast<long long>(it.head * p.group + row % 128 - tok * p.group) * D + 4 * lane;
#pragma unroll
    for (int q = 0; q < kPieces; ++q)
        *reinterpret_cast<uint2 *>(out + 32 * q) = make_uint2(pack16<T>(acc[q][0] * inv, acc[q][1] * inv), pack16<T>(acc[q][2] * inv, acc[q][3] * inv));
}

// Tensor maps of the queries (rows of heads) and of keys or values (pages), 128-byte swizzle, boxes 64 values wide.
inline int make_attn_map(CUtensorMap *map, int type, const void *base, int rank, const cuuint64_t *dim, const cuuint64_t *stride, const cuuint32_t *box) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return cudaErrorNotSupported;
    const cuuint32_t step[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, type == DMM_T_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, static_cast<cuuint32_t>(rank),
                          const_cast<void *>(base), dim, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : cudaErrorInvalidValue;
}

template <class T, int D>
inline int launch_prompt_typed(PromptParams &p, int type, bool pdl, cudaStream_t stream) {
    using Plan = PromptPlan<D>;
    p.tile_tokens = 128 / p.group;
    CUtensorMap maps[3];
    {
        const cuuint64_t dim[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(p.heads), static_cast<cuuint64_t>(p.tokens)};
        const cuuint64_t stride[2] = {2ull * D, 2ull * static_cast<cuuint64_t>(p.q_ld)};
        const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(p.group), static_cast<cuuint32_t>(p.tile_tokens)};
        const int rc = make_attn_map(&maps[0], type, p.q, 3, dim, stride, box);
        if (rc) return rc;
    }
    const int page = 1 << p.cache.page_shift;
    for (int kv = 0; kv < 2; ++kv) {
        const cuuint64_t dim[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(page), static_cast<cuuint64_t>(p.cache.kv_heads),
                                   static_cast<cuuint64_t>(p.cache.num_pages)};
        // (the stride of a dimension of size 1 says nothing)
        const auto bytes = [](long long s, long long n) { return 2ull * static_cast<cuuint64_t>(n > 1 ? s : D); };
        const cuuint64_t stride[3] = {bytes(p.cache.row_stride, page), bytes(p.cache.head_stride, p.cache.kv_heads),
                                      bytes(p.cache.page_stride, p.cache.num_pages)};
        const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(page < kPromptKeys ? page : kPromptKeys), 1, 1};
        const int rc = make_attn_map(&maps[1 + kv], type, kv ? p.cache.v : p.cache.k, 4, dim, stride, box);
        if (rc) return rc;
    }
    // every sequence adds at most one pair of tiles that is not full
    const long long items = (p.tokens / (2 * p.tile_tokens) + static_cast<long long>(p.cache.num_seqs < p.tokens ? p.cache.num_seqs : p.tokens)) * p.cache.kv_heads;
    if (items > 0x3fffffff) return DMM_ERR_SHAPE;
    const auto kernel = prompt_attention_kernel<T, D>;
    static SmemAllowance allowance;
    const int rc = allowance.get(reinterpret_cast<const void *>(kernel), Plan::kBytes);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(items > p.ctas ? items : p.ctas));  // (even shares: a block for each CTA)
    cfg.blockDim = dim3(kPromptThreads);
    cfg.dynamicSmemBytes = Plan::kBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], maps[2], p);
    if (err != cudaSuccess) return err;
    cfg.gridDim = dim3(256 / kJoinRows, static_cast<unsigned>(p.ctas));
    cfg.blockDim = dim3(8 * kJoinRows);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, prompt_join_kernel<T, D>, p);
}

inline int launch_prompt(PromptParams &p, int type, int head_dim, bool pdl, cudaStream_t stream) {
    if (type == DMM_T_F16) return head_dim == 64 ? launch_prompt_typed<__half, 64>(p, type, pdl, stream) : launch_prompt_typed<__half, 128>(p, type, pdl, stream);
    return head_dim == 64 ? launch_prompt_typed<__nv_bfloat16, 64>(p, type, pdl, stream) : launch_prompt_typed<__nv_bfloat16, 128>(p, type, pdl, stream);
}

}  // namespace dmm
