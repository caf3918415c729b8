// What a CTA of the prompt kernel works on, as CTAs that share an item hand it to the kernel that joins their parts.  No CUDA in here,
// so that a test can compile and check it without a GPU.
#pragma once

#ifdef __CUDACC__
#define DMM_HOST_DEVICE __host__ __device__
#else
#define DMM_HOST_DEVICE
#endif

namespace dmm {

// A pair of tiles of one key head, or a part of its key tiles.
struct PromptItem {
    int seq, head, begin, n, len, token0;  // token0: first token of tile 0 within the sequence's new tokens
    int first, end;                        // key tiles
    int slot;                              // of the workspace, for a part; -1 for the whole
    int ctas;                              // for the first part: how many CTAs have one
};

// Whether `it` is an item that can begin in CTA x of `ctas` and go on in others: a record that was written follows from the tables
// of the call and is; of one that was not, because a wait gave up before, nothing is known, and no address may come from it.  What passes
// lies within the 2 * ctas slots of the workspace, the key heads and the `tokens` rows.
DMM_HOST_DEVICE inline bool prompt_item_crosses(const PromptItem &it, int x, int ctas, int kv_heads, int tokens) {
    return it.ctas > 1 && it.ctas <= ctas - x && it.slot == 2 * x + 1 && it.head >= 0 && it.head < kv_heads && it.n > 0 && it.n <= tokens &&
           it.begin >= 0 && it.begin <= tokens - it.n && it.token0 >= 0 && it.token0 < it.n;
}

}  // namespace dmm
