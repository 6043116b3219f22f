// Block-selected attention: what its translation units share.
#pragma once

#include "mat_common.cuh"

namespace mat {

struct SelProblem {
    const void *q, *k, *v, *o, *dout;
    void *out, *dq, *dk, *dv;
    const float *lse_in;
    float *lse;
    int64_t B, S, H, Hkv, D;
    int dtype;
    const int32_t *blocks;
    int64_t block, topk, nb;
    int causal;
    float scale;
    cudaStream_t stream;
};

// Which queries chose a block, the selection turned round, for a group of (batch, key head) pairs: for pair bh of the group
// and block n the entries
// [base[bh * (nb + 1) + n], base[bh * (nb + 1) + n + 1]) of entry[bh * S * topk + ...], ascending, each
// query * topk + the place of the block in the query's list.
struct SelLists {
    int32_t *counts;   // [bh][tiles][nb] queries of a tile that chose a block, then their offset within the block's list
    int32_t *base;     // [bh][nb + 1]
    int32_t *entry;    // [bh][S * topk]
    int64_t tiles;
};
size_t sel_lists_bytes(int64_t pairs, int64_t S, int64_t nb, int64_t topk);
SelLists sel_lists_at(void *ws, int64_t pairs, int64_t S, int64_t nb, int64_t topk);
// Fills the lists of pairs [bh0, bh0 + pairs) and cuts each block's rows (entries x query heads of a key head) into items of
// rows_per_item: items[bh * max_items + x] = (block, first row) for x in [item_base[bh * (nb + 1) + n], ...[n + 1]).
int launch_sel_lists(const SelProblem &p, const SelLists &l, int64_t bh0, int64_t pairs, int2 *items, int32_t *item_base, int64_t max_items,
                     int rows_per_item);

// selected_tiles.cu
size_t sel_workspace_bytes(int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t D, int dtype, int64_t block, int64_t topk, bool bwd);
int launch_sel(const SelProblem &p, void *workspace, bool bwd);

// An entry of a query's list counts when it names a block of the sequence, is above every entry before it and, with
// causal, not behind the query's own block.  `prev` carries the largest entry so far (start at -1).
__device__ __forceinline__ bool sel_entry_counts(int n, int &prev, int limit) {
    if (n <= prev) return false;
    prev = n;
    return n < limit;
}

static inline size_t sel_align(size_t x) { return (x + 255) / 256 * 256; }

}  // namespace mat
