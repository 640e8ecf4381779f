// Attention of drafted token trees: what its kernels share (internal to libpagedkv).
#pragma once

#include "attention.h"

namespace pkv {

// AttnParams (qsl set) with the nodes' masks: bit j % 64 of word j / 64 of row t says whether token t
// sees node j of its sequence, the key at position context - query length + j. Keys before those are
// seen by all.
struct TreeParams : AttnParams {
    const uint64_t* masks;
    int64_t mask_stride;                 // words between rows
    int mask_words;
    int row_waves;                       // of a workgroup's four waves, those with rows of their own: 1, 2, 4
};

// Workgroups of `rows` rows: the splits' items, or room for every row tile the batch can hold (a
// sequence's last one may be partial), whichever is more; a multiple of 8.
inline int64_t tree_workgroups(const TreeParams& p, int rows) {
    const int64_t grid = ceil_div((int64_t)p.max_query_len * p.group, rows) * p.num_seqs;
    const int64_t fill = p.num_tokens * p.group / rows + p.num_seqs;
    int64_t items = (grid < fill || p.num_seqs > kPrefillSortSeqs ? grid : fill) * p.num_kv_heads;
    if (p.splits > 1 && p.split_items > items) items = p.split_items;
    return ceil_div(items, 8) * 8;
}

// The matrix kernels (tree_mfma.h).
template <typename T>
int launch_tree_mfma(const TreeParams& p, hipStream_t stream);

// The kernel for any shape.
int launch_tree_generic(const TreeParams& p, int dtype, hipStream_t stream);

}  // namespace pkv
