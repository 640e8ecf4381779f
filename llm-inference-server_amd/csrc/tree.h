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
    int64_t max_context_len;
};

// The kernel for any shape.
int launch_tree_generic(const TreeParams& p, int dtype, hipStream_t stream);

}  // namespace pkv
