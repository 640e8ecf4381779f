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

// Row tiles of `rows` rows that a sequence has at most.
inline int64_t tree_row_tiles(const TreeParams& p, int rows) { return ceil_div((int64_t)p.max_query_len * p.group, rows); }

// Workgroups of `rows` rows: the splits' items, or room for every row tile the batch can hold (a
// sequence's last one may be partial), whichever is more; whole rounds of tree_item's deal.
inline int64_t tree_workgroups(const TreeParams& p, int rows) {
    const int64_t most = tree_row_tiles(p, rows);
    const int64_t grid = most * p.num_seqs;
    const int64_t fill = p.num_tokens * p.group / rows + p.num_seqs;
    int64_t items = (grid < fill || p.num_seqs > kPrefillSortSeqs ? grid : fill) * p.num_kv_heads;
    if (p.splits > 1 && p.split_items > items) items = p.split_items;
    return ceil_div(items, 8 * most) * 8 * most;
}

// This workgroup's item (256 threads, all of them call it: it may hold two barriers). False: none.
// Items are numbered row tile fastest, then KV head, then split, then sequence, the longest context
// first whatever its head, and dealt to the XCDs (the hardware hands workgroup L to XCD L % 8) in turn, as
// many at a time as a sequence has row tiles at most: those share K and V, and so an L2. Contiguous
// eighths, as prompts are numbered, put long contexts of some heads behind others' short ones: with few
// workgroups, one a CU, the last ones started late (32 sequences of 16-990 keys, 12 fp32 heads of 64: the
// CUs were busy for 58% of 55 us).
template <int ROWS, int KEYS>
__device__ __forceinline__ bool tree_item(const TreeParams& p, PrefillItem& r) {
    const int t = (int)threadIdx.x, lane = t & 63;
    const uint32_t G = (uint32_t)p.group, K = (uint32_t)p.num_kv_heads;
    const uint32_t deal = ((uint32_t)p.max_query_len * G + ROWS - 1) / ROWS;
    const uint32_t xcd = blockIdx.x % 8, at = blockIdx.x / 8;
    const uint32_t item = (at / deal * 8 + xcd) * deal + at % deal;
    const int64_t cap = p.table_width * p.block_size;
    if (p.num_seqs > kPrefillSortSeqs) {
        // Index order over the full rectangle, never split.
        const uint32_t per_seq = deal * K;
        if (item >= per_seq * (uint32_t)p.num_seqs) return false;
        r.seq = (int)(item / per_seq);
        r.kvh = (int)(item % per_seq / deal);
        r.row_tile = (int)(item % deal);
        r.split = 0;
        r.splits = 1;
        r.q_first = p.qsl[r.seq];
        r.q_len = (int)(p.qsl[r.seq + 1] - r.q_first);
        const int64_t c = p.ctx_lens[r.seq];
        r.ctx = (int)(c < cap ? c : cap);
        return r.row_tile * ROWS < r.q_len * (int)G;
    }
    // Up to a wave of sequences: every wave for itself, without LDS or a barrier.
    const bool in_wave = p.num_seqs <= 64;
    const int s = in_wave ? lane : t;
    int64_t q_first = 0;
    int q_len = 0, ctx = 0, key = -1;
    uint32_t tiles = 0, items = 0;                 // of the sequence, all KV heads
    if (s < p.num_seqs) {
        const int64_t c = p.ctx_lens[s];
        q_first = p.qsl[s];
        q_len = (int)(p.qsl[s + 1] - q_first);
        ctx = (int)(c < cap ? c : cap);
        tiles = q_len > 0 ? ((uint32_t)q_len * G + ROWS - 1) / ROWS : 0;
        items = tiles * K * (uint32_t)split_count((ctx + KEYS - 1) / KEYS, p.splits, p.split_tiles);
        // Longest context first, ties by index (contexts of 2^23 tokens count as tied).
        const int k = ctx < 0 ? 0 : ctx < (1 << 23) ? ctx : (1 << 23) - 1;
        key = k << 8 | (255 - s);
    }
    const bool cut = p.splits > 1;
    uint32_t before = 0, total = 0, uncut_before = 0;
    if (in_wave) {
        for (int u = 0; u < p.num_seqs; ++u) {
            const bool first = __builtin_amdgcn_readlane(key, u) > key;
            const uint32_t iu = (uint32_t)__builtin_amdgcn_readlane((int)items, u);
            total += iu;
            before += first ? iu : 0;
            if (cut) uncut_before += first ? (uint32_t)__builtin_amdgcn_readlane((int)(tiles * K), u) : 0;
        }
    } else {
        __shared__ uint4 s_seq[kPrefillSortSeqs];  // one LDS read a step of the loop below
        if (t < p.num_seqs) s_seq[t] = make_uint4((uint32_t)key, items, tiles * K, 0u);
        __syncthreads();
#pragma unroll 4
        for (int u = 0; u < p.num_seqs; ++u) {
            const uint4 o = s_seq[u];
            const bool first = (int)o.x > key;
            total += o.y;
            before += first ? o.y : 0;
            uncut_before += first ? o.z : 0;
        }
    }
    r.splits = p.splits;
    if (cut && total > gridDim.x) {
        // Longer contexts than the grid was sized for: unsplit.
        r.splits = 1;
        before = uncut_before;
        items = tiles * K;
    }
    const uint32_t in_seq = item - before;         // wraps below the sequence's first
    const bool mine = s < p.num_seqs && in_seq < items;
    if (mine) {
        r.split = (int)(in_seq / (tiles * K));
        r.kvh = (int)(in_seq % (tiles * K) / tiles);
        r.row_tile = (int)(in_seq % tiles);
    }
    bool found;
    if (in_wave) {
        const uint64_t lanes = __builtin_amdgcn_ballot_w64(mine);
        found = lanes != 0;
        const int src = found ? __builtin_ctzll(lanes) : 0;
        r = PrefillItem{src,
                        __builtin_amdgcn_readlane(r.kvh, src),
                        __builtin_amdgcn_readlane(r.split, src),
                        __builtin_amdgcn_readlane(r.row_tile, src),
                        __builtin_amdgcn_readlane(q_len, src),
                        __builtin_amdgcn_readlane(ctx, src),
                        __builtin_amdgcn_readlane(r.splits, src),
                        readlane64(q_first, src)};
    } else {
        __shared__ PrefillItem s_pick;
        __shared__ int s_found;
        if (t == 0) s_found = 0;
        __syncthreads();
        if (mine) {
            s_pick = PrefillItem{t, r.kvh, r.split, r.row_tile, q_len, ctx, r.splits, q_first};
            s_found = 1;
        }
        __syncthreads();
        found = s_found != 0;
        r = s_pick;
    }
    if (!__builtin_amdgcn_readfirstlane((int)found)) return false;
    // Uniform: into scalar registers.
    r.seq = __builtin_amdgcn_readfirstlane(r.seq);
    r.kvh = __builtin_amdgcn_readfirstlane(r.kvh);
    r.split = __builtin_amdgcn_readfirstlane(r.split);
    r.row_tile = __builtin_amdgcn_readfirstlane(r.row_tile);
    r.q_len = __builtin_amdgcn_readfirstlane(r.q_len);
    r.ctx = __builtin_amdgcn_readfirstlane(r.ctx);
    r.splits = __builtin_amdgcn_readfirstlane(r.splits);
    r.q_first = readlane64(r.q_first, 0);
    return true;
}

// The matrix kernels: 16-bit pools (tree_mfma.h), rows of 32 a wave, and fp32 pools (attn_tree_f32.hip), of 16.
template <typename T>
int launch_tree_mfma(const TreeParams& p, hipStream_t stream);
int launch_tree_f32(const TreeParams& p, hipStream_t stream);
// Keys of an fp32 tile: two workgroups a CU.
template <int D>
constexpr int kTreeKeysF32 = D <= 64 ? 64 : 32;

// The kernel for any shape.
int launch_tree_generic(const TreeParams& p, int dtype, hipStream_t stream);

}  // namespace pkv
