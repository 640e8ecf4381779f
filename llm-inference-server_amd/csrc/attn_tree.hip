// Attention of drafted token trees over the paged pool: the generic kernel and the extern "C" entry
// points.
//
// A node sees the sequence's cached keys, all of them, and of the drafted ones those whose bit is in
// its mask row:
//
//   out = sum_j w_j v_j / sum_j w_j,   w_j = e^(scale q.k_j) over the keys j that it sees; 0 if none
//
// Generic kernel: any block size, head_dim <= 512, GQA group, stride and softmax scale; it takes the
// shapes that the matrix kernels decline. A workgroup has one (token, query head). A lane holds 16
// dims of a key, LPK lanes a key, so that a wave has 64 / LPK keys side by side; each such group of
// lanes runs an online softmax of its own, in fp32, over every so-manieth key, and the groups meet at
// the end. A group whose sums are not finite walks its keys once more, takes what of V is not finite, and keeps that
// however little the key weighs. Bound: vector instructions and the latency of a step's loads (8 sequences of 16 nodes behind 4,000
// keys, 16/4 heads of 256, bf16: 500 us, fp32 1,440).
#include "prefill_common.h"
#include "tree.h"

namespace pkv {
namespace {

// (Token, head) pairs that get 16 waves each instead of 4.
constexpr int kGenericFew = 1024;

template <int L>
__device__ __forceinline__ float lanes_sum(float x) {
    x = quad_sum(x);
    if constexpr (L >= 8) x += dpp_f32<kDppRowHalfMirror>(x);
    if constexpr (L >= 16) x += dpp_f32<kDppRowMirror>(x);
    if constexpr (L >= 32) {
        const SwapPair s = swap16(x);
        x = s.a + s.b;
    }
    return x;
}

// WIDE: rows in 16-byte steps and head_dim a multiple of 16.
template <typename T, int LPK, bool WIDE>
__global__ __launch_bounds__(1024) void tree_generic_kernel(const TreeParams p) {
    constexpr int U = WIDE ? 2 : 1;           // keys of a group in a step
    constexpr int DP = 16 * LPK;              // dims that the lanes have room for
    __shared__ float s_m[16], s_l[16];
    __shared__ __attribute__((aligned(16))) float s_o[16 * DP];
    const int lane = lane_id(), sub = lane % LPK, d0 = 16 * sub;
    const int groups = (int)blockDim.x / LPK, group = (int)threadIdx.x / LPK;
    const int64_t tok = blockIdx.x;
    const int head = (int)blockIdx.y;
    // The last sequence with query_start_loc <= tok owns it; tokens past the last one belong to none.
    if (tok >= p.qsl[p.num_seqs]) return;
    int lo = 0, hi = p.num_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.qsl[mid] <= tok) lo = mid; else hi = mid;
    }
    const int seq = lo;
    const int64_t nodes = p.qsl[seq + 1] - p.qsl[seq];
    const int64_t cap = p.table_width * p.block_size;           // fits 31 bits
    const int64_t ctx = p.ctx_lens[seq];
    // (Without blocks all ids are bad: zeros, as without keys.)
    const int n_keys = (int)(ctx < 0 || p.num_blocks < 1 ? 0 : ctx < cap ? ctx : cap);
    const int64_t cached = ctx - nodes;
    const uint64_t* mask = p.masks + tok * p.mask_stride;
    const int kvh = head / p.group;
    const T* qrow = reinterpret_cast<const T*>(p.q) + tok * p.q_st + (int64_t)head * p.q_sh;
    float q[16], acc[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        q[e] = d0 + e < p.head_dim ? to_f32(qrow[d0 + e]) : 0.f;
        acc[e] = 0.f;
    }
    const T* kb = reinterpret_cast<const T*>(p.k) + kvh * p.sh;
    const T* vb = reinterpret_cast<const T*>(p.v) + kvh * p.sh;
    const int64_t* table = p.tables + (int64_t)seq * p.table_stride;
    // The lane's 16 dims of a row. Those past head_dim read the row's first ones: whole lanes (WIDE), whose share of a
    // score is left out and whose outputs are not stored, or elements, which are zeros.
    auto dims = [&](const T* row, float* x) {
        if constexpr (WIDE) {
            const T* at = row + (d0 < p.head_dim ? d0 : 0);
            constexpr int PER = 16 / sizeof(T);
#pragma unroll
            for (int i = 0; i < 16 / PER; ++i) {
                const Vec16 v = load16(at + i * PER);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    if constexpr (sizeof(T) == 4) {
                        x[4 * i + w] = __builtin_bit_cast(float, v.w[w]);
                    } else {
                        x[8 * i + 2 * w] = Pair<T>::lo(v.w[w]);
                        x[8 * i + 2 * w + 1] = Pair<T>::hi(v.w[w]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float at = to_f32(row[d0 + e < p.head_dim ? d0 + e : 0]);
                x[e] = d0 + e < p.head_dim ? at : 0.f;
            }
        }
    };
    float m = kNegInf, l = 0.f;
    for (int first = 0; first < n_keys; first += U * groups) {
        float k[U][16], v[U][16], dot[U], m_new = m;
        bool seen[U], good[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = first + u * groups + group;
            const uint32_t key = (uint32_t)(at < n_keys ? at : n_keys - 1);
            const int64_t node = (int64_t)key - cached;
            seen[u] = at < n_keys &&
                      (node < 0 || (node < 64ll * p.mask_words && (mask[node >> 6] >> (node & 63) & 1)));
            const uint32_t blk = p.block_shift >= 0 ? key >> p.block_shift : key / (uint32_t)p.block_size;
            const int64_t id = table[blk];
            good[u] = (uint64_t)id < (uint64_t)p.num_blocks;    // a bad id reads as zeros
            const int64_t row = (good[u] ? id : 0) * p.sb + (int64_t)(key - blk * (uint32_t)p.block_size) * p.ss;
            dims(kb + row, k[u]);
            dims(vb + row, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) x += q[e] * k[u][e];
            if (WIDE) x = d0 < p.head_dim ? x : 0.f;            // (0 * infinity)
            x = lanes_sum<LPK>(x);
            dot[u] = good[u] ? x : 0.f;
            if (seen[u]) m_new = fmaxf(m_new, dot[u] * p.scale_log2);
        }
        const float m_off = m_new == kNegInf ? 0.f : m_new;
        const float alpha = fast_exp2(m - m_off);               // 0 on the first keys (m = -inf)
        l *= alpha;
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] *= alpha;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // (One rounding: that of a large product would be the weight's.)
            const float pj = seen[u] ? fast_exp2(fmaf(dot[u], p.scale_log2, -m_off)) : 0.f;
            l += pj;
            // A key that is not seen does not reach the row, whatever it holds.
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e] += pj * (seen[u] && good[u] ? v[u][e] : 0.f);
        }
        m = m_new;
    }
    // What is not finite in V, for rows that see it: the sums may have lost it (0 * infinity is NaN).
    float any = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) any += acc[e] * 0.f;
    if (any != any && l == l) {
        float rest[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) rest[e] = 0.f;
        for (int key = group; key < n_keys; key += groups) {
            const int64_t node = (int64_t)key - cached;
            if (node >= 0 && (node >= 64ll * p.mask_words || !(mask[node >> 6] >> (node & 63) & 1))) continue;
            const uint32_t blk = p.block_shift >= 0 ? (uint32_t)key >> p.block_shift : (uint32_t)key / (uint32_t)p.block_size;
            const int64_t id = table[blk];
            if ((uint64_t)id >= (uint64_t)p.num_blocks) continue;
            float v[16];
            dims(vb + id * p.sb + (int64_t)((uint32_t)key - blk * (uint32_t)p.block_size) * p.ss, v);
#pragma unroll
            for (int e = 0; e < 16; ++e) rest[e] += fabsf(v[e]) < __builtin_huge_valf() ? 0.f : v[e];
        }
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (rest[e] != 0.f) acc[e] = rest[e];
    }
    // The wave's groups, then the waves.
    float M = m;
#pragma unroll
    for (int off = LPK; off < 64; off *= 2) M = fmaxf(M, __shfl_xor(M, off));
    const float a = fast_exp2(m - (M == kNegInf ? 0.f : M));
    l *= a;
#pragma unroll
    for (int off = LPK; off < 64; off *= 2) l += __shfl_xor(l, off);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        acc[e] = share_of(acc[e], a);
#pragma unroll
        for (int off = LPK; off < 64; off *= 2) acc[e] += __shfl_xor(acc[e], off);
    }
    const int wave = (int)threadIdx.x >> 6, waves = (int)blockDim.x >> 6;
    if (lane < LPK)
#pragma unroll
        for (int e = 0; e < 16; ++e) s_o[wave * DP + d0 + e] = acc[e];
    if (lane == 0) {
        s_m[wave] = M;
        s_l[wave] = l;
    }
    __syncthreads();
    T* orow = reinterpret_cast<T*>(p.out) + tok * p.out_st + (int64_t)head * p.out_sh;
    for (int d = (int)threadIdx.x; d < p.head_dim; d += (int)blockDim.x) {
        float top = kNegInf, L = 0.f, o = 0.f;
        for (int w = 0; w < waves; ++w) top = fmaxf(top, s_m[w]);
        if (top == kNegInf) top = 0.f;
        for (int w = 0; w < waves; ++w) {
            const float b = fast_exp2(s_m[w] - top);
            L += b * s_l[w];
            o += share_of(s_o[w * DP + d], b);
        }
        // (No key, or weights of 0 alone: o is 0 where it is finite.)
        orow[d] = from_f32<T>(L == 0.f ? o : o / L);
    }
}

template <typename T, int LPK>
int launch_generic_l(const TreeParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)p.num_tokens, (unsigned)p.num_heads);
    const int threads = p.num_tokens * p.num_heads <= kGenericFew ? 1024 : 256;
    const uint64_t rows = (uint64_t)(uintptr_t)p.k | (uint64_t)(uintptr_t)p.v | (uint64_t)(p.sb * sizeof(T)) |
                          (uint64_t)(p.ss * sizeof(T)) | (uint64_t)(p.sh * sizeof(T));
    if (rows % 16 == 0 && p.head_dim % 16 == 0) tree_generic_kernel<T, LPK, true><<<grid, threads, 0, stream>>>(p);
    else tree_generic_kernel<T, LPK, false><<<grid, threads, 0, stream>>>(p);
    return check_launch("tree attention, generic");
}

template <typename T>
int launch_generic_t(const TreeParams& p, hipStream_t stream) {
    if (p.head_dim <= 64) return launch_generic_l<T, 4>(p, stream);
    if (p.head_dim <= 128) return launch_generic_l<T, 8>(p, stream);
    if (p.head_dim <= 256) return launch_generic_l<T, 16>(p, stream);
    return launch_generic_l<T, 32>(p, stream);
}

}  // namespace

// How the matrix kernels take a batch: rows a workgroup, and runs that contexts are cut into (splits = 1:
// none), with the workspace that takes.
struct TreePlan : SplitPlan {
    int row_waves;
};

// The cheapest of a few run lengths in a model of the launch, in us: a workgroup takes kStart before and
// after its tiles, a tile's time depends on how full the GPU is; once there are more workgroups than slots
// the last ones, the shortest, start late, a third of a workgroup's time on average; a split launch adds the merge kernel and
// its partials' way to memory and back.
TreePlan tree_plan(int64_t num_seqs, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t num_tokens,
                   int64_t max_query_len, int dtype, const int64_t* ctx, const int64_t* qlen) {
    constexpr float kStart = 6.f, kMerge = 4.f, kBytesPerUs = 4.5e6f, kWorth = 0.9f;
    constexpr int64_t kMaxBytes = 128 << 20;     // of workspace
    static const int kRuns[] = {2, 3, 4, 5, 6, 8, 10, 12, 14, 17, 20, 24, 28, 34, 40, 48, 56, 68, 80, 96, 112, 136, 160, 192};
    TreePlan plan = {};
    plan.splits = 1;
    plan.split_tiles = 0x7fffffff;
    const int64_t group = num_heads / num_kv_heads;
    const int64_t most = (max_query_len && max_query_len < num_tokens ? max_query_len : num_tokens) * group;
    const bool f32 = dtype == PKV_FLOAT32;
    const int64_t wave_rows = f32 ? 16 : 32;
    // (fp32: its tiles of 32 keys have no 16 for each of four waves, and two workgroups of 16 rows beat one of 32.)
    plan.row_waves = most <= 32 && (!f32 || head_dim <= 64) ? 1 : most <= 64 ? 2 : 4;
    if (!ctx || !qlen || num_seqs > kPrefillSortSeqs) return plan;
    const int64_t rows_of_wg = wave_rows * plan.row_waves;
    const int64_t keys = f32 ? (head_dim <= 64 ? 64 : 32) : plan.row_waves == 1 ? 128 : 64;
    // Workgroups that the GPU holds, by LDS and by registers; us a tile, alone and in a full GPU.
    const int64_t lds = (f32 ? 16 : 8) * keys * head_dim;
    const int64_t slots = 256 * (lds <= 72 * 1024 ? 2 : 1);
    float alone = plan.row_waves == 4 ? 1.4f : 1.2f;
    float full = plan.row_waves == 4 ? 2.4f : (float)(slots * lds / 2) / 5.5e6f;
    if (f32) {
        // 64 keys of 16 rows: 2 * 64 * 16 * head_dim products at 64 a cycle, shared by the waves of the rows.
        alone = 0.5f + (float)(keys * head_dim) * plan.row_waves / 4.f * 2.2e-4f;
        full = 2.f * alone - 0.5f;
    }
    auto launch_us = [&](int64_t wgs, int64_t longest, int64_t work) {
        const float fill = wgs < slots ? (float)wgs / slots : 1.f;
        const float tile = full > alone ? alone + (full - alone) * fill : alone;
        const float one = longest * tile + kStart;
        if (wgs <= slots) return one;
        const float all = (work * tile + wgs * kStart) / slots + 0.35f * one;
        return all > one ? all : one;
    };
    int64_t wgs = 0, work = 0, longest = 0;
    auto each = [&](auto f) {
        for (int64_t i = 0; i < num_seqs; ++i) {
            if (ctx[i] <= 0 || qlen[i] <= 0) continue;
            const int64_t c = ctx[i] < (1ll << 36) ? ctx[i] : 1ll << 36;
            f(ceil_div(c, keys), ceil_div(qlen[i] * group, rows_of_wg) * num_kv_heads, qlen[i] * num_heads);
        }
    };
    each([&](int64_t tiles, int64_t w, int64_t) {
        wgs += w;
        work += w * tiles;
        longest = longest > tiles ? longest : tiles;
    });
    const int64_t rows = num_tokens * num_heads;
    float best = kWorth * launch_us(wgs, longest, work);
    for (const int64_t run : kRuns) {
        if (run >= longest) break;
        const int64_t splits = ceil_div(longest, run);
        if (kMergeCounterBytes + 3 * 256 + rows * 4 + rows * splits * (head_dim + 2) * 4 > kMaxBytes) continue;
        int64_t items = 0, top = 0, parts = 0;
        each([&](int64_t tiles, int64_t w, int64_t r) {
            const int64_t n = ceil_div(tiles, run), even = ceil_div(tiles, n);
            items += w * n;
            top = top > even ? top : even;
            parts += n > 1 ? r * n : 0;
        });
        const float us = launch_us(items, top, work) + kMerge + 2.f * parts * (head_dim + 2) * 4 / kBytesPerUs;
        if (us >= best) continue;
        best = us;
        plan.splits = (int)splits;
        plan.split_tiles = (int)run;
        plan.items = items;
    }
    if (plan.splits == 1) return plan;
    auto round256 = [](int64_t b) { return ceil_div(b, 256) * 256; };
    plan.rows_bytes = round256(rows * 4);
    plan.ml_bytes = round256(rows * plan.splits * 8);
    plan.o_bytes = round256(rows * plan.splits * head_dim * 4);
    return plan;
}

// Whether the matrix kernels take these parameters.
bool tree_tiled(const TreeParams& p, int dtype) {
    const int64_t isz = dtype == PKV_FLOAT32 ? 4 : 2;
    if (!prefill_shape(p.block_size, p.head_dim, PKV_FLOAT16) || p.num_blocks < 1 || p.ss < 0) return false;
    // They mask to -inf and take the maximum before they scale.
    if (!(p.scale > 0.f)) return false;
    // One grid dimension; keys and rows of a sequence in 32 bits.
    const int rows_of_wg = (dtype == PKV_FLOAT32 ? 16 : 32) * p.row_waves;
    if (tree_workgroups(p, rows_of_wg) > 0x7fffffff || p.table_width * p.block_size > (1 << 30)) return false;
    if (((int64_t)p.max_query_len + 128) * p.group > 0x7fffffff) return false;
    const uint64_t probe = (uint64_t)(uintptr_t)p.q | (uint64_t)(uintptr_t)p.k | (uint64_t)(uintptr_t)p.v |
                           (uint64_t)(uintptr_t)p.out | (uint64_t)(p.q_st * isz) | (uint64_t)(p.q_sh * isz) |
                           (uint64_t)(p.sb * isz) | (uint64_t)(p.ss * isz) | (uint64_t)(p.sh * isz) |
                           (uint64_t)(p.out_st * isz) | (uint64_t)(p.out_sh * isz);
    return probe % 16 == 0;
}

int launch_tree_generic(const TreeParams& p, int dtype, hipStream_t stream) {
    switch (dtype) {
        case PKV_FLOAT32: return launch_generic_t<float>(p, stream);
        case PKV_FLOAT16: return launch_generic_t<_Float16>(p, stream);
        default: return launch_generic_t<bf16_t>(p, stream);
    }
}

}  // namespace pkv

using namespace pkv;

extern "C" int64_t pkv_tree_attention_workspace_bytes(int64_t num_seqs, int64_t num_heads, int64_t num_kv_heads,
                                                      int64_t head_dim, int64_t num_tokens, int64_t max_query_len,
                                                      int dtype, const int64_t* host_context_lens,
                                                      const int64_t* host_query_lens) {
    if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || num_tokens <= 0 ||
        num_seqs > 0x7fffffff || num_tokens > 0x7fffffff || num_heads > 65535 || num_heads % num_kv_heads)
        return 0;
    const TreePlan plan = tree_plan(num_seqs, num_heads, num_kv_heads, head_dim, num_tokens, max_query_len, dtype,
                                    host_context_lens, host_query_lens);
    return plan.splits > 1 ? kMergeCounterBytes + plan.total() : 0;
}

extern "C" int pkv_tree_attention(
    void* out, int64_t out_stride_t, int64_t out_stride_h, const void* query, int64_t q_stride_t, int64_t q_stride_h,
    const void* k_pool, const void* v_pool, int64_t pool_stride_block, int64_t pool_stride_slot,
    int64_t pool_stride_head, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads, int64_t head_dim,
    const int64_t* block_tables, int64_t table_stride, int64_t table_width, const int64_t* context_lens,
    const int64_t* query_start_loc, const int64_t* masks, int64_t mask_stride, int64_t mask_words, int64_t num_seqs,
    int64_t num_heads, int64_t num_tokens, int64_t max_query_len, const int64_t* host_context_lens,
    const int64_t* host_query_lens, float scale, int dtype, void* workspace, int64_t workspace_bytes,
    hipStream_t stream) {
    clear_error();
    if (dtype != PKV_FLOAT32 && dtype != PKV_FLOAT16 && dtype != PKV_BFLOAT16)
        return fail(PKV_EINVAL, "tree_attention: unknown dtype %d", dtype);
    if (num_seqs < 0 || num_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 ||
        num_blocks < 0 || table_width < 0 || max_query_len < 0 || mask_words < 0 || mask_stride < mask_words)
        return fail(PKV_EINVAL, "tree_attention: bad sizes");
    if (num_heads % num_kv_heads)
        return fail(PKV_EINVAL, "tree_attention: %lld query heads not divisible by %lld kv heads",
                    (long long)num_heads, (long long)num_kv_heads);
    if (num_seqs > 0x7fffffff || num_tokens > 0x7fffffff || num_heads > 65535 || head_dim > 512 ||
        block_size > 0x7fffffff || table_width > 0x7fffffff / block_size || mask_words > 0x1ffffff)
        return fail(PKV_EUNSUPPORTED, "tree_attention: sizes beyond what the kernels index");
    if (num_tokens == 0 || num_seqs == 0) return PKV_OK;
    if (!out || !query || !k_pool || !v_pool || !context_lens || !query_start_loc || (!masks && mask_words > 0) ||
        (!block_tables && table_width > 0))
        return fail(PKV_EINVAL, "tree_attention: null pointer");
    TreeParams p = {};
    p.out = out;
    p.out_st = out_stride_t;
    p.out_sh = out_stride_h;
    p.q = query;
    p.q_st = q_stride_t;
    p.q_sh = q_stride_h;
    p.k = k_pool;
    p.v = v_pool;
    p.sb = pool_stride_block;
    p.ss = pool_stride_slot;
    p.sh = pool_stride_head;
    p.num_blocks = num_blocks;
    p.block_size = (int)block_size;
    p.block_shift = block_size & (block_size - 1) ? -1 : 63 - __builtin_clzll((unsigned long long)block_size);
    p.num_kv_heads = (int)num_kv_heads;
    p.head_dim = (int)head_dim;
    p.tables = block_tables;
    p.table_stride = table_stride;
    p.table_width = table_width;
    p.ctx_lens = context_lens;
    p.qsl = query_start_loc;
    p.masks = reinterpret_cast<const uint64_t*>(masks);
    p.mask_stride = mask_stride;
    p.mask_words = (int)mask_words;
    p.num_seqs = (int)num_seqs;
    p.num_heads = (int)num_heads;
    p.group = (int)(num_heads / num_kv_heads);
    p.num_tokens = num_tokens;
    p.max_query_len = (int)(max_query_len && max_query_len < num_tokens ? max_query_len : num_tokens);
    p.scale = scale;
    p.scale_log2 = scale * kLog2e;
    p.splits = 1;
    p.split_tiles = 0x7fffffff;
    const TreePlan plan = tree_plan(num_seqs, num_heads, num_kv_heads, head_dim, num_tokens, p.max_query_len, dtype,
                                    host_context_lens, host_query_lens);
    p.row_waves = plan.row_waves;
    if (!tree_tiled(p, dtype)) return launch_tree_generic(p, dtype, stream);
    if (plan.splits > 1 && workspace && workspace_bytes >= kMergeCounterBytes + plan.total()) {
        // Behind the decode calls' counters, which stay zero.
        char* ws = reinterpret_cast<char*>(workspace) + kMergeCounterBytes;
        p.splits = plan.splits;
        p.split_tiles = plan.split_tiles;
        p.split_items = plan.items;
        p.ws_rows = reinterpret_cast<int*>(ws);
        p.ws_ml = reinterpret_cast<float*>(ws + plan.rows_bytes);
        p.ws_o = reinterpret_cast<float*>(ws + plan.rows_bytes + plan.ml_bytes);
    }
    switch (dtype) {
        case PKV_FLOAT32: return launch_tree_f32(p, stream);
        case PKV_FLOAT16: return launch_tree_mfma<_Float16>(p, stream);
        default: return launch_tree_mfma<bf16_t>(p, stream);
    }
}
