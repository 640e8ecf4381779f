// Attention over the 8-bit paged cache: the generic kernel and the extern "C" entry points.
//
// Generic kernel: any block size, head_dim <= 512, GQA group, stride and softmax scale; it takes
// the shapes that the matrix kernels decline. A workgroup has one (token, query head). A lane holds
// 16 dims of a key, LPK lanes a key, so that a wave has 64 / LPK keys side by side; each such group
// of lanes runs an online softmax of its own, in fp32, over every so-manieth key, and the groups
// meet at the end. Bound: vector instructions (a code is converted and multiplied by itself), and
// in small batches the latency of a step's loads, block ids and then rows: they go out for several
// keys together, the next ids with them, and small batches get 16 waves a workgroup instead of 4.
// Measured at 16/4 heads of 256, us a call: 8 sequences of 4k keys 66 (67 MB: 1.0 TB/s; one wave a
// head, a key a step, took 8,332), 64 of them 262 (2.0 TB/s), one of 60,000 789, 2 of 200 new tokens
// behind 2,000 635; 64 sequences of 500, 8 heads of 40, 19.6.
#include "kv8.h"

namespace pkv {
namespace {

// (Token, head) pairs that get 16 waves each: 8 sequences of 4k at 16 heads took 179 us with 16 and 482
// with 4 before lanes held 16 dims, 64 of them the same with both; 1,024 tokens of prompts 422 and 194.
constexpr int kGenericFew = 1024;

template <int L>
__device__ __forceinline__ float group_sum(float x) {
    x = quad_sum(x);
    if constexpr (L >= 8) x += dpp_f32<kDppRowHalfMirror>(x);
    if constexpr (L >= 16) x += dpp_f32<kDppRowMirror>(x);
    if constexpr (L >= 32) {
        const SwapPair s = swap16(x);
        x = s.a + s.b;
    }
    return x;
}

// ALIGN: of codes, 1, 4 or 16; head_dim is a multiple of it.
template <typename T, int LPK, int ALIGN>
__global__ __launch_bounds__(1024) void kv8_generic_kernel(const Kv8Params p) {
    constexpr int U = ALIGN == 16 ? 4 : ALIGN == 4 ? 2 : 1;   // keys of a group in a step: what registers have room for
    constexpr int DP = 16 * LPK;              // dims that the lanes have room for
    __shared__ float s_m[16], s_l[16];
    __shared__ __attribute__((aligned(16))) float s_o[16 * DP];
    const int lane = lane_id(), sub = lane % LPK, d0 = 16 * sub;
    const int groups = (int)blockDim.x / LPK, group = (int)threadIdx.x / LPK;
    const int64_t tok = blockIdx.x;
    const int head = (int)blockIdx.y;
    int seq = (int)tok;
    int64_t q_start = tok, q_len = 1;
    if (p.qsl) {
        // The last sequence with query_start_loc <= tok owns it; tokens past the last one
        // belong to no sequence.
        if (tok >= p.qsl[p.num_seqs]) return;
        int lo = 0, hi = p.num_seqs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.qsl[mid] <= tok) lo = mid; else hi = mid;
        }
        seq = lo;
        q_start = p.qsl[seq];
        q_len = p.qsl[seq + 1] - q_start;
    }
    const int64_t cap = p.table_width * p.block_size;           // fits 31 bits
    const int64_t sees = p.ctx_lens[seq] - q_len + (tok - q_start) + 1;
    // (Without blocks all ids are bad: zeros, as without keys.)
    const int n_keys = (int)(sees < 0 || p.num_blocks < 1 ? 0 : sees < cap ? sees : cap);
    const int kvh = head / p.group;
    const T* qrow = reinterpret_cast<const T*>(p.q) + tok * p.q_st + (int64_t)head * p.q_sh;
    float q[16], acc[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        q[e] = d0 + e < p.head_dim ? to_f32(qrow[d0 + e]) : 0.f;
        acc[e] = 0.f;
    }
    const uint8_t* kc = reinterpret_cast<const uint8_t*>(p.k) + kvh * p.sh;
    const uint8_t* vc = reinterpret_cast<const uint8_t*>(p.v) + kvh * p.sh;
    const uint8_t* ksb = p.ks + kvh * p.ssh;
    const uint8_t* vsb = p.vs + kvh * p.ssh;
    const int64_t* table = p.tables + (int64_t)seq * p.table_stride;
    // The lane's codes of a row. No load stands in a branch, where it would be waited for by itself:
    // dims past head_dim read the row's first ones (against queries of 0, into outputs that are not
    // stored).
    auto codes = [&](const uint8_t* row) {
        auto from = [&](int d) { return row + (d < p.head_dim ? d : 0); };
        if constexpr (ALIGN == 16) return load16(from(d0));
        Vec16 x;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if constexpr (ALIGN == 4) {
                x.w[w] = *reinterpret_cast<const uint32_t*>(from(d0 + 4 * w));
            } else {
                x.w[w] = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) x.w[w] |= (uint32_t)*from(d0 + 4 * w + e) << (8 * e);
            }
        }
        return x;
    };
    // Key u of a group's step from `first`; past the last key, that one again, of weight 0.
    auto key_of = [&](int64_t first, int u) {
        const int64_t key = first + u * groups + group;
        return (uint32_t)(key < n_keys ? key : n_keys - 1);
    };
    auto block_of = [&](uint32_t key) {
        return p.block_shift >= 0 ? key >> p.block_shift : key / (uint32_t)p.block_size;
    };
    float m = kNegInf, l = 0.f;
    int64_t ids[U];
    if (n_keys > 0)
#pragma unroll
        for (int u = 0; u < U; ++u) ids[u] = table[block_of(key_of(0, u))];
    for (int64_t first = 0; first < n_keys; first += U * groups) {
        Vec16 k[U], v[U];
        uint32_t ks[U], vs[U], good = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t key = key_of(first, u);
            const bool ok = (uint64_t)ids[u] < (uint64_t)p.num_blocks;  // a bad id reads as zeros
            good |= ok ? 1u << u : 0u;
            const int64_t id = ok ? ids[u] : 0;
            const int64_t at = key - block_of(key) * (uint32_t)p.block_size;
            const int64_t row = id * p.sb + at * p.ss, sc = id * p.ssb + at * p.sss;
            ks[u] = ksb[sc];
            vs[u] = vsb[sc];
            k[u] = codes(kc + row);
            v[u] = codes(vc + row);
        }
        if (first + U * groups < n_keys)
#pragma unroll
            for (int u = 0; u < U; ++u) ids[u] = table[block_of(key_of(first + U * groups, u))];
        float s[U], m_new = m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)k[u].w[w], false);
                const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)k[u].w[w], true);
                x += q[4 * w] * lo[0];
                x += q[4 * w + 1] * lo[1];
                x += q[4 * w + 2] * hi[0];
                x += q[4 * w + 3] * hi[1];
            }
            x = group_sum<LPK>(x) * scale_of(ks[u]) * p.scale_log2;
            x = good >> u & 1 ? x : 0.f;
            s[u] = first + u * groups + group < n_keys ? x : kNegInf;
            m_new = fmaxf(m_new, s[u]);
        }
        const float m_off = m_new == kNegInf ? 0.f : m_new;
        const float alpha = fast_exp2(m - m_off);               // 0 on the first keys (m = -inf)
        l *= alpha;
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] *= alpha;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool live = first + u * groups + group < n_keys, ok = good >> u & 1;
            const float pj = fast_exp2(s[u] - m_off), x = live && ok ? pj * scale_of(vs[u]) : 0.f;
            l += pj;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int c = (int)(ok ? v[u].w[w] : 0u);
                const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
                acc[4 * w] += x * lo[0];
                acc[4 * w + 1] += x * lo[1];
                acc[4 * w + 2] += x * hi[0];
                acc[4 * w + 3] += x * hi[1];
            }
        }
        m = m_new;
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
        acc[e] *= a;
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
            o += b * s_o[w * DP + d];
        }
        orow[d] = from_f32<T>(n_keys > 0 ? o / L : 0.f);        // a row without keys is zero
    }
}

template <typename T, int LPK>
int launch_generic_l(const Kv8Params& p, hipStream_t stream) {
    if (p.num_tokens > 0x7fffffff) return fail(PKV_EUNSUPPORTED, "kv8_attention: grid too large");
    const dim3 grid((unsigned)p.num_tokens, (unsigned)p.num_heads);
    const int threads = p.num_tokens * p.num_heads <= kGenericFew ? 1024 : 256;
    const uint64_t codes = (uint64_t)(uintptr_t)p.k | (uint64_t)(uintptr_t)p.v | (uint64_t)p.sb | (uint64_t)p.ss |
                           (uint64_t)p.sh | (uint64_t)p.head_dim;
    if (codes % 16 == 0) kv8_generic_kernel<T, LPK, 16><<<grid, threads, 0, stream>>>(p);
    else if (codes % 4 == 0) kv8_generic_kernel<T, LPK, 4><<<grid, threads, 0, stream>>>(p);
    else kv8_generic_kernel<T, LPK, 1><<<grid, threads, 0, stream>>>(p);
    return check_launch("kv8 generic attention");
}

template <typename T>
int launch_generic_t(const Kv8Params& p, hipStream_t stream) {
    if (p.head_dim <= 64) return launch_generic_l<T, 4>(p, stream);
    if (p.head_dim <= 128) return launch_generic_l<T, 8>(p, stream);
    if (p.head_dim <= 256) return launch_generic_l<T, 16>(p, stream);
    if (p.head_dim <= 512) return launch_generic_l<T, 32>(p, stream);
    return fail(PKV_EUNSUPPORTED, "kv8_attention: head_dim %d > 512", p.head_dim);
}

}  // namespace

int launch_kv8_generic(const Kv8Params& p, int dtype, hipStream_t stream) {
    switch (dtype) {
        case PKV_FLOAT32: return launch_generic_t<float>(p, stream);
        case PKV_FLOAT16: return launch_generic_t<_Float16>(p, stream);
        default: return launch_generic_t<bf16_t>(p, stream);
    }
}

// ------------------------------------------------------------------ decode
bool kv8_decode_applies(const Kv8Params& p, int dtype) {
    if (p.head_dim % 16 || p.head_dim < 32 || p.head_dim > 128 || p.block_shift < 2) return false;
    if (p.num_seqs > kKv8DecodeMaxSeqs || p.num_blocks < 1) return false;
    if ((int64_t)p.max_query_len * p.group > kKv8DecodeRows) return false;
    // Keys and units in 32 bits; so are the offsets of a lane inside 16 slots.
    const int64_t cap = p.table_width * p.block_size;
    if (cap > (1 << 30) || (cap / 32 + 1) * p.num_seqs > (1 << 30)) return false;
    if (!kv8_offsets_fit(p)) return false;
    // 4 scale bytes are one load.
    const uint64_t scales = (uint64_t)(uintptr_t)p.ks | (uint64_t)(uintptr_t)p.vs | (uint64_t)p.ssb | (uint64_t)p.ssh;
    if (p.sss != 1 || scales % 4) return false;
    const int64_t isz = dtype == PKV_FLOAT32 ? 4 : 2;
    const uint64_t rows = (uint64_t)(uintptr_t)p.q | (uint64_t)(uintptr_t)p.out | (uint64_t)(p.q_st * isz) |
                          (uint64_t)(p.q_sh * isz) | (uint64_t)(p.out_st * isz) | (uint64_t)(p.out_sh * isz);
    const uint64_t codes = (uint64_t)(uintptr_t)p.k | (uint64_t)(uintptr_t)p.v | (uint64_t)p.sb | (uint64_t)p.ss |
                           (uint64_t)p.sh;
    return rows % 8 == 0 && codes % 4 == 0;
}

// How a decode batch is cut; the bytes of partials that it takes (0: none are wanted, or there are
// more (sequence, KV head) pairs than merge counters).
int64_t kv8_decode_plan(Kv8Params& p, const int64_t* host_ctx, const int64_t* host_qlen) {
    // Workgroups that the GPU holds, three of four waves a CU. (Of 8 waves, as 16-bit heads up to
    // 64 have in runs of a workgroup, it holds 512, and what a plan has more starts late.)
    constexpr int64_t kWorkgroups = 256 * 3;
    const int64_t keys = p.head_dim <= 64 ? 64 : 32;    // of a unit
    // Even runs from this many keys a workgroup on: below, runs inside sequences are as good (us a
    // call, 32/8 heads of 128: 16 sequences of 1-8k 34.1 even, 34.4 not; 64 of 1-16k 191 and 204;
    // 128 of 0.5-8k 198 and 232). Not up to head_dim 64, where two heads share a line and the runs'
    // heads, a workgroup each at the same place, find it in L2 (12 heads of 64: 64 sequences up to
    // 8k 128 even, 106 not; 256 up to 1k 88 and 64).
    constexpr int64_t kEvenKeys = 768;
    // Two workgroups a CU read as fast as three, and leave fewer parts to merge (a lone sequence of
    // 100k tokens 48.7 us with 768, 47.2 with 512).
    constexpr int64_t kEvenWorkgroups = 256 * 2;
    const int64_t heads = p.num_kv_heads, seqs = p.num_seqs, pairs = seqs * heads;
    int64_t units = 0, runs = 0;
    auto each = [&](auto f) {
        for (int64_t i = 0; i < seqs; ++i) {
            if (host_qlen && host_qlen[i] <= 0) continue;
            const int64_t c = host_ctx ? host_ctx[i] : p.max_context_len;
            f(c > keys ? ceil_div(c, keys) : 1);
        }
    };
    each([&](int64_t u) { units += u; });
    p.decode_rows = (int)((int64_t)p.max_query_len * p.group);
    const bool cuts = pairs * 4 <= kMergeCounterBytes;
    auto bytes = [&](int64_t numbers) { return numbers * heads * p.decode_rows * (p.head_dim + 2) * 4; };
    if (cuts && p.head_dim > 64 && units * keys * heads >= kWorkgroups * kEvenKeys) {
        p.decode_mode = kKv8Even;
        p.decode_min_units = 8;
        const int64_t most = kEvenWorkgroups / heads;
        p.decode_slots = p.decode_grid = (int)(most < 1 ? 1 : most);
        return bytes(2 * p.decode_slots);
    }
    p.decode_mode = pairs >= kWorkgroups ? kKv8WaveRuns : kKv8Runs;
    p.decode_min_units = p.decode_mode == kKv8Runs ? 8 : 4;
    const int64_t most = kWorkgroups * (p.decode_mode == kKv8Runs ? 1 : 4) / heads;
    p.decode_slots = (int)(most < 1 ? 1 : most);
    each([&](int64_t u) { runs += ceil_div(u, p.decode_min_units); });
    const int64_t room = p.decode_slots > 2 * seqs ? p.decode_slots : 2 * seqs;
    p.decode_whole = !cuts || runs <= seqs;
    p.decode_grid = (int)(p.decode_whole ? seqs : runs < room ? runs : room);
    return p.decode_whole ? 0 : bytes(p.decode_grid);
}

// ------------------------------------------------------------------ chunks
bool kv8_chunk_applies(const Kv8Params& p, int dtype) {
    if (p.head_dim % 16 || p.head_dim < 32 || p.head_dim > 128 || p.block_shift < 0 || p.num_blocks < 1) return false;
    if (!(p.scale > 0.f) || p.table_width * p.block_size > (1 << 30) || p.num_blocks > 0x7fffffff) return false;
    const int64_t isz = dtype == PKV_FLOAT32 ? 4 : 2;
    const uint64_t probe = (uint64_t)(uintptr_t)p.q | (uint64_t)(uintptr_t)p.out | (uint64_t)(p.q_st * isz) |
                           (uint64_t)(p.q_sh * isz) | (uint64_t)(p.out_st * isz) | (uint64_t)(p.out_sh * isz) |
                           (uint64_t)(uintptr_t)p.k | (uint64_t)(uintptr_t)p.v | (uint64_t)p.sb | (uint64_t)p.ss |
                           (uint64_t)p.sh;
    return probe % 16 == 0;
}

namespace {

// Whether the decode kernel takes a batch of these sizes, strides and addresses aside.
Kv8Params sizes_of(int64_t num_seqs, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t num_tokens,
                   int64_t max_query_len, int64_t max_context_len) {
    Kv8Params p = {};
    p.num_seqs = (int)num_seqs;
    p.num_heads = (int)num_heads;
    p.num_kv_heads = (int)num_kv_heads;
    p.group = (int)(num_heads / num_kv_heads);
    p.head_dim = (int)head_dim;
    p.num_tokens = num_tokens;
    p.max_query_len = (int)(max_query_len && max_query_len < num_tokens ? max_query_len : num_tokens);
    p.max_context_len = max_context_len;
    p.splits = 1;
    p.split_tiles = 0x7fffffff;
    return p;
}

// One token per sequence: the merge then finds its splits from the contexts, so the grid has to
// hold them for any contexts up to the bound.
SplitPlan chunk_plan(const Kv8Params& p, const int64_t* host_ctx, const int64_t* host_qlen) {
    const bool single = p.max_query_len == 1 && p.num_tokens == p.num_seqs;
    return prefill_split_plan(p.num_seqs, p.num_heads, p.num_kv_heads, p.head_dim, p.num_tokens,
                              single ? nullptr : host_ctx, single ? nullptr : host_qlen, p.max_context_len);
}

bool few_rows(const Kv8Params& p) {
    return p.num_seqs <= kKv8DecodeMaxSeqs && (int64_t)p.max_query_len * p.group <= kKv8DecodeRows;
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int64_t pkv_kv8_attention_workspace_bytes(int64_t num_seqs, int64_t num_heads, int64_t num_kv_heads,
                                                     int64_t head_dim, int64_t num_tokens, int64_t max_query_len,
                                                     int64_t max_context_len, const int64_t* host_context_lens,
                                                     const int64_t* host_query_lens) {
    if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || num_tokens <= 0 ||
        num_seqs > 0x7fffffff || num_tokens > 0x7fffffff || num_heads % num_kv_heads)
        return 0;
    Kv8Params p = sizes_of(num_seqs, num_heads, num_kv_heads, head_dim, num_tokens, max_query_len, max_context_len);
    // Few rows: strides and addresses decide between the kernels.
    const int64_t parts = few_rows(p) ? kv8_decode_plan(p, host_context_lens, host_query_lens) : 0;
    const SplitPlan plan = chunk_plan(p, host_context_lens, host_query_lens);
    const int64_t chunks = plan.splits > 1 ? plan.total() : 0, most = parts > chunks ? parts : chunks;
    return most ? kMergeCounterBytes + most : 0;
}

extern "C" int pkv_kv8_attention(
    void* out, int64_t out_stride_t, int64_t out_stride_h, const void* query, int64_t q_stride_t, int64_t q_stride_h,
    const void* k_codes, const void* v_codes, int64_t code_stride_block, int64_t code_stride_slot,
    int64_t code_stride_head, const void* k_scales, const void* v_scales, int64_t scale_stride_block,
    int64_t scale_stride_slot, int64_t scale_stride_head, int64_t num_blocks, int64_t block_size,
    int64_t num_kv_heads, int64_t head_dim, const int64_t* block_tables, int64_t table_stride, int64_t table_width,
    const int64_t* context_lens, const int64_t* query_start_loc, int64_t num_seqs, int64_t num_heads,
    int64_t num_tokens, int64_t max_query_len, int64_t max_context_len, const int64_t* host_context_lens,
    const int64_t* host_query_lens, float scale, int dtype, void* workspace, int64_t workspace_bytes,
    hipStream_t stream) {
    clear_error();
    if (dtype != PKV_FLOAT32 && dtype != PKV_FLOAT16 && dtype != PKV_BFLOAT16)
        return fail(PKV_EINVAL, "kv8_attention: unknown dtype %d", dtype);
    if (num_seqs < 0 || num_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 ||
        num_blocks < 0 || table_width < 0 || max_query_len < 0 || max_context_len < 0)
        return fail(PKV_EINVAL, "kv8_attention: bad sizes");
    if (num_heads % num_kv_heads)
        return fail(PKV_EINVAL, "kv8_attention: %lld query heads not divisible by %lld kv heads", (long long)num_heads,
                    (long long)num_kv_heads);
    if (num_seqs > 0x7fffffff || num_tokens > 0x7fffffff || num_heads > 65535 || head_dim > 512 ||
        block_size > 0x7fffffff || table_width > 0x7fffffff / block_size)
        return fail(PKV_EUNSUPPORTED, "kv8_attention: sizes beyond what the kernels index");
    if (!query_start_loc && num_tokens != num_seqs)
        return fail(PKV_EINVAL, "kv8_attention: %lld tokens of %lld sequences need query_start_loc",
                    (long long)num_tokens, (long long)num_seqs);
    if (num_tokens == 0 || num_seqs == 0) return PKV_OK;
    if (!out || !query || !k_codes || !v_codes || !k_scales || !v_scales || !context_lens ||
        (!block_tables && table_width > 0))
        return fail(PKV_EINVAL, "kv8_attention: null pointer");
    Kv8Params p = sizes_of(num_seqs, num_heads, num_kv_heads, head_dim, num_tokens,
                           query_start_loc ? max_query_len : 1, max_context_len);
    p.out = out;
    p.out_st = out_stride_t;
    p.out_sh = out_stride_h;
    p.q = query;
    p.q_st = q_stride_t;
    p.q_sh = q_stride_h;
    p.k = k_codes;
    p.v = v_codes;
    p.sb = code_stride_block;
    p.ss = code_stride_slot;
    p.sh = code_stride_head;
    p.ks = (const uint8_t*)k_scales;
    p.vs = (const uint8_t*)v_scales;
    p.ssb = scale_stride_block;
    p.sss = scale_stride_slot;
    p.ssh = scale_stride_head;
    p.num_blocks = num_blocks;
    p.block_size = (int)block_size;
    p.block_shift = block_size & (block_size - 1) ? -1 : 63 - __builtin_clzll((unsigned long long)block_size);
    p.tables = block_tables;
    p.table_stride = table_stride;
    p.table_width = table_width;
    p.ctx_lens = context_lens;
    p.qsl = query_start_loc;
    p.scale = scale;
    p.scale_log2 = scale * kLog2e;
    if (kv8_decode_applies(p, dtype)) {
        const int64_t parts = kv8_decode_plan(p, host_context_lens, host_query_lens);
        if (parts && workspace && workspace_bytes >= kMergeCounterBytes + parts) {
            char* ws = reinterpret_cast<char*>(workspace);
            p.ws_cnt = reinterpret_cast<uint32_t*>(ws);
            p.ws_o = reinterpret_cast<float*>(ws + kMergeCounterBytes);
            p.ws_ml = p.ws_o + parts / (4 * (head_dim + 2)) * head_dim;
        } else {
            // No room for partials, or no need: a workgroup or wave a sequence.
            if (p.decode_mode == kKv8Even) p.decode_mode = kKv8Runs;
            p.decode_whole = 1;
            p.decode_grid = p.num_seqs;
        }
        switch (dtype) {
            case PKV_FLOAT32: return launch_kv8_decode<float>(p, stream);
            case PKV_FLOAT16: return launch_kv8_decode<_Float16>(p, stream);
            default: return launch_kv8_decode<bf16_t>(p, stream);
        }
    }
    if (kv8_chunk_applies(p, dtype)) {
        const SplitPlan plan = chunk_plan(p, host_context_lens, host_query_lens);
        if (plan.splits > 1 && workspace && workspace_bytes >= kMergeCounterBytes + plan.total()) {
            // Behind the counters' room, which stays zero.
            char* ws = reinterpret_cast<char*>(workspace) + kMergeCounterBytes;
            p.splits = plan.splits;
            p.split_tiles = plan.split_tiles;
            p.split_items = plan.items;
            p.ws_rows = reinterpret_cast<int*>(ws);
            p.ws_ml = reinterpret_cast<float*>(ws + plan.rows_bytes);
            p.ws_o = reinterpret_cast<float*>(ws + plan.rows_bytes + plan.ml_bytes);
        }
        int rc;
        switch (dtype) {
            case PKV_FLOAT32: rc = launch_kv8_chunk<float>(p, stream); break;
            case PKV_FLOAT16: rc = launch_kv8_chunk<_Float16>(p, stream); break;
            default: rc = launch_kv8_chunk<bf16_t>(p, stream);
        }
        if (rc != PKV_EUNSUPPORTED) return rc;
    }
    return launch_kv8_generic(p, dtype, stream);
}
