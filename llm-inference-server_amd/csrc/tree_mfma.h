// Attention of drafted token trees on MFMA (gfx950): the kernel, instantiated by type in
// attn_tree_*.hip. fp16 and bf16 pools, head_dim a multiple of 16 from 32 to 128, any GQA group, block sizes that are powers
// of two from 8 up, softmax scale > 0.
//
// The formulation is the prefill kernel's (attn_prefill.hip): rows are (token, query head) pairs of a
// sequence and KV head; S^T = K Q^T and O^T += V^T P^T on 32x32x16, so that a lane owns one row, its
// softmax is lane-local but for one swap, and P^T feeds the second product from the accumulator; K/V
// tiles go HBM -> LDS by DMA, double buffered. What differs:
//
//  * Few rows. A tree has some dozens of rows at most a KV head, where a prompt fills the 128 of a
//    workgroup, and the kernel is bound by the K/V stream. RW of the workgroup's four waves have 32 rows
//    each, and 4 / RW waves share the keys of a tile: with RW = 1 each has 32 keys of 128, with
//    RW = 2 32 of 64, with RW = 4 all 64. Waves of the same rows merge through LDS at the end.
//  * Masks. All rows see all cached keys, so only the tiles that reach past them are masked, by a 32-bit
//    window of the row's mask words.
//  * What is not seen must not reach a row, and 0 * NaN would: in those tiles V's elements that are not finite
//    are taken out of LDS (zeros), as are rows past the last key. A wave that took some out, or whose
//    output turned NaN under finite weights (0 * infinity, or an infinity times two pieces of opposite
//    signs), walks its keys once more at the end and puts into each row's dims what it sees of them; it stays
//    there where waves and runs are joined, however little they weigh (share_of).
//
// Weights enter the second product as two pieces of the type: one alone is off by up to 2^-9 of a weight in
// bf16, as much as the output's rounding. Two bf16 pieces have 16 bits of any weight. fp16 ends at 2^-24, so
// its weights reach up to the type's other end: the reference m that scores are taken from is 13 to 15 bits below
// the largest score so far, where bf16's is at most 8 below it. Two pieces are then off by 2^-22 of a weight, or by 2^-38 of
// the row's largest where that is more. (With bf16's rule a tail of keys at 2^-24.9 of the largest weight came out 24% off,
// and one below 2^-25 not at all.)
//
// Bound: by matrix and vector instructions in turn where rows are many (64 sequences of 16-64 nodes behind
// 1,024-8,192 keys, 32/8 heads of 128, bf16: 412 us; one piece of the weights 321), by start, a round trip
// a tile and the longest context where they are few (32 of 8-32 nodes behind 16-960 keys, 12 heads of 64, fp16:
// 19.0 us; RW = 2 21.8, RW = 4 24.0 where it took 18.7), by HBM and by the partials' way to memory and back in a lone long context
// (32 nodes behind 100,000 keys, 32/8 heads of 128: 121 us, of which the merge is 10). The next
// tile's loads start ahead of a tile's products: behind them, 422 and 122.
#pragma once

#include "tree_common.h"

namespace pkv {
namespace {

// Keys of a tile.
template <int RW>
constexpr int kTreeTile = RW == 1 ? 128 : 64;

// Whether a row's reference for its scores (in base 2) is raised in a tile whose largest is `top`, and to what. Weights are
// 2^(score - reference); fp16 holds less than 2^16. `top` is rounded, the scores are not: those of 2^22 and more
// can be well above it, which the last term makes room for (up to 2^27).
template <typename T>
__device__ __forceinline__ bool tree_raises(float top, float ref) {
    if constexpr (__is_same(T, _Float16)) return fmaf(fabsf(top), 0x1p-23f, top - ref) > 15.f;
    else return top > ref + kRescaleThreshold;
}
template <typename T>
__device__ __forceinline__ float tree_reference(float top) {
    if constexpr (__is_same(T, _Float16)) return fmaf(fabsf(top), 0x1p-23f, top - 13.f);
    else return top;
}

// Waves a SIMD: LDS has room for two workgroups a CU, or for one.
template <int D, int RW>
constexpr int kTreeWaves = 8 * kTreeTile<RW> * D <= 72 * 1024 ? 2 : 1;

template <typename T, int D, int RW>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kTreeWaves<D, RW>))) void tree_mfma_kernel(const TreeParams p) {
    static_assert(D % 16 == 0 && D >= 32 && D <= 128, "head_dim");
    constexpr int KW = 4 / RW;                // waves that share a tile's keys
    constexpr int KT = kTreeTile<RW>;
    constexpr int NH = KT / 32 / KW;          // 32-key halves of a wave and tile
    constexpr int ROWS = 32 * RW;
    constexpr int KREADS = D / 16;            // 16-byte reads of a K row by a lane: S^T contraction steps
    constexpr int DTILES = (D + 31) / 32;     // O^T tiles of 32 dims (the last may be half a tile)
    constexpr int ROWB = D * 2;               // bytes of a K/V row
    constexpr int CPR = ROWB / 16;            // its 16-byte chunks
    constexpr int G16 = KT / 64;              // groups of 16 keys that a wave stages
    constexpr int IPB = (16 * CPR + 63) / 64; // DMA instructions of a group, of K or V
    constexpr bool kWholeDma = 16 * CPR % 64 == 0;
    constexpr bool kHalfDma = 64 % CPR == 0 && 64 / CPR <= 8;   // rows of one all in an 8-row half

    __shared__ __attribute__((aligned(1024))) char s_all[4 * KT * ROWB];      // K, V, K, V
    __shared__ int s_taken;                   // whether V held what is not finite behind the cached keys
    __shared__ int s_walked;                  // whether a wave has put such into its rows
    __shared__ float2 s_ml[4][32];

    PrefillItem it;
    if (!tree_item<ROWS, KT>(p, it)) return;
    const uint32_t G = (uint32_t)p.group;
    const int kvh = it.kvh, split = it.split, seq = it.seq;
    const int64_t q_first = it.q_first;
    const int q_len = it.q_len;
    const int kmax = it.ctx < 0 || p.num_blocks < 1 ? 0 : it.ctx;             // keys that there are
    const int n_rows = q_len * (int)G;
    const int row0 = it.row_tile * ROWS;
    const int pos0 = it.ctx - q_len;          // first drafted key
    const int rows = n_rows - row0 < ROWS ? n_rows - row0 : ROWS;
    const int n_tiles = (kmax + KT - 1) / KT;
    // A sequence without cached keys is not cut: a row of it may see nothing, which the merge cannot tell.
    int t_begin = 0, t_end = n_tiles, run = n_tiles;
    if (it.splits > 1 && n_tiles > 0 && pos0 > 0) {
        run = split_run(n_tiles, it.splits, p.split_tiles);
        t_begin = split * run;
        t_end = n_tiles - t_begin < run ? n_tiles : t_begin + run;
    }
    // A later split of a sequence that ends before it; without keys the first one writes zeros.
    if (split > 0 && (t_begin >= n_tiles || run == n_tiles)) return;

    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int rw = wave / KW, kw = wave % KW;
    const int h = lane >> 5, col = lane & 31;
    const int wrow = rw * 32 + col;
    const bool my_live = wrow < rows;         // rows past the last one repeat it, not stored
    const uint32_t my_row = (uint32_t)(row0 + (my_live ? wrow : rows - 1));
    const int my_q = (int)(my_row / G);
    const int my_head = kvh * (int)G + (int)(my_row - (uint32_t)my_q * G);
    const bool has_rows = rw * 32 < rows;     // else the wave only stages

    f32x16 o[DTILES];
#pragma unroll
    for (int t = 0; t < DTILES; ++t) o[t] = f32x16{};
    float m_run = kNegInf, l_run = 0.f;

    const int64_t* table = p.tables + (int64_t)seq * p.table_stride;
    const char* kbase = reinterpret_cast<const char*>(p.k) + (int64_t)kvh * p.sh * (int64_t)sizeof(T);
    const char* vbase = reinterpret_cast<const char*>(p.v) + (int64_t)kvh * p.sh * (int64_t)sizeof(T);
    const int64_t block_bytes = p.sb * (int64_t)sizeof(T);
    const int64_t slot_bytes = p.ss * (int64_t)sizeof(T);

    // ---- staging, as in the prefill kernel: lane l holds the block id of the tile's 8-key group l %
    // (KT / 8), the index clamped to the last block with a key.
    const int nb_last = (kmax - 1) >> p.block_shift;
    auto tile_ids = [&](int kt) -> int64_t {
        const int b = (kt * KT + 8 * (lane & (KT / 8 - 1))) >> p.block_shift;
        return table[b < nb_last ? b : nb_last];
    };
    auto dma_row = [&](int j) { return (64 * j + lane) / CPR; };
    auto dma_chunk = [&](int j) { return 16 * ((64 * j + lane) % CPR ^ lds_swizzle<D>(dma_row(j))); };
    uint32_t lane_off[IPB];
#pragma unroll
    for (int j = 0; j < IPB; ++j) lane_off[j] = (uint32_t)((dma_row(j) & 7) * slot_bytes) + (uint32_t)dma_chunk(j);
    const bool offs_fit = 8 * slot_bytes + ROWB <= (int64_t)0xffffffff;
    // (Inlined by force: as calls, lambdas get their captures through memory.)
    auto dma_tile = [&](int kt, int64_t ids, uint32_t sk, uint32_t sv) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < G16; ++g) {
            const int at = wave * G16 + g;                       // the group in the tile
            const int first = kt * KT + 16 * at;                 // its first key
            const int64_t id0 = readlane64(ids, 2 * at), id1 = readlane64(ids, 2 * at + 1);
            const int64_t half0 = id0 * block_bytes + (first & (p.block_size - 1)) * slot_bytes;
            const int64_t half1 = id1 * block_bytes + ((first + 8) & (p.block_size - 1)) * slot_bytes;
            const bool ok = ((uint64_t)id0 < (uint64_t)p.num_blocks) & ((uint64_t)id1 < (uint64_t)p.num_blocks);
            const uint32_t dk = sk + (uint32_t)(16 * at * ROWB), dv = sv + (uint32_t)(16 * at * ROWB);
            if (ok & offs_fit & (first + 16 <= kmax)) {
#pragma unroll
                for (int j = 0; j < IPB; ++j) {
                    if constexpr (kHalfDma) {
                        const int64_t half = 64 * j / CPR < 8 ? half0 : half1;
                        dma16(kbase + half, lane_off[j], dk + j * 1024);
                        dma16(vbase + half, lane_off[j], dv + j * 1024);
                    } else if (kWholeDma || 64 * j + lane < 16 * CPR) {
                        const int64_t half = dma_row(j) < 8 ? half0 : half1;
                        dma16(kbase + half + lane_off[j], dk + j * 1024);
                        dma16(vbase + half + lane_off[j], dv + j * 1024);
                    }
                }
                continue;
            }
            // Rows past the last key (masked, their V zeroed below) and those of blocks outside the pool are
            // read from the pool's first row.
#pragma unroll
            for (int j = 0; j < IPB; ++j) {
                const int r = dma_row(j);
                const int64_t id = r < 8 ? id0 : id1;
                int64_t off = 0;
                if ((uint64_t)id < (uint64_t)p.num_blocks && first + r < kmax)
                    off = (r < 8 ? half0 : half1) + (int64_t)(r & 7) * slot_bytes;
                if (kWholeDma || 64 * j + lane < 16 * CPR) {
                    dma16(kbase + off + dma_chunk(j), dk + j * 1024);
                    dma16(vbase + off + dma_chunk(j), dv + j * 1024);
                }
            }
        }
    };

    // ---- LDS operands of this lane (as in the prefill kernel).
    const int grp = lane >> 4;
    const int tr_key = (lane & 15) >> 2;
    const int tr_col = 16 * (grp & 1) + 4 * (lane & 3);
    const int k_swz = lds_swizzle<D>(col);
    const int v_cb = tr_col >> 3;
    const int v_row = 4 * (grp >> 1) + tr_key, v_byte = 8 * (lane & 1);
    const uint32_t wave_off = (uint32_t)(kw * NH * 32 * ROWB);   // of the wave's keys
    uint32_t koff[KREADS], voff_lo[DTILES], voff_hi[DTILES];
#pragma unroll
    for (int s = 0; s < KREADS; ++s) {
        koff[s] = wave_off + (uint32_t)(col * ROWB + (((2 * s + h) ^ k_swz) << 4));
        asm volatile("" : "+v"(koff[s]));
    }
#pragma unroll
    for (int t = 0; t < DTILES; ++t) {
        // Columns past head_dim re-read the tile's first chunks: output rows never stored.
        const int c = 4 * t + v_cb < CPR ? 4 * t + v_cb : 4 * t + (v_cb & 1);
        voff_lo[t] = wave_off + (uint32_t)(v_row * ROWB + v_byte + ((c ^ lds_swizzle<D>(v_row)) << 4));
        voff_hi[t] = wave_off + (uint32_t)((v_row + 8) * ROWB + v_byte + ((c ^ lds_swizzle<D>(v_row + 8)) << 4));
        asm volatile("" : "+v"(voff_lo[t]), "+v"(voff_hi[t]));
    }

    int64_t ids = 0;
    if (t_begin < t_end) ids = tile_ids(t_begin);
    // Q^T: lane supplies Q[its row][16 s + 8 h .. + 7].
    u32x4 qfrag[KREADS];
    {
        const T* qrow = reinterpret_cast<const T*>(p.q) + (q_first + my_q) * p.q_st + (int64_t)my_head * p.q_sh;
#pragma unroll
        for (int s = 0; s < KREADS; ++s) {
            const Vec16 v = load16(qrow + 16 * s + 8 * h);
            qfrag[s] = u32x4{v.w[0], v.w[1], v.w[2], v.w[3]};
        }
    }
    if (threadIdx.x == 0) s_taken = s_walked = 0;

    const TreeRow seen(p.masks + (q_first + my_q) * p.mask_stride, t_end * KT > pos0 ? p.mask_words : 0);
    auto window = [&](int key0) __attribute__((always_inline)) { return seen.window(p.mask_words, key0, pos0, kmax); };

    auto tile = [&](auto tail, int kt, const char* tile_k, char* tile_v, uint32_t nk) __attribute__((always_inline)) {
        constexpr bool drafted = decltype(tail)::value;          // keys past the cached ones among the tile's
        __builtin_amdgcn_s_waitcnt(0);
        lds_barrier();                        // tile kt is staged, tile kt - 1 is done with
        if (kt + 1 < t_end) {
            dma_tile(kt + 1, ids, nk, nk + KT * ROWB);
            ids = tile_ids(kt + 2);
        }
        f32x16 st[NH];
        __builtin_amdgcn_s_setprio(1);
        if (has_rows) {
#pragma unroll
            for (int i = 0; i < NH; ++i) st[i] = f32x16{};
            u32x4 kf[NH][KREADS];
#pragma unroll
            for (int i = 0; i < NH; ++i)
#pragma unroll
                for (int s = 0; s < KREADS; ++s) {
                    const uint4 a = *reinterpret_cast<const uint4*>(tile_k + i * 32 * ROWB + koff[s]);
                    kf[i][s] = u32x4{a.x, a.y, a.z, a.w};
                }
#pragma unroll
            for (int s = 0; s < KREADS; ++s)
#pragma unroll
                for (int i = 0; i < NH; ++i) st[i] = Mfma<T>::run(kf[i][s], qfrag[s], st[i]);
        }
        __builtin_amdgcn_s_setprio(0);
        if constexpr (drafted) {
            tree_take_out<T, KT, CPR>(tile_v, kt * KT, pos0, kmax, s_taken);
            lds_barrier();
        }
        if (!has_rows) return;
        if constexpr (drafted) {
#pragma unroll
            for (int i = 0; i < NH; ++i) {
                const uint32_t mine = window(kt * KT + (kw * NH + i) * 32) >> (4 * h);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!(mine >> (8 * (r >> 2) + (r & 3)) & 1)) st[i][r] = kNegInf;
            }
        }
        float mt = kNegInf;
#pragma unroll
        for (int i = 0; i < NH; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) mt = fmaxf(mt, st[i][r]);
        mt = max_across32(mt) * p.scale_log2;   // scale > 0: max commutes with it
        asm("" : "+v"(mt));                     // stays rounded: m_run - mt below is not contracted into an fma
        const bool raise = tree_raises<T>(mt, m_run);
        const float m_new = raise ? tree_reference<T>(mt) : m_run;
        const float alpha = raise ? fast_exp2(m_run - m_new) : 1.f;
        if (__builtin_amdgcn_ballot_w64(raise)) {
#pragma unroll
            for (int t = 0; t < DTILES; ++t) o[t] *= alpha;
        }
        m_run = m_new;
        const float m_off = m_new == kNegInf ? 0.f : m_new;
        float psum = 0.f;
#pragma unroll
        for (int i = 0; i < NH; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float e = fast_exp2(fmaf(st[i][r], p.scale_log2, -m_off));
                st[i][r] = e;
                psum += e;
            }
        psum = sum_across32(psum);
        l_run = l_run * alpha + psum;
#pragma unroll
        for (int s = 0; s < 2 * NH; ++s) {
            f32x16& sv = st[s >> 1];
            const int r0 = 8 * (s & 1);
            u32x4 pb[2];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = sv[r0 + 2 * e], y = sv[r0 + 2 * e + 1];
                const uint32_t w = Mfma<T>::pack(x, y);
                pb[0][e] = w;
                pb[1][e] = Mfma<T>::pack(x - Pair<T>::lo(w), y - Pair<T>::hi(w));
            }
            const char* vgrp = tile_v + ((s >> 1) * 32 + 16 * (s & 1)) * ROWB;
#pragma unroll
            for (int t = 0; t < DTILES; ++t) {
                const uint2 lo = lds_read_tr16(reinterpret_cast<const uint16_t*>(vgrp + voff_lo[t]));
                const uint2 hi = lds_read_tr16(reinterpret_cast<const uint16_t*>(vgrp + voff_hi[t]));
#pragma unroll
                for (int i = 0; i < 2; ++i) o[t] = Mfma<T>::run(u32x4{lo.x, lo.y, hi.x, hi.y}, pb[i], o[t]);
            }
        }
    };

    // Tile t is in the buffers of t's parity: K, then V.
    constexpr int BUF = 2 * KT * ROWB;
    const uint32_t lds = lds_u32(s_all);
    if (t_begin < t_end) {
        dma_tile(t_begin, ids, lds + (t_begin & 1) * BUF, lds + (t_begin & 1) * BUF + KT * ROWB);
        ids = tile_ids(t_begin + 1);
    }
    const int t_cached = pos0 / KT < t_end ? pos0 / KT : t_end;  // tiles of cached keys alone (pos0 >= 0 if it is cut)
    int kt = t_begin;
    if (kt < t_cached && (kt & 1)) {
        tile(std::false_type{}, kt, s_all + BUF, s_all + BUF + KT * ROWB, lds);
        ++kt;
    }
    for (; kt + 1 < t_cached; kt += 2) {
        tile(std::false_type{}, kt, s_all, s_all + KT * ROWB, lds + BUF);
        tile(std::false_type{}, kt + 1, s_all + BUF, s_all + BUF + KT * ROWB, lds);
    }
    for (; kt < t_end; ++kt) {
        char* const k = s_all + (kt & 1) * BUF;
        tile(std::true_type{}, kt, k, k + KT * ROWB, lds + (~kt & 1) * BUF);
    }

    // ---- what is not finite in V, for the rows that see it.
    constexpr int UNITS = D / 8;              // of the output: dims 8 u .. + 7, four of each half
    if (has_rows && t_begin < t_end) {
        float any = 0.f;                      // NaN if some output is
#pragma unroll
        for (int t = 0; t < DTILES; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (32 * t + 8 * (r >> 2) < D) any += o[t][r] * 0.f;
        if (s_taken || __builtin_amdgcn_ballot_w64(any != any && l_run == l_run)) {
            s_walked = 1;
            float4 extra[UNITS];
#pragma unroll
            for (int u = 0; u < UNITS; ++u) extra[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int at = t_begin; at < t_end; ++at)
                for (int k = 0; k < 32 * NH; ++k) {
                    const int first = at * KT + kw * NH * 32 + (k & ~31), key = first + (k & 31);
                    if (key >= kmax) break;
                    const int64_t id = table[key >> p.block_shift];
                    const bool sees = key < pos0 || (window(first) >> (k & 31) & 1);
                    if ((uint64_t)id >= (uint64_t)p.num_blocks || !sees) continue;
                    const T* row = reinterpret_cast<const T*>(vbase + id * block_bytes + (key & (p.block_size - 1)) * slot_bytes) + 4 * h;
#pragma unroll
                    for (int u = 0; u < UNITS; ++u) extra[u] = Four<T>::load(row + 8 * u).add_rest(extra[u]);
                }
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                auto put = [&](int r, float x) {
                    if (x != 0.f) o[u / 4][4 * (u % 4) + r] = x;
                };
                put(0, extra[u].x);
                put(1, extra[u].y);
                put(2, extra[u].z);
                put(3, extra[u].w);
            }
        }
    }

    // ---- the waves of the same rows: unit u of the output is summed by wave u % KW of them.
    float inv, m_all = m_run, l_all = l_run, f_own = 1.f;
    if constexpr (KW > 1) {
        if (h == 0) s_ml[wave][col] = make_float2(m_run, l_run);
        lds_barrier();                        // the tiles are done with
        float* so = reinterpret_cast<float*>(s_all);
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
            if (u % KW != kw)
                *reinterpret_cast<float4*>(so + ((wave * UNITS + u) * 64 + lane) * 4) =
                    make_float4(o[u / 4][4 * (u % 4)], o[u / 4][4 * (u % 4) + 1], o[u / 4][4 * (u % 4) + 2], o[u / 4][4 * (u % 4) + 3]);
        lds_barrier();
        float2 ml[KW];
        m_all = kNegInf;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
            ml[w] = s_ml[rw * KW + w][col];
            m_all = fmaxf(m_all, ml[w].x);
        }
        const float m_off = m_all == kNegInf ? 0.f : m_all;
        float f[KW];
        l_all = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
            f[w] = fast_exp2(ml[w].x - m_off);
            l_all += f[w] * ml[w].y;
        }
        f_own = fast_exp2(m_run - m_off);
        auto join = [&](auto times) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                if (u % KW != kw) continue;
                float4 x = make_float4(times(o[u / 4][4 * (u % 4)], f_own), times(o[u / 4][4 * (u % 4) + 1], f_own),
                                       times(o[u / 4][4 * (u % 4) + 2], f_own), times(o[u / 4][4 * (u % 4) + 3], f_own));
#pragma unroll
                for (int w = 0; w < KW; ++w) {
                    if (w == kw) continue;
                    const float4 y = *reinterpret_cast<const float4*>(so + (((rw * KW + w) * UNITS + u) * 64 + lane) * 4);
                    x.x += times(y.x, f[w]);
                    x.y += times(y.y, f[w]);
                    x.z += times(y.z, f[w]);
                    x.w += times(y.w, f[w]);
                }
                o[u / 4][4 * (u % 4)] = x.x;
                o[u / 4][4 * (u % 4) + 1] = x.y;
                o[u / 4][4 * (u % 4) + 2] = x.z;
                o[u / 4][4 * (u % 4) + 3] = x.w;
            }
        };
        if (s_walked) join(share_of);
        else join([](float x, float y) { return x * y; });
    }
    if (!my_live) return;
    const int64_t tok = q_first + my_q;
    if (run < n_tiles) {
        // One of several splits: this row's partial, unnormalised. (The merge skips a part whose maximum
        // is -inf; one whose scores were all NaN has to count.)
        const int64_t row = tok * p.num_heads + my_head;
        const int64_t slot = row * p.splits + split;
        float* po = p.ws_o + slot * D + 4 * h;
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
            if (u % KW == kw)
                *reinterpret_cast<float4*>(po + 8 * u) =
                    make_float4(o[u / 4][4 * (u % 4)], o[u / 4][4 * (u % 4) + 1], o[u / 4][4 * (u % 4) + 2], o[u / 4][4 * (u % 4) + 3]);
        if (h == 0 && kw == 0) {
            *reinterpret_cast<float2*>(p.ws_ml + slot * 2) =
                make_float2(m_all == kNegInf && l_all != 0.f ? 0.f : m_all, l_all);
            if (split == 0) p.ws_rows[row] = (n_tiles + run - 1) / run;
        }
        return;
    }
    if (p.ws_rows && h == 0 && kw == 0) p.ws_rows[tok * p.num_heads + my_head] = 0;    // finished here
    inv = l_all == 0.f ? 1.f : 1.f / l_all;                    // no key, or weights of 0 alone: o is 0 where it is finite
    T* orow = reinterpret_cast<T*>(p.out) + tok * p.out_st + (int64_t)my_head * p.out_sh + 4 * h;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        if (u % KW != kw) continue;
        const float4 x = make_float4(o[u / 4][4 * (u % 4)] * inv, o[u / 4][4 * (u % 4) + 1] * inv,
                                     o[u / 4][4 * (u % 4) + 2] * inv, o[u / 4][4 * (u % 4) + 3] * inv);
        *reinterpret_cast<uint2*>(orow + 8 * u) = make_uint2(Mfma<T>::pack(x.x, x.y), Mfma<T>::pack(x.z, x.w));
    }
}

template <typename T, int D, int RW>
int launch_tree_rows(const TreeParams& p, hipStream_t stream) {
    tree_mfma_kernel<T, D, RW><<<dim3((unsigned)tree_workgroups(p, 32 * RW)), 256, 0, stream>>>(p);
    const int rc = check_launch("tree attention");
    if (rc || p.splits == 1) return rc;
    const int64_t rows = p.num_tokens * p.num_heads;
    prefill_merge_kernel<T, D, true><<<dim3((unsigned)ceil_div(rows, kMergeRows<D>)), 256, 0, stream>>>(p);
    return check_launch("tree attention, merge");
}

template <typename T, int D>
int launch_tree_d(const TreeParams& p, hipStream_t stream) {
    switch (p.row_waves) {
        case 1: return launch_tree_rows<T, D, 1>(p, stream);
        case 2: return launch_tree_rows<T, D, 2>(p, stream);
        default: return launch_tree_rows<T, D, 4>(p, stream);
    }
}

}  // namespace

template <typename T>
int launch_tree_mfma(const TreeParams& p, hipStream_t stream) {
    switch (p.head_dim) {
        case 32: return launch_tree_d<T, 32>(p, stream);
        case 48: return launch_tree_d<T, 48>(p, stream);
        case 64: return launch_tree_d<T, 64>(p, stream);
        case 80: return launch_tree_d<T, 80>(p, stream);
        case 96: return launch_tree_d<T, 96>(p, stream);
        case 112: return launch_tree_d<T, 112>(p, stream);
        default: return launch_tree_d<T, 128>(p, stream);
    }
}

}  // namespace pkv
