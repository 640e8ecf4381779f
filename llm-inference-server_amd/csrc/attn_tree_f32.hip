// Attention of drafted token trees over fp32 pools on v_mfma_f32_16x16x4_f32 (gfx950): head_dim a multiple of
// 16 from 32 to 128, any GQA group, block sizes that are powers of two from 8 up, softmax scale > 0. The
// formulation, masks and what is not finite as in the 16-bit kernel (tree_mfma.h); nothing below fp32.
//
// Rows come 16 a wave, since an fp32 product of 32 rows takes as long as 16 times the 16-bit one and a tree often has
// no more: RW of the four waves have rows of their own, 4 / RW share the keys of a tile (64 keys up to
// head_dim 64, else 32), so that two workgroups fit a CU's LDS and their waves fill one another's waits
// (32 trees of 8-32 nodes behind 16-960 keys, 12 heads of 64: 31.4 us, 3.3 TB/s; 32-row waves of 32x32x2, one
// workgroup a CU, 43.5). RW = 1 up to 32 rows, although two workgroups then read the same keys, the second
// from L2: RW = 2 takes 39.9 there. The next tile's loads start before a tile's products: behind them, 33.1.
//
// S^T = K Q^T: a step contracts four elements of head_dim, one from each quarter (lanes 16 g .. + 15: quarter g), so
// that one 16-byte LDS read of a K row feeds four steps; register r of lane l is the score of key
// 4 (l / 16) + r and row l % 16. O^T += V^T P^T: register r, as it is, is the operand of one step over the
// keys 4 g + r, V[that key][16 t + l % 16] the other.
#include "tree_common.h"

namespace pkv {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma16(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 share_of(f32x4 x, float f) {
    return f32x4{share_of(x[0], f), share_of(x[1], f), share_of(x[2], f), share_of(x[3], f)};
}
__device__ __forceinline__ float max_of_row(float x) {
    const SwapPair a = swap16(x);
    return max_across32(fmaxf(a.a, a.b));
}
__device__ __forceinline__ float sum_of_row(float x) {
    const SwapPair a = swap16(x);
    return sum_across32(a.a + a.b);
}

// Where chunk c (16 bytes) of row r stands in LDS, and back. K: 16 rows' reads of one chunk in different
// banks. V: 4 rows 4 apart, 16 consecutive elements of each, likewise (up to two in one bank where a row is
// no whole sweep of the banks).
template <int D>
__device__ __forceinline__ int k_swap(int r) {
    if constexpr (D % 64 == 0) return r & 15;
    else if constexpr (D % 32 == 0) return (r >> 1) & 7;
    else return (r >> 2) & 3;
}
template <int D>
__device__ __forceinline__ int v_place(int r, int c) {
    constexpr int CPR = D / 4;
    const int by = 4 * ((r >> 2) & 3);
    if constexpr (CPR % 16 == 0) return c ^ by;
    else return (c + by) % CPR;
}
template <int D>
__device__ __forceinline__ int v_chunk_at(int r, int place) {
    constexpr int CPR = D / 4;
    const int by = 4 * ((r >> 2) & 3);
    if constexpr (CPR % 16 == 0) return place ^ by;
    else return (place + 4 * CPR - by) % CPR;
}

template <int D, int RW>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void tree_f32_kernel(const TreeParams p) {
    constexpr int KW = 4 / RW;                // waves that share a tile's keys
    constexpr int KT = kTreeKeysF32<D>;
    constexpr int NK = KT / 16 / KW;          // 16-key groups of a wave and tile
    static_assert(NK >= 1, "a wave has 16 keys at least");
    constexpr int ROWS = 16 * RW;
    constexpr int KREADS = D / 16;            // 16-byte reads of a K row by a lane
    constexpr int DT = D / 16;                // O^T tiles of 16 dims
    constexpr int ROWB = D * 4, CPR = D / 4;
    constexpr int STAGED = KT / 4;            // keys that a wave stages
    constexpr int IPB = (STAGED * CPR + 63) / 64;
    constexpr bool kWholeDma = STAGED * CPR % 64 == 0;
    constexpr bool kHalfDma = 64 % CPR == 0 && 64 / CPR <= 8;   // rows of one instruction all in an 8-row half

    __shared__ __attribute__((aligned(1024))) char s_all[4 * KT * ROWB];      // K, V, K, V
    __shared__ int s_taken;                   // whether V held what is not finite behind the cached keys
    __shared__ int s_walked;                  // whether a wave has put such into its rows
    __shared__ float2 s_ml[4][16];

    PrefillItem it;
    if (!tree_item<ROWS, KT>(p, it)) return;
    const uint32_t G = (uint32_t)p.group;
    const int kvh = it.kvh, split = it.split, seq = it.seq;
    const int64_t q_first = it.q_first;
    const int kmax = it.ctx < 0 || p.num_blocks < 1 ? 0 : it.ctx;             // keys that there are
    const int n_rows = it.q_len * (int)G;
    const int row0 = it.row_tile * ROWS;
    const int pos0 = it.ctx - it.q_len;       // first drafted key
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
    const int g = lane >> 4, col = lane & 15;
    const int wrow = rw * 16 + col;
    const bool my_live = wrow < rows;         // rows past the last one repeat it, not stored
    const uint32_t my_row = (uint32_t)(row0 + (my_live ? wrow : rows - 1));
    const int my_q = (int)(my_row / G);
    const int my_head = kvh * (int)G + (int)(my_row - (uint32_t)my_q * G);
    const bool has_rows = rw * 16 < rows;     // else the wave only stages

    f32x4 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = f32x4{};
    float m_run = kNegInf, l_run = 0.f;

    const int64_t* table = p.tables + (int64_t)seq * p.table_stride;
    const char* kbase = reinterpret_cast<const char*>(p.k) + (int64_t)kvh * p.sh * 4;
    const char* vbase = reinterpret_cast<const char*>(p.v) + (int64_t)kvh * p.sh * 4;
    const int64_t block_bytes = p.sb * 4, slot_bytes = p.ss * 4;

    // ---- staging: lane l holds the block id of the tile's 8-key group l % (KT / 8), the index clamped to the
    // last block with a key. Wave w stages keys STAGED w .. of the tile.
    const int nb_last = (kmax - 1) >> p.block_shift;
    auto tile_ids = [&](int kt) -> int64_t {
        const int b = (kt * KT + 8 * (lane & (KT / 8 - 1))) >> p.block_shift;
        return table[b < nb_last ? b : nb_last];
    };
    auto dma_row = [&](int j) { return (64 * j + lane) / CPR; };
    auto k_chunk = [&](int j) { return 16 * ((64 * j + lane) % CPR ^ k_swap<D>((STAGED * wave + dma_row(j)) & 15)); };
    auto v_chunk = [&](int j) { return 16 * v_chunk_at<D>(STAGED * wave + dma_row(j), (64 * j + lane) % CPR); };
    uint32_t k_off[IPB], v_off[IPB];
#pragma unroll
    for (int j = 0; j < IPB; ++j) {
        k_off[j] = (uint32_t)((dma_row(j) & 7) * slot_bytes) + (uint32_t)k_chunk(j);
        v_off[j] = (uint32_t)((dma_row(j) & 7) * slot_bytes) + (uint32_t)v_chunk(j);
    }
    const bool offs_fit = 8 * slot_bytes + ROWB <= (int64_t)0xffffffff;
    const uint32_t lds = lds_u32(s_all);
    // (Inlined by force: as calls, lambdas get their captures through memory.)
    auto dma_tile = [&](int kt, int64_t ids, uint32_t to) __attribute__((always_inline)) {
        const int first = kt * KT + STAGED * wave;
        const int64_t id0 = readlane64(ids, STAGED / 8 * wave), id1 = readlane64(ids, STAGED / 8 * wave + STAGED / 8 - 1);
        const int64_t half0 = id0 * block_bytes + (first & (p.block_size - 1)) * slot_bytes;
        const int64_t half1 = id1 * block_bytes + ((first + STAGED - 8) & (p.block_size - 1)) * slot_bytes;
        const bool ok = ((uint64_t)id0 < (uint64_t)p.num_blocks) & ((uint64_t)id1 < (uint64_t)p.num_blocks);
        const uint32_t dk = to + (uint32_t)(STAGED * wave * ROWB), dv = dk + KT * ROWB;
        if (ok & offs_fit & (first + STAGED <= kmax)) {
#pragma unroll
            for (int j = 0; j < IPB; ++j) {
                if constexpr (kHalfDma) {
                    const int64_t half = 64 * j / CPR < 8 ? half0 : half1;
                    dma16(kbase + half, k_off[j], dk + j * 1024);
                    dma16(vbase + half, v_off[j], dv + j * 1024);
                } else if (kWholeDma || 64 * j + lane < STAGED * CPR) {
                    const int64_t half = dma_row(j) < 8 ? half0 : half1;
                    dma16(kbase + half + k_off[j], dk + j * 1024);
                    dma16(vbase + half + v_off[j], dv + j * 1024);
                }
            }
            return;
        }
        // Rows past the last key (masked, their V zeroed below) and those of blocks outside the pool are read from
        // the pool's first row.
#pragma unroll
        for (int j = 0; j < IPB; ++j) {
            const int r = dma_row(j);
            int64_t off = 0;
            if ((uint64_t)(r < 8 ? id0 : id1) < (uint64_t)p.num_blocks && first + r < kmax)
                off = (r < 8 ? half0 : half1) + (int64_t)(r & 7) * slot_bytes;
            if (kWholeDma || 64 * j + lane < STAGED * CPR) {
                dma16(kbase + off + k_chunk(j), dk + j * 1024);
                dma16(vbase + off + v_chunk(j), dv + j * 1024);
            }
        }
    };

    // ---- LDS operands of this lane: its K row's chunks, and V[4 g][16 t + col] (rows r on, and 16 rows on, at
    // the same places: neither moves the swizzle).
    const uint32_t wave_off = (uint32_t)(kw * NK * 16 * ROWB);   // of the wave's keys
    uint32_t koff[KREADS], voff[DT];
#pragma unroll
    for (int c = 0; c < KREADS; ++c) {
        koff[c] = wave_off + (uint32_t)(col * ROWB + (((g * KREADS + c) ^ k_swap<D>(col)) << 4));
        asm volatile("" : "+v"(koff[c]));
    }
#pragma unroll
    for (int t = 0; t < DT; ++t) {
        const int d = 16 * t + col;
        voff[t] = wave_off + (uint32_t)(4 * g * ROWB + (v_place<D>(4 * g, d >> 2) << 4) + 4 * (d & 3));
        asm volatile("" : "+v"(voff[t]));
    }

    int64_t ids = 0;
    if (t_begin < t_end) ids = tile_ids(t_begin);
    // Q^T: lane supplies Q[its row][(D / 4) g ..], element by element.
    float qf[4 * KREADS];
    {
        const float* qrow = reinterpret_cast<const float*>(p.q) + (q_first + my_q) * p.q_st + (int64_t)my_head * p.q_sh;
#pragma unroll
        for (int c = 0; c < KREADS; ++c) {
            const float4 v = *reinterpret_cast<const float4*>(qrow + g * (D / 4) + 4 * c);
            qf[4 * c] = v.x;
            qf[4 * c + 1] = v.y;
            qf[4 * c + 2] = v.z;
            qf[4 * c + 3] = v.w;
        }
    }
    if (threadIdx.x == 0) s_taken = s_walked = 0;

    const TreeRow seen(p.masks + (q_first + my_q) * p.mask_stride, t_end * KT > pos0 ? p.mask_words : 0);
    auto window = [&](int key0) __attribute__((always_inline)) { return seen.window(p.mask_words, key0, pos0, kmax); };

    auto tile = [&](auto tail, int kt, const char* tile_k, char* tile_v, uint32_t next) __attribute__((always_inline)) {
        constexpr bool drafted = decltype(tail)::value;          // keys past the cached ones among the tile's
        __builtin_amdgcn_s_waitcnt(0);
        lds_barrier();                        // tile kt is staged, tile kt - 1 is done with
        if (kt + 1 < t_end) {
            dma_tile(kt + 1, ids, next);
            ids = tile_ids(kt + 2);
        }
        f32x4 st[NK];
        if (has_rows) {
#pragma unroll
            for (int i = 0; i < NK; ++i) st[i] = f32x4{};
#pragma unroll
            for (int c = 0; c < KREADS; ++c)
#pragma unroll
                for (int i = 0; i < NK; ++i) {
                    const float4 a = *reinterpret_cast<const float4*>(tile_k + i * 16 * ROWB + koff[c]);
                    st[i] = mfma16(a.x, qf[4 * c], st[i]);
                    st[i] = mfma16(a.y, qf[4 * c + 1], st[i]);
                    st[i] = mfma16(a.z, qf[4 * c + 2], st[i]);
                    st[i] = mfma16(a.w, qf[4 * c + 3], st[i]);
                }
        }
        if constexpr (drafted) {
            tree_take_out<float, KT, CPR>(tile_v, kt * KT, pos0, kmax, s_taken);
            lds_barrier();
        }
        if (!has_rows) return;
        if constexpr (drafted) {
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                const uint32_t mine = window(kt * KT + (kw * NK + i) * 16) >> (4 * g);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!(mine >> r & 1)) st[i][r] = kNegInf;
            }
        }
        float mt = kNegInf;
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) mt = fmaxf(mt, st[i][r]);
        mt = max_of_row(mt) * p.scale_log2;   // scale > 0: max commutes with it
        asm("" : "+v"(mt));                   // stays rounded: m_run - mt below is not contracted into an fma
        const bool raise = mt > m_run + kRescaleThreshold;
        const float m_new = raise ? mt : m_run;
        const float alpha = raise ? fast_exp2(m_run - mt) : 1.f;
        if (__builtin_amdgcn_ballot_w64(raise)) {
#pragma unroll
            for (int t = 0; t < DT; ++t) o[t] *= alpha;
        }
        m_run = m_new;
        const float m_off = m_new == kNegInf ? 0.f : m_new;
        float psum = 0.f;
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = fast_exp2(fmaf(st[i][r], p.scale_log2, -m_off));
                st[i][r] = e;
                psum += e;
            }
        l_run = l_run * alpha + sum_of_row(psum);
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const char* vrow = tile_v + (i * 16 + r) * ROWB;
                const float w = st[i][r];
#pragma unroll
                for (int t = 0; t < DT; ++t) o[t] = mfma16(*reinterpret_cast<const float*>(vrow + voff[t]), w, o[t]);
            }
    };

    // Tile t is in the buffers of t's parity: K, then V.
    constexpr int BUF = 2 * KT * ROWB;
    if (t_begin < t_end) {
        dma_tile(t_begin, ids, lds + (t_begin & 1) * BUF);
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
    if (has_rows && t_begin < t_end) {
        float any = 0.f;                      // NaN if some output is not finite
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) any += o[t][r] * 0.f;
        if (s_taken || __builtin_amdgcn_ballot_w64(any != any && l_run == l_run)) {
            s_walked = 1;
            float4 extra[DT];
#pragma unroll
            for (int t = 0; t < DT; ++t) extra[t] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int at = t_begin; at < t_end; ++at)
                for (int k = 0; k < 16 * NK; ++k) {
                    const int first = at * KT + kw * NK * 16 + (k & ~15), key = first + (k & 15);
                    if (key >= kmax) break;
                    const int64_t id = table[key >> p.block_shift];
                    const bool sees = key < pos0 || (window(first) >> (k & 15) & 1);
                    if ((uint64_t)id >= (uint64_t)p.num_blocks || !sees) continue;
                    const float* row = reinterpret_cast<const float*>(vbase + id * block_bytes + (key & (p.block_size - 1)) * slot_bytes) + 4 * g;
#pragma unroll
                    for (int t = 0; t < DT; ++t) extra[t] = Four<float>::load(row + 16 * t).add_rest(extra[t]);
                }
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                if (extra[t].x != 0.f) o[t][0] = extra[t].x;
                if (extra[t].y != 0.f) o[t][1] = extra[t].y;
                if (extra[t].z != 0.f) o[t][2] = extra[t].z;
                if (extra[t].w != 0.f) o[t][3] = extra[t].w;
            }
        }
    }

    // ---- the waves of the same rows: tile t of the output is summed by wave t % KW of them.
    float m_all = m_run, l_all = l_run;
    if constexpr (KW > 1) {
        if (g == 0) s_ml[wave][col] = make_float2(m_run, l_run);
        lds_barrier();                        // the tiles are done with
        f32x4* so = reinterpret_cast<f32x4*>(s_all);
#pragma unroll
        for (int t = 0; t < DT; ++t)
            if (t % KW != kw) so[(wave * DT + t) * 64 + lane] = o[t];
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
        const float f_own = fast_exp2(m_run - m_off);
        auto join = [&](auto times) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                if (t % KW != kw) continue;
                f32x4 x = times(o[t], f_own);
#pragma unroll
                for (int w = 0; w < KW; ++w)
                    if (w != kw) x += times(so[((rw * KW + w) * DT + t) * 64 + lane], f[w]);
                o[t] = x;
            }
        };
        if (s_walked) join([](f32x4 x, float y) { return share_of(x, y); });
        else join([](f32x4 x, float y) { return x * y; });
    }
    if (!my_live) return;
    const int64_t tok = q_first + my_q;
    if (run < n_tiles) {
        // One of several splits: this row's partial, unnormalised. (The merge skips a part whose maximum
        // is -inf; one whose scores were all NaN has to count.)
        const int64_t row = tok * p.num_heads + my_head;
        const int64_t slot = row * p.splits + split;
        float* po = p.ws_o + slot * D + 4 * g;
#pragma unroll
        for (int t = 0; t < DT; ++t)
            if (t % KW == kw) *reinterpret_cast<f32x4*>(po + 16 * t) = o[t];
        if (g == 0 && kw == 0) {
            *reinterpret_cast<float2*>(p.ws_ml + slot * 2) =
                make_float2(m_all == kNegInf && l_all != 0.f ? 0.f : m_all, l_all);
            if (split == 0) p.ws_rows[row] = (n_tiles + run - 1) / run;
        }
        return;
    }
    if (p.ws_rows && g == 0 && kw == 0) p.ws_rows[tok * p.num_heads + my_head] = 0;    // finished here
    const float inv = l_all == 0.f ? 1.f : 1.f / l_all;        // no key, or weights of 0 alone: o is 0 where it is finite
    float* orow = reinterpret_cast<float*>(p.out) + tok * p.out_st + (int64_t)my_head * p.out_sh + 4 * g;
#pragma unroll
    for (int t = 0; t < DT; ++t)
        if (t % KW == kw) *reinterpret_cast<f32x4*>(orow + 16 * t) = o[t] * inv;
}

template <int D, int RW>
int launch_rows(const TreeParams& p, hipStream_t stream) {
    tree_f32_kernel<D, RW><<<dim3((unsigned)tree_workgroups(p, 16 * RW)), 256, 0, stream>>>(p);
    const int rc = check_launch("tree attention");
    if (rc || p.splits == 1) return rc;
    const int64_t rows = p.num_tokens * p.num_heads;
    prefill_merge_kernel<float, D, true><<<dim3((unsigned)ceil_div(rows, kMergeRows<D>)), 256, 0, stream>>>(p);
    return check_launch("tree attention, merge");
}

template <int D>
int launch_d(const TreeParams& p, hipStream_t stream) {
    switch (p.row_waves) {
        case 1:
            // (Tiles of 32 keys have no 16 for each of four waves, tree_plan does not ask for it.)
            if constexpr (kTreeKeysF32<D> == 64) return launch_rows<D, 1>(p, stream);
        case 2: return launch_rows<D, 2>(p, stream);
        default: return launch_rows<D, 4>(p, stream);
    }
}

}  // namespace

int launch_tree_f32(const TreeParams& p, hipStream_t stream) {
    switch (p.head_dim) {
        case 32: return launch_d<32>(p, stream);
        case 48: return launch_d<48>(p, stream);
        case 64: return launch_d<64>(p, stream);
        case 80: return launch_d<80>(p, stream);
        case 96: return launch_d<96>(p, stream);
        case 112: return launch_d<112>(p, stream);
        default: return launch_d<128>(p, stream);
    }
}

}  // namespace pkv
