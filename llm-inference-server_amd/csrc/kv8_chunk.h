// Attention of chunks of new tokens over the 8-bit paged cache on MFMA (gfx950): the kernel,
// instantiated by type in attn_kv8_chunk_*.hip. Head_dim a multiple of 16 from 32 to 128, any
// GQA group, block sizes that are powers of two, codes in 16-byte steps, softmax scale > 0.
//
// Bound: MFMA and VALU for long chunks. The formulation is the 16-bit prefill kernel's
// (attn_prefill.hip): 128 (token, query head) rows a workgroup, 32 a wave; S^T = K Q^T and
// O^T += V^T P^T on 32x32x16, so that a lane owns one query row, its softmax is lane-local but
// for one swap, and P^T feeds the second product from the accumulator; contexts of few rows cut
// into runs (prefill_split_plan) and merged. What differs is the staging:
//
//  * 64 keys of K and V a tile are loaded as codes (16 bytes, 16 dims, a piece; a thread has one or
//    two pieces of each), converted to the cached values - code * 2^(b - 127) in one
//    v_cvt_scalef32_pk a pair - and written to LDS as 16-bit rows. Converting once for the
//    workgroup instead of in each of its four waves costs a quarter of the VALU time, of which
//    the softmax leaves little; a tile's LDS traffic is the 16-bit kernel's.
//  * A tile is loaded during the one before the one before it, and converted while the matrix unit
//    is at the first product of the one before it; its block ids come a tile further ahead.
//  * NaN: a row whose scale is NaN (its codes are 0) makes its key's scores NaN, also if it is
//    V's, whose row is staged as zeros: the causal mask then hides it from rows that do not see
//    it, which a weight of 0 times NaN would not.
//
// Values are bf16; for fp16 queries K is its codes as fp16, its scales multiply the scores. Weights
// enter the second product as bf16 pieces, two for 16-bit types (16 bits of them: one of the type's
// own width left up to 2^-9 of a weight in the output), three for fp32 (24 bits), fp32 queries the
// first one as three. The second piece costs a third of the time of long chunks (16 chunks of
// 512 behind 0-4,096, 32/8 heads of 128, bf16: 342 -> 442-460 us): half as many MFMAs again.
#pragma once

#include "kv8.h"
#include "prefill_common.h"

namespace pkv {
namespace {

// Two codes (the lower or upper half of w) times a power of two, as bf16.
template <bool HI>
__device__ __forceinline__ uint32_t scaled_bf16(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}

// What keys are in LDS: their values as bf16, or for fp16 queries their codes as fp16, which has not
// the range of the values; their scales are then multiplied to the scores (kAfter).
template <typename T>
struct Keys {
    typedef bf16_t E;
    static constexpr bool kAfter = false;
    static constexpr uint32_t kNan2 = 0x7fc07fc0u;
    template <bool HI>
    __device__ __forceinline__ static uint32_t cvt(uint32_t w, float scale) {
        return scaled_bf16<HI>(w, scale);
    }
};
template <>
struct Keys<_Float16> {
    typedef _Float16 E;
    static constexpr bool kAfter = true;
    static constexpr uint32_t kNan2 = 0x7e007e00u;
    template <bool HI>
    __device__ __forceinline__ static uint32_t cvt(uint32_t w, float) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HI));
    }
};

// Waves a SIMD that registers are held to. Three for 16-bit types gain nothing at head_dim 64 (92.5 us
// and 92.3) and keep registers in scratch from 80 on (32 fp16 heads of 80: 12 sequences of 1-200 new
// tokens behind 0-1,500 52.2 us, two 49.6; 4 of 256-512 behind 0-3,000 124.8 and 120.4, heads of 96
// 165.5 and 131.2).
template <typename T>
constexpr int kChunkWaves = sizeof(T) == 4 ? 1 : 2;

// UNI: block sizes from 16 up: a wave's pieces of one load are 8 or 16 neighbouring rows of one
// block, so that addresses are uniform and loads cost no vector arithmetic.
template <typename T, int D, bool UNI>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kChunkWaves<T>))) void kv8_chunk_kernel(
    const Kv8Params p) {
    typedef typename Keys<T>::E E;
    constexpr bool kAfter = Keys<T>::kAfter;
    constexpr int DSTEPS = D / 16;            // S^T contraction steps
    constexpr int DTILES = (D + 31) / 32;     // O^T tiles of 32 dims (the last may be half a tile)
    constexpr int ROWB = D * 2;               // bytes of a staged row
    constexpr int CPR = ROWB / 16;            // its 16-byte chunks
    constexpr int PPR = D / 16;               // its pieces of 16 codes
    constexpr int PIECES = (PPR + 3) / 4;     // per thread and tile, of K and of V
    constexpr bool kWhole = PPR % 4 == 0;     // all threads have as many
    constexpr bool LINES = D == 128 && UNI;   // a thread's pieces are of PIECES rows, else of one
    constexpr int NR = LINES ? PIECES : 1;
    constexpr int NQ = sizeof(T) == 4 ? 3 : 1, NP = sizeof(T) == 4 ? 3 : 2;   // pieces of queries and weights

    __shared__ __attribute__((aligned(1024))) uint16_t s_k0[kKT * D];
    __shared__ __attribute__((aligned(1024))) uint16_t s_v0[kKT * D];
    __shared__ __attribute__((aligned(1024))) uint16_t s_k1[kKT * D];
    __shared__ __attribute__((aligned(1024))) uint16_t s_v1[kKT * D];
    __shared__ __attribute__((aligned(16))) float s_ks[2][kAfter ? kKT : 4];    // key scales of either tile

    PrefillItem it;
    if (!prefill_item<kRows, kKT>(p, p.block_size, it)) return;
    const uint32_t G = (uint32_t)p.group;
    const int kvh = it.kvh, split = it.split, seq = it.seq;
    const int64_t q_first = it.q_first;
    const int q_len = it.q_len;
    const int ctx = it.ctx < 0 ? 0 : it.ctx;
    const int n_rows = q_len * (int)G;
    const int row0 = it.row_tile * kRows;
    const int pos0 = ctx - q_len;             // position of the sequence's first query
    const int rows = n_rows - row0 < kRows ? n_rows - row0 : kRows;
    const int q0 = (int)((uint32_t)row0 / G);
    const int q_last = (int)((uint32_t)(row0 + rows - 1) / G);
    const int kmax = pos0 + q_last + 1 < 0 ? 0 : pos0 + q_last + 1;   // keys that the workgroup sees
    const int first_pos = pos0 + q0;
    const int n_tiles = (kmax + kKT - 1) / kKT;
    int t_begin = 0, t_end = n_tiles, run = n_tiles;
    if (it.splits > 1 && n_tiles > 0) {
        run = split_run(n_tiles, it.splits, p.split_tiles);
        t_begin = split * run;
        t_end = n_tiles - t_begin < run ? n_tiles : t_begin + run;
    }
    // A later split of a sequence whose tile ends before it; without keys the first one writes zeros.
    if (t_begin >= n_tiles && split > 0) return;

    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int h = lane >> 5, col = lane & 31;
    const int wrow = wave * kQT + col;
    const bool my_live = wrow < rows;         // rows past the last one repeat it, not stored
    const uint32_t my_row = (uint32_t)(row0 + (my_live ? wrow : rows - 1));
    const int my_q = (int)(my_row / G);
    const int my_head = kvh * (int)G + (int)(my_row - (uint32_t)my_q * G);
    const int my_pos = pos0 + my_q;
    const int wave_rows = rows - wave * kQT < kQT ? rows - wave * kQT : kQT;
    const int wave_kmax = wave_rows > 0 ? pos0 + (int)((uint32_t)(row0 + wave * kQT + wave_rows - 1) / G) + 1 : 0;

    f32x16 o[DTILES];
#pragma unroll
    for (int t = 0; t < DTILES; ++t) o[t] = f32x16{};
    float m_run = kNegInf, l_run = 0.f;
    const float scale_log2 = p.scale_log2;

    // ---- staging: piece j of a thread is codes 16 c .. 16 c + 15 of key row r of the tile.
    const uint8_t* kc = reinterpret_cast<const uint8_t*>(p.k) + kvh * p.sh;
    const uint8_t* vc = reinterpret_cast<const uint8_t*>(p.v) + kvh * p.sh;
    const uint8_t* ksb = p.ks + kvh * p.ssh;
    const uint8_t* vsb = p.vs + kvh * p.ssh;
    const int64_t* table = p.tables + (int64_t)seq * p.table_stride;
    // A wave's load is 16 rows of 64 bytes, or at head_dim 128 (LINES) 8 whole ones. The 8 lanes of
    // one LDS write cycle have 4 pieces of each of two rows whose swizzles differ in parity (4 or 8
    // rows apart, as the width has it), so that they hit all 32 banks; a whole row's pieces, even
    // chunks only, hit half of them twice.
    constexpr bool FOUR = D % 32 == 0 && D != 64;
    const int pair = lane >> 2 & 1;
    const int lane_row = LINES ? (lane >> 4) + 4 * pair
                               : FOUR ? (lane >> 3 & 3) + 4 * pair + 8 * (lane >> 5) : (lane >> 3) + 8 * pair;
    const int lane_c = LINES ? (lane & 3) + 4 * (lane >> 3 & 1) : lane & 3;
    auto wave_row = [&](int j) { return LINES ? 32 * j + 8 * wave : 16 * wave; };   // of the wave's first piece
    auto row_of = [&](int j) { return wave_row(j) + lane_row; };
    auto live = [&](int j) { return kWhole || lane_c + 4 * j < PPR; };
    uint32_t lds0[PIECES], lds1[PIECES], at_row[PIECES];        // at_row: dims, inside the row for all
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
        const int r = row_of(j), c = LINES ? lane_c : live(j) ? lane_c + 4 * j : 0;
        at_row[j] = (uint32_t)(16 * c);
        lds0[j] = (uint32_t)(r * ROWB + (((2 * c) ^ lds_swizzle<D>(r)) << 4));
        lds1[j] = (uint32_t)(r * ROWB + (((2 * c + 1) ^ lds_swizzle<D>(r)) << 4));
    }
    const int in_block = p.block_size - 1, last = kmax - 1;     // last: the workgroup's last key
    // UNI: a lane's offset from the wave's first row.
    const uint32_t lane_off = (uint32_t)(lane_row * (int)p.ss), lane_sc = (uint32_t)(lane_row * (int)p.sss);
    int64_t id;                               // LINES: lane j holds that of load j
    uint32_t ks_raw[NR], vs_raw[NR];
    Vec16 k_raw[PIECES], v_raw[PIECES];
    auto load_ids = [&](int kt) {
        const int key = kt * kKT + (LINES ? wave_row(lane % PIECES) : UNI ? wave_row(0) : row_of(0));
        id = table[(key < last ? key : last) >> p.block_shift];
    };
    auto load_tile = [&](int kt) {
        const uint32_t blk = (uint64_t)id < (uint64_t)p.num_blocks ? (uint32_t)id : 0u;   // none is followed out of the cache
        if constexpr (UNI) {
            auto rsrc = [](const uint8_t* base) {
                return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, -1, 0x00027000);
            };
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                const uint32_t b = (uint32_t)__builtin_amdgcn_readlane((int)blk, LINES ? j : 0);
                const int at = (kt * kKT + wave_row(j)) & in_block;
                const uint64_t off = (uint64_t)b * (uint32_t)p.sb + (uint32_t)(at * (int)p.ss);
                const u32x4 k = __builtin_amdgcn_raw_buffer_load_b128(rsrc(kc + off), (int)(lane_off + at_row[j]), 0, 0);
                const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rsrc(vc + off), (int)(lane_off + at_row[j]), 0, 0);
                k_raw[j] = Vec16{{k.x, k.y, k.z, k.w}};
                v_raw[j] = Vec16{{v.x, v.y, v.z, v.w}};
                if (j < NR) {
                    const uint64_t so = (uint64_t)b * (uint32_t)p.ssb + (uint32_t)(at * (int)p.sss);
                    ks_raw[j] = __builtin_amdgcn_raw_buffer_load_b8(rsrc(ksb + so), (int)lane_sc, 0, 0);
                    vs_raw[j] = __builtin_amdgcn_raw_buffer_load_b8(rsrc(vsb + so), (int)lane_sc, 0, 0);
                }
            }
        } else {
            const int key = kt * kKT + row_of(0), at = (key < last ? key : last) & in_block;
            const int64_t off = (int64_t)blk * p.sb + at * p.ss, so = (int64_t)blk * p.ssb + at * p.sss;
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                k_raw[j] = load16(kc + off + at_row[j]);
                v_raw[j] = load16(vc + off + at_row[j]);
            }
            ks_raw[0] = ksb[so];
            vs_raw[0] = vsb[so];
        }
    };
    // Rows past the last key are zeros (whatever was loaded there): masked in S, and V finite.
    auto store_tile = [&](int kt, uint16_t* sk, uint16_t* sv, float* sks) {
        const bool ends = kt * kKT + kKT - 1 > last;
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const int jr = LINES ? j : 0;
            auto scale = [&](uint32_t b) {    // 2^(b - 127), infinite for 255
                const uint32_t e = b << 23;
                return __builtin_bit_cast(float, e > 0x00400000u ? e : 0x00400000u);
            };
            const float ks = scale(ks_raw[jr]), vs = scale(vs_raw[jr]);
            uint32_t a[8], b[8];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                a[2 * w] = Keys<T>::template cvt<false>(k_raw[j].w[w], ks);
                a[2 * w + 1] = Keys<T>::template cvt<true>(k_raw[j].w[w], ks);
                b[2 * w] = scaled_bf16<false>(v_raw[j].w[w], vs);
                b[2 * w + 1] = scaled_bf16<true>(v_raw[j].w[w], vs);
            }
            const bool bad = ks_raw[jr] == (uint32_t)kScaleNan || vs_raw[jr] == (uint32_t)kScaleNan;
            const bool none = ends && kt * kKT + row_of(j) > last;
            if (__builtin_amdgcn_ballot_w64(bad || none)) {
                asm volatile("");             // a branch, not selects in every tile
                const uint32_t fill = none ? 0u : Keys<T>::kNan2;
#pragma unroll
                for (int w = 0; w < 8; ++w) {
                    a[w] = bad || none ? fill : a[w];
                    b[w] = bad || none ? 0u : b[w];
                }
            }
            if (kAfter && j < NR && lane_c == 0) sks[row_of(j)] = ks;
            if (!live(j)) continue;
            store16((char*)sk + lds0[j], Vec16{{a[0], a[1], a[2], a[3]}});
            store16((char*)sk + lds1[j], Vec16{{a[4], a[5], a[6], a[7]}});
            store16((char*)sv + lds0[j], Vec16{{b[0], b[1], b[2], b[3]}});
            store16((char*)sv + lds1[j], Vec16{{b[4], b[5], b[6], b[7]}});
        }
    };

    // ---- LDS operands of this lane (as in the 16-bit kernel).
    const int grp = lane >> 4;
    const int tr_key = (lane & 15) >> 2;
    const int tr_col = 16 * (grp & 1) + 4 * (lane & 3);
    const int k_swz = lds_swizzle<D>(col);
    const int v_cb = tr_col >> 3;
    const int v_lo_swz = lds_swizzle<D>(4 * (grp >> 1) + tr_key);
    const int v_hi_swz = lds_swizzle<D>(4 * (grp >> 1) + tr_key + 8);
    const int v_byte = 8 * (lane & 1);
    uint32_t koff[DSTEPS], voff_lo[DTILES], voff_hi[DTILES];
#pragma unroll
    for (int s = 0; s < DSTEPS; ++s) {
        koff[s] = (uint32_t)(col * ROWB + (((2 * s + h) ^ k_swz) << 4));
        asm volatile("" : "+v"(koff[s]));
    }
#pragma unroll
    for (int t = 0; t < DTILES; ++t) {
        // Columns past head_dim re-read the tile's first chunks: output rows never stored.
        const int c = 4 * t + v_cb < CPR ? 4 * t + v_cb : 4 * t + (v_cb & 1);
        voff_lo[t] = (uint32_t)((4 * (grp >> 1) + tr_key) * ROWB + v_byte + ((c ^ v_lo_swz) << 4));
        voff_hi[t] = (uint32_t)((4 * (grp >> 1) + tr_key + 8) * ROWB + v_byte + ((c ^ v_hi_swz) << 4));
        asm volatile("" : "+v"(voff_lo[t]), "+v"(voff_hi[t]));
    }

    if (t_begin < t_end) load_ids(t_begin);
    // Q^T: lane supplies Q[its row][16 s + 8 h .. + 7], in NQ pieces.
    u32x4 qf[NQ][DSTEPS];
    {
        const T* q = reinterpret_cast<const T*>(p.q) + (q_first + my_q) * p.q_st + (int64_t)my_head * p.q_sh;
#pragma unroll
        for (int s = 0; s < DSTEPS; ++s) {
            if constexpr (sizeof(T) == 2) {
                const Vec16 v = load16(q + s * 16 + h * 8);
                qf[0][s] = u32x4{v.w[0], v.w[1], v.w[2], v.w[3]};
            } else {
                const Vec16 a = load16(q + s * 16 + h * 8), b = load16(q + s * 16 + h * 8 + 4);
                float x[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = __builtin_bit_cast(float, a.w[i]);
                    x[4 + i] = __builtin_bit_cast(float, b.w[i]);
                }
#pragma unroll
                for (int i = 0; i < NQ; ++i) {
                    qf[i][s] = u32x4{Mfma<E>::pack(x[0], x[1]), Mfma<E>::pack(x[2], x[3]), Mfma<E>::pack(x[4], x[5]),
                                     Mfma<E>::pack(x[6], x[7])};
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] -= (float)(__bf16)x[e];
                }
            }
        }
    }

    auto tile = [&](int kt, const uint16_t* tile_k, const uint16_t* tile_v, const float* tile_ks, uint16_t* nk,
                    uint16_t* nv, float* nks) {
        lds_barrier();                        // tile kt is staged, tile kt - 1 is done with
        const bool sees = kt * kKT < wave_kmax;
        f32x16 st[2];
        if (sees) {
            __builtin_amdgcn_s_setprio(1);
            st[0] = f32x16{};
            st[1] = f32x16{};
#pragma unroll
            for (int s = 0; s < DSTEPS; ++s)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint4 a = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(tile_k) +
                                                                    half * 32 * ROWB + koff[s]);
#pragma unroll
                    for (int i = 0; i < NQ; ++i) st[half] = Mfma<E>::run(u32x4{a.x, a.y, a.z, a.w}, qf[i][s], st[half]);
                }
            __builtin_amdgcn_s_setprio(0);
        }
        // The next tile's rows, loaded a tile ago, go to LDS in the shadow of the first product; the
        // loads of the one after it follow.
        if (kt + 1 < t_end) store_tile(kt + 1, nk, nv, nks);
        if (kt + 2 < t_end) load_tile(kt + 2);
        if (kt + 3 < t_end) load_ids(kt + 3);
        if (sees) {
            if constexpr (kAfter) {
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 ks = *reinterpret_cast<const float4*>(tile_ks + half * 32 + 8 * i + 4 * h);
                        st[half][4 * i] *= ks.x;
                        st[half][4 * i + 1] *= ks.y;
                        st[half][4 * i + 2] *= ks.z;
                        st[half][4 * i + 3] *= ks.w;
                    }
            }
            if (kt * kKT + kKT - 1 > first_pos) {
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int key = kt * kKT + half * 32 + 8 * (r >> 2) + 4 * h + (r & 3);
                        if (key > my_pos) st[half][r] = kNegInf;
                    }
            }
            float mt = kNegInf;
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int r = 0; r < 16; ++r) mt = fmaxf(mt, st[half][r]);
            mt = max_across32(mt) * scale_log2;   // scale > 0: max commutes with it
            asm("" : "+v"(mt));
            const bool raise = mt > m_run + kRescaleThreshold;
            const float m_new = raise ? mt : m_run;
            const float alpha = raise ? fast_exp2(m_run - mt) : 1.f;
            if (__builtin_amdgcn_ballot_w64(raise)) {
                asm volatile("");             // likewise
#pragma unroll
                for (int t = 0; t < DTILES; ++t) o[t] *= alpha;
            }
            m_run = m_new;
            const float m_off = m_new == kNegInf ? 0.f : m_new;
            float psum = 0.f;
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float e = fast_exp2(fmaf(st[half][r], scale_log2, -m_off));
                    st[half][r] = e;
                    psum += e;
                }
            psum = sum_across32(psum);
            l_run = l_run * alpha + psum;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                f32x16& sv = st[s >> 1];
                const int r0 = 8 * (s & 1);
                u32x4 pb[NP];
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    pb[i] = u32x4{Mfma<bf16_t>::pack(sv[r0 + 0], sv[r0 + 1]), Mfma<bf16_t>::pack(sv[r0 + 2], sv[r0 + 3]),
                                  Mfma<bf16_t>::pack(sv[r0 + 4], sv[r0 + 5]), Mfma<bf16_t>::pack(sv[r0 + 6], sv[r0 + 7])};
                    if (i + 1 < NP)
#pragma unroll
                        for (int e = 0; e < 8; ++e) sv[r0 + e] -= (float)(__bf16)sv[r0 + e];
                }
                const char* vgrp = reinterpret_cast<const char*>(tile_v) + ((s >> 1) * 32 + 16 * (s & 1)) * ROWB;
#pragma unroll
                for (int t = 0; t < DTILES; ++t) {
                    const uint2 lo = lds_read_tr16(reinterpret_cast<const uint16_t*>(vgrp + voff_lo[t]));
                    const uint2 hi = lds_read_tr16(reinterpret_cast<const uint16_t*>(vgrp + voff_hi[t]));
#pragma unroll
                    for (int i = 0; i < NP; ++i) o[t] = Mfma<bf16_t>::run(u32x4{lo.x, lo.y, hi.x, hi.y}, pb[i], o[t]);
                }
            }
        }
    };
    if (t_begin < t_end) {
        load_tile(t_begin);
        if (t_begin + 1 < t_end) load_ids(t_begin + 1);
        store_tile(t_begin, s_k0, s_v0, s_ks[0]);
        if (t_begin + 1 < t_end) load_tile(t_begin + 1);
        if (t_begin + 2 < t_end) load_ids(t_begin + 2);
    }
    for (int kt = t_begin; kt < t_end; kt += 2) {
        tile(kt, s_k0, s_v0, s_ks[0], s_k1, s_v1, s_ks[1]);
        if (kt + 1 < t_end) tile(kt + 1, s_k1, s_v1, s_ks[1], s_k0, s_v0, s_ks[0]);
    }

    // ---- store: the lane holds dims 32 t + 8 (r / 4) + 4 h + r % 4 of its row.
    if (!my_live) return;
    const int64_t tok = q_first + my_q;
    if (run < n_tiles && my_pos >= 0) {
        const int64_t row = tok * p.num_heads + my_head;
        const int64_t slot = row * p.splits + split;
        float* po = p.ws_o + slot * D + 4 * h;
#pragma unroll
        for (int t = 0; t < DTILES; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (32 * t + 8 * i < D)
                    *reinterpret_cast<float4*>(po + 32 * t + 8 * i) =
                        make_float4(o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]);
        // The merge skips a part whose maximum is -inf; one whose scores were all NaN has to count.
        if (h == 0)
            *reinterpret_cast<float2*>(p.ws_ml + slot * 2) =
                make_float2(m_run == kNegInf && l_run != 0.f ? 0.f : m_run, l_run);
        if (p.ws_rows && h == 0 && split == 0) p.ws_rows[row] = my_pos / (run * kKT) + 1;
        return;
    }
    if (split > 0) return;
    if (p.ws_rows && h == 0) p.ws_rows[tok * p.num_heads + my_head] = 0;   // finished here
    const float inv = l_run == 0.f ? 0.f : 1.f / l_run;                    // no key: zero
    T* orow = reinterpret_cast<T*>(p.out) + tok * p.out_st + (int64_t)my_head * p.out_sh;
#pragma unroll
    for (int t = 0; t < DTILES; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (32 * t + 8 * i >= D) continue;
            T* to = orow + 32 * t + 8 * i + 4 * h;
            const float4 v = make_float4(o[t][4 * i] * inv, o[t][4 * i + 1] * inv, o[t][4 * i + 2] * inv,
                                         o[t][4 * i + 3] * inv);
            if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(to) = v;
            else *reinterpret_cast<uint2*>(to) = make_uint2(Mfma<T>::pack(v.x, v.y), Mfma<T>::pack(v.z, v.w));
        }
}

template <typename T, int D>
int launch_kv8_chunk_d(const Kv8Params& p, hipStream_t stream) {
    const dim3 grid((unsigned)prefill_workgroups(p));
    if (p.block_size >= 16 && kv8_offsets_fit(p)) kv8_chunk_kernel<T, D, true><<<grid, 256, 0, stream>>>(p);
    else kv8_chunk_kernel<T, D, false><<<grid, 256, 0, stream>>>(p);
    const int rc = check_launch("kv8 chunk attention");
    if (rc || p.splits == 1) return rc;
    const int64_t rows = p.num_tokens * p.num_heads;
    prefill_merge_kernel<T, D><<<dim3((unsigned)ceil_div(rows, kMergeRows<D>)), 256, 0, stream>>>(p);
    return check_launch("kv8 chunk merge");
}

}  // namespace

template <typename T>
int launch_kv8_chunk(const Kv8Params& p, hipStream_t stream) {
    // One grid dimension; rows of a sequence in 32 bits.
    if (prefill_workgroups(p) > 0x7fffffff) return PKV_EUNSUPPORTED;
    if (((int64_t)p.max_query_len + kRows) * p.group > 0x7fffffff) return PKV_EUNSUPPORTED;
    switch (p.head_dim) {
        case 32: return launch_kv8_chunk_d<T, 32>(p, stream);
        case 48: return launch_kv8_chunk_d<T, 48>(p, stream);
        case 64: return launch_kv8_chunk_d<T, 64>(p, stream);
        case 80: return launch_kv8_chunk_d<T, 80>(p, stream);
        case 96: return launch_kv8_chunk_d<T, 96>(p, stream);
        case 112: return launch_kv8_chunk_d<T, 112>(p, stream);
        default: return launch_kv8_chunk_d<T, 128>(p, stream);
    }
}

}  // namespace pkv
