// What the MFMA prefill kernels share: matrix instructions and their operands' lane layouts, the
// LDS swizzle, split contexts and their merge kernel. (Internal to libpagedkv; every file that
// includes it has its own copies.)
#pragma once

#include "attention.h"

namespace pkv {
namespace {

constexpr int kKT = 64;          // keys per staged tile
constexpr int kQT = 32;          // query rows per wave
constexpr int kRows = 4 * kQT;   // query rows per workgroup

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Mfma;
template <>
struct Mfma<_Float16> {
    __device__ __forceinline__ static f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                      0, 0, 0);
    }
    __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
        half2_t v = {(_Float16)lo, (_Float16)hi};
        return __builtin_bit_cast(uint32_t, v);
    }
};
template <>
struct Mfma<bf16_t> {
    __device__ __forceinline__ static f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       c, 0, 0, 0);
    }
    __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
        bf16x2_t v = {(__bf16)lo, (__bf16)hi};
        return __builtin_bit_cast(uint32_t, v);
    }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Transposing LDS read (gfx950 ds_read_b64_tr_b16). Within each group of 16 lanes the
// 16 source addresses name 4 consecutive 16-bit elements each; taking those 64
// elements in (lane, element) order, result lane i receives elements i, i+16, i+32
// and i+48. With source lane c of a group pointing at V[key0 + c/4][d0 + 4*(c%4)] of a
// row-major tile, lane i therefore receives V[key0 .. key0+3][d0 + i]: four keys of
// one head_dim column, the MFMA A-operand slice of V^T. (Semantics pinned on the
// MI355X with an in-bounds probe.)
__device__ __forceinline__ uint2 lds_read_tr16(const uint16_t* ptr) {
    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(ptr));
    return __builtin_bit_cast(uint2, v);
}

// XOR swizzle of a K/V tile row in LDS: logical 16-byte chunk c of row r sits in
// physical slot c ^ lds_swizzle<D>(r) of the unpadded row (period 16 rows). Two
// constraints, for 16- and 32-lane LDS passes alike:
//  * a b128 K read takes one logical chunk of 16 consecutive rows: the swizzle is a
//    permutation over any 16 aligned rows, so the 16 reads hit 16 distinct slots;
//  * 32 lanes of a transposing V read take 4 aligned rows x 4 consecutive logical
//    chunks (one aligned 4-chunk block): the 4 rows' swizzles move that block to 4
//    different blocks, so the 16 reads are distinct too.
// D = 128 (16 chunks = 256 bytes per row, one bank sweep): slot c ^ (4 (r % 4) + r / 4 % 4).
// D = 64 (8 chunks per 128-byte row, two rows per bank sweep): rows of one parity share
// the sweep half, so the same two rules apply to each parity: c ^ (4 bit1 + 2 bit2 + bit3).
// Other widths only meet the first rule: rows 4 apart start in the same banks at D = 32
// and 96 (c ^ r / 4 % 4), rows 8 apart at 48, 80 and 112 (c ^ r / 8 % 2).
template <int D>
__device__ __forceinline__ int lds_swizzle(int r) {
    if constexpr (D == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (D == 64) return (((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1) | ((r >> 3) & 1);
    else if constexpr (D % 32 == 0) return (r >> 2) & 3;
    else return (r >> 3) & 1;
}

// Softmax maxima are only raised when a tile's max exceeds the running one by more
// than 2^8: until then probabilities are exp2(s - m) <= 256 (exact enough in fp32 and
// in the pool dtype), and the O accumulators need no rescale, which removes the per-tile
// multiply of every accumulator.
constexpr float kRescaleThreshold = 8.f;

// Tiles per split of a workgroup with n_tiles key tiles: its splits are of even lengths.
__device__ __forceinline__ int split_run(int n_tiles, int splits, int split_tiles) {
    const int n = split_count(n_tiles, splits, split_tiles);
    return (n_tiles + n - 1) / n;
}

// Merge of the splits, launched after the kernel above on the same stream: D / 4 lanes per
// query row (four head_dim elements each), log-sum-exp rule over the row's splits in key
// order. Rows that one workgroup finished are marked 0 and skipped, as are tokens of no
// sequence (rows the launch above never wrote: tokens past query_start_loc's end). Bound by
// the latency of its two dependent loads and by workgroup launches, hence as many rows per
// wave as fit.
template <int D>
constexpr int kMergeRows = 4 * (64 / (D / 4));   // query rows per 256-thread workgroup

template <typename T, int D>
__global__ __launch_bounds__(256) void prefill_merge_kernel(const AttnParams p) {
    constexpr int LPR = D / 4, RPW = 64 / LPR;
    const int lane = lane_id();
    if (lane >= RPW * LPR) return;
    const int64_t row = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * RPW + lane / LPR;
    const int64_t end = p.qsl ? p.qsl[p.num_seqs] : p.num_tokens;
    if (row >= end * p.num_heads) return;
    const int64_t tok = row / p.num_heads;
    int n;
    if (p.qsl) {
        n = p.ws_rows[row];
    } else {
        // A decode batch: the splits of the row's own context, none if it has only one.
        const int64_t cap = p.table_width * p.block_size;
        int64_t c = p.ctx_lens[tok];
        c = c < cap ? c : cap;
        const int tiles = (int)((c + kKT - 1) / kKT);
        const int run = split_run(tiles, p.splits, p.split_tiles);
        n = run > 0 && run < tiles ? (tiles + run - 1) / run : 0;
    }
    if (n <= 0 || n > p.splits) return;
    const int d = 4 * (lane % LPR);
    const float2* ml = reinterpret_cast<const float2*>(p.ws_ml) + row * p.splits;
    const float* o = p.ws_o + row * p.splits * D + d;
    constexpr int CH = 8;   // splits whose loads are in flight together
    float M = kNegInf, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < n; s0 += CH) {
        float2 mlv[CH];
        float4 ov[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const bool in = s0 + j < n;
            mlv[j] = in ? ml[s0 + j] : make_float2(kNegInf, 0.f);
            ov[j] = in ? *reinterpret_cast<const float4*>(o + (int64_t)(s0 + j) * D) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float Mc = M;
#pragma unroll
        for (int j = 0; j < CH; ++j) Mc = fmaxf(Mc, mlv[j].x);
        const float rescale = M == kNegInf ? 0.f : fast_exp2(M - Mc);
        L *= rescale;
        acc.x *= rescale;
        acc.y *= rescale;
        acc.z *= rescale;
        acc.w *= rescale;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const float sc = mlv[j].x == kNegInf ? 0.f : fast_exp2(mlv[j].x - Mc);
            L += sc * mlv[j].y;
            acc.x += sc * ov[j].x;
            acc.y += sc * ov[j].y;
            acc.z += sc * ov[j].z;
            acc.w += sc * ov[j].w;
        }
        M = Mc;
    }
    T* orow = reinterpret_cast<T*>(p.out) + tok * p.out_st + (row - tok * p.num_heads) * p.out_sh + d;
    const float inv = 1.f / L;
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(orow) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    else
        *reinterpret_cast<uint2*>(orow) =
            make_uint2(Mfma<T>::pack(acc.x * inv, acc.y * inv), Mfma<T>::pack(acc.z * inv, acc.w * inv));
}

// Workgroups of the flat grid, a multiple of 8: the splits' items, or room for every row
// tile the batch can hold (a sequence's last tile may be partial), whichever is more.
int64_t prefill_workgroups(const AttnParams& p) {
    const int64_t grid = ceil_div((int64_t)p.max_query_len * p.group, kRows) * p.num_seqs;
    const int64_t fill = p.num_tokens * p.group / kRows + p.num_seqs;
    int64_t items = (grid < fill || p.num_seqs > kPrefillSortSeqs ? grid : fill) * p.num_kv_heads;
    if (p.splits > 1 && p.split_items > items) items = p.split_items;
    return ceil_div(items, 8) * 8;
}

}  // namespace
}  // namespace pkv
