// Decode attention over the 8-bit paged cache on MFMA (gfx950): the kernel, instantiated by
// type in attn_kv8_decode_*.hip. Head_dim a multiple of 16 from 32 to 128, at most 16 rows
// ((token, query head) pairs) per (sequence, KV head), block sizes that are powers of two from
// 4 up, scale bytes of a block together (slot stride 1) and 4-byte aligned, codes in 4-byte
// steps, queries and output in 8-byte ones.
//
// Bound: HBM for batches of hundreds of MB (head_dim + 1 bytes a cached row: 64 sequences of
// 1-16k tokens, 8 KV heads of 128, 1.10 GB in 179-190 us, 5.8-6.2 TB/s, of which the arithmetic
// is 4 us); latency below that (32 sequences of 12 heads of 64, 23.5 MB, 13.9 us).
//
//  * Split: a batch's keys are taken in units of 32 (64 up to head_dim 64), a wave a unit at a
//    time, and cut into runs by one of three rules (attn_kv8.hip has the choice). Large batches:
//    even runs, over the ends of sequences, one a workgroup. Others: runs inside a sequence, a
//    workgroup each, or a wave each where there are more sequences than workgroups; a batch of
//    which none is cut is not summed up at all. Every workgroup finds its run by running sums of
//    its own over the lengths, so a graph's replays may change them.
//  * A sequence in several runs leaves fp32 partials, which the last workgroup to finish it
//    merges inside the launch, in an order that the number of parts fixes, so results do not depend
//    on timing.
//  * Operands as they lie: S^T = K Q^T on 16x16x32 takes quarters of K rows (the order of a
//    contraction is free as long as Q's is the same). Its result leaves a lane with 8 keys of one
//    query row, which are the B operand of O^T += V^T P^T as they stand. V^T's operand is 8 keys
//    of one dim a lane: the lane loads 4 (or 8) neighbouring dims of those 8 keys, and byte
//    permutes turn 4 x 4 blocks. Only at head_dim 128 does K pass through LDS, so that loads take
//    whole lines (below).
//  * Codes are converted in pairs (v_cvt_scalef32_pk): exact. Key scales multiply the scores,
//    value scales the weights, both in fp32.
//  * Weights enter the second product as bf16 pieces (two for 16-bit types: 16 bits of them,
//    three for fp32), fp32 queries the first one as three: the product is then as exact as its
//    fp32 accumulation, and the matrix unit has time to spare (20-24 MFMAs a unit of up to 8 KiB,
//    36-48 for fp32).
//  * A unit stays in registers; K of the next one is loaded when the first product has used
//    this one's, V after the second, the other waves of the SIMD (2-4) being the cover. Two
//    units in registers and half the waves were slower (64 sequences as above 203 us, 190 so).
//  * Heads of one run share an XCD (workgroup L runs on XCD L % 8): a line of scale bytes holds
//    several heads.
#pragma once

#include "kv8.h"

namespace pkv {
namespace {

// Keys a wave takes at a time: 8 KiB of K and V at most.
constexpr int unit_keys(int head_dim) { return head_dim <= 64 ? 64 : 32; }
constexpr int kDecodeRows = kKv8DecodeRows;
constexpr int kDecodeMaxSeqs = kKv8DecodeMaxSeqs;   // prefix sums in LDS
constexpr float kLazy = 8.f;                    // base 2: maxima are raised past 2^8 only

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_a4 __attribute__((ext_vector_type(2), aligned(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// N dwords at a 4-byte aligned address that the lane has, or at a lane's offset from a uniform one
// (a buffer load: no address arithmetic on the vector unit, where the compiler spends 64-bit
// adds and register pairs on every load of the plain form). Nontemporal.
template <int N>
__device__ __forceinline__ void load_dwords(const uint8_t* p, uint32_t (&w)[N]) {
#pragma unroll
    for (int i = 0; i + 4 <= N; i += 4) {
        const u32x4_a4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_a4*>(p + 4 * i));
        w[i] = v.x;
        w[i + 1] = v.y;
        w[i + 2] = v.z;
        w[i + 3] = v.w;
    }
    if constexpr (N % 4 >= 2) {
        const u32x2_a4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2_a4*>(p + 4 * (N & ~3)));
        w[N & ~3] = v.x;
        w[(N & ~3) + 1] = v.y;
    }
    if constexpr (N % 2) w[N - 1] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p + 4 * (N - 1)));
}
struct Uniform {
    __amdgpu_buffer_rsrc_t r;
    __device__ __forceinline__ explicit Uniform(const uint8_t* p)
        : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, -1, 0x00027000)) {}
};
// The nontemporal bit of a buffer load, for rows of whole 128-byte lines: shorter ones share lines
// with other heads' rows, which other workgroups of the XCD are to find in its L2 (32 GPT-2
// sequences 16.2 us with it, 14.8 without; 64 of 1-16k at head_dim 128 197 us, 205 without).
template <int D>
constexpr int kNt = D == 128 ? 2 : 0;
template <int NT, int N>
__device__ __forceinline__ void load_dwords(const Uniform& base, uint32_t lane_off, int off, uint32_t (&w)[N]) {
#pragma unroll
    for (int i = 0; i + 4 <= N; i += 4) {
        const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(base.r, (int)lane_off + 4 * i, off, NT);
        w[i] = v.x;
        w[i + 1] = v.y;
        w[i + 2] = v.z;
        w[i + 3] = v.w;
    }
    if constexpr (N % 4 >= 2) {
        const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(base.r, (int)lane_off + 4 * (N & ~3), off, NT);
        w[N & ~3] = v.x;
        w[(N & ~3) + 1] = v.y;
    }
    if constexpr (N % 2) w[N - 1] = __builtin_amdgcn_raw_buffer_load_b32(base.r, (int)lane_off + 4 * (N - 1), off, NT);
}

__device__ __forceinline__ f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const bf16x2_t v = {(__bf16)lo, (__bf16)hi};
    return __builtin_bit_cast(uint32_t, v);
}
// Two codes (the lower or upper half of w) as bf16.
template <bool HI>
__device__ __forceinline__ uint32_t codes_bf16(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HI));
}

// The first product by query type: pieces of q, and the keys' type.
template <typename T>
struct Qk {
    static constexpr int kPieces = 1;
    __device__ __forceinline__ static u32x4 keys(uint32_t a, uint32_t b) {
        return u32x4{codes_bf16<false>(a), codes_bf16<true>(a), codes_bf16<false>(b), codes_bf16<true>(b)};
    }
    __device__ __forceinline__ static f32x4 run(u32x4 a, u32x4 b, f32x4 c) { return mfma_bf16(a, b, c); }
};
template <>
struct Qk<_Float16> {
    static constexpr int kPieces = 1;
    template <bool HI>
    __device__ __forceinline__ static uint32_t cvt(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HI));
    }
    __device__ __forceinline__ static u32x4 keys(uint32_t a, uint32_t b) {
        return u32x4{cvt<false>(a), cvt<true>(a), cvt<false>(b), cvt<true>(b)};
    }
    __device__ __forceinline__ static f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                      0);
    }
};
template <>
struct Qk<float> : Qk<bf16_t> {
    static constexpr int kPieces = 3;
};

// Four scale bytes as 2^(b - 127). Infinity stands for NaN (255): the codes under it are 0, and
// 0 times infinity is NaN.
__device__ __forceinline__ void scales4(uint32_t w, float (&s)[4]) {
    const uint32_t e[4] = {w << 23, w << 15, w << 7, w >> 1};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t b = e[i] & 0x7f800000u;
        s[i] = __builtin_bit_cast(float, b > 0x00400000u ? b : 0x00400000u);
    }
}

// dims[j] = byte j of rows 0..3.
__device__ __forceinline__ void transpose4(const uint32_t (&row)[4], uint32_t (&dim)[4]) {
    const uint32_t l01 = __builtin_amdgcn_perm(row[1], row[0], 0x05010400), h01 = __builtin_amdgcn_perm(row[1], row[0], 0x07030602);
    const uint32_t l23 = __builtin_amdgcn_perm(row[3], row[2], 0x05010400), h23 = __builtin_amdgcn_perm(row[3], row[2], 0x07030602);
    dim[0] = __builtin_amdgcn_perm(l23, l01, 0x05040100);
    dim[1] = __builtin_amdgcn_perm(l23, l01, 0x07060302);
    dim[2] = __builtin_amdgcn_perm(h23, h01, 0x05040100);
    dim[3] = __builtin_amdgcn_perm(h23, h01, 0x07060302);
}

__device__ __forceinline__ float max_across16(float x) {
    const SwapPair s = swap16(x);
    return fmaxf(s.a, s.b);
}
__device__ __forceinline__ float sum_across16(float x) {
    const SwapPair s = swap16(x);
    return s.a + s.b;
}

// Four consecutive output elements.
template <typename T>
__device__ __forceinline__ void store4(T* to, float4 v);
template <>
__device__ __forceinline__ void store4<float>(float* to, float4 v) {
    *reinterpret_cast<float2*>(to) = make_float2(v.x, v.y);
    *reinterpret_cast<float2*>(to + 2) = make_float2(v.z, v.w);
}
template <>
__device__ __forceinline__ void store4<bf16_t>(bf16_t* to, float4 v) {
    *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}
template <>
__device__ __forceinline__ void store4<_Float16>(_Float16* to, float4 v) {
    const half2_t a = {(_Float16)v.x, (_Float16)v.y}, b = {(_Float16)v.z, (_Float16)v.w};
    *reinterpret_cast<uint2*>(to) = make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
}

__device__ __forceinline__ uint64_t pair_bits(float lo, float hi) {
    return (uint64_t)__builtin_bit_cast(uint32_t, hi) << 32 | __builtin_bit_cast(uint32_t, lo);
}
__device__ __forceinline__ float lo_of(uint64_t x) { return __builtin_bit_cast(float, (uint32_t)x); }
__device__ __forceinline__ float hi_of(uint64_t x) { return __builtin_bit_cast(float, (uint32_t)(x >> 32)); }
// Written through to, and read from, where every XCD sees it.
__device__ __forceinline__ void agent_store(uint64_t* p, uint64_t v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t agent_load(const uint64_t* p) {
    return __hip_atomic_load(const_cast<uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A running (maximum, denominator, 4 elements of the unnormalised output). l = 0: nothing yet.
// (The maximum of a part whose scores are all NaN is -inf; its l is NaN and must not be lost.)
struct Part {
    float m, l;
    float4 o;
    __device__ __forceinline__ void add(float pm, float pl, float4 po) {
        const float M = fmaxf(m, pm);
        const float a = l == 0.f ? 0.f : fast_exp2(m - M), b = pl == 0.f ? 0.f : fast_exp2(pm - M);
        m = M;
        l = a * l + b * pl;
        o = make_float4(a * o.x + b * po.x, a * o.y + b * po.y, a * o.z + b * po.z, a * o.w + b * po.w);
    }
    // A row that sees no key is zero.
    __device__ __forceinline__ float4 result() const {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        return make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
};

// LDS of a workgroup of W waves: the waves' parts of a segment.
template <int D, int W>
struct DecodeLds {
    __attribute__((aligned(16))) float o[W][kDecodeRows * D];
    float2 ml[W][kDecodeRows];
    uint32_t arrived[W];
};

__device__ __forceinline__ int decode_ctx(const Kv8Params& p, int seq) {
    const int64_t cap = p.table_width * (int64_t)p.block_size, c = p.ctx_lens[seq];
    return (int)(c < 0 ? 0 : c < cap ? c : cap);
}
// Units of a sequence; one that has queries has one at least.
template <int D>
__device__ __forceinline__ int decode_units(const Kv8Params& p, int seq) {
    const int u = (int)(((uint32_t)decode_ctx(p, seq) + unit_keys(D) - 1) / unit_keys(D));
    if (p.qsl && p.qsl[seq + 1] <= p.qsl[seq]) return 0;
    return u > 0 ? u : 1;
}

// The threads of a run of NW waves: its workgroup's, or its wave's.
template <int NW>
__device__ __forceinline__ void run_sync() {
    if constexpr (NW > 1) lds_barrier(); else wave_lds_sync();
}

// Units [a, b) of sequence `seq` for KV head kvh by NW waves. parts = 1: all of the sequence (b
// is not looked at). Else the sequence is cut into so many parts, of which this is one: its
// partial is number own(), the k-th one part_of(k).
// BIG: block sizes from 16 up, where 16 keys share a block and addresses are uniform.
template <typename T, int D, bool BIG, int NW, typename Lds, typename Own, typename PartOf>
__device__ __forceinline__ void decode_segment(const Kv8Params& p, Lds& lds, int seq, int kvh, int a, int b, int parts,
                                               Own own, PartOf part_of) {
    const bool whole = parts == 1;
    constexpr int KD = D / 16;                  // dwords of K a lane holds of each row
    constexpr int KS = (D + 31) / 32;           // contraction steps of S^T
    // Neighbouring dims of V that a lane holds: 8 at head_dim 128, else 4 of each 64.
    constexpr int VD = D == 128 ? 2 : (D + 63) / 64;   // dwords
    constexpr int NQ = Qk<T>::kPieces, NP = sizeof(T) == 4 ? 3 : 2;
    constexpr int kUnit = unit_keys(D), NT = kUnit / 16;    // tiles of 16 keys
    constexpr int NI = BIG ? 1 : 2 * NT;

    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int n = lane & 15, kb = lane >> 4;
    const int G = p.group, heads = p.num_kv_heads;
    int x = a + (NW > 1 ? wave : 0);            // this wave's unit, in steps of NW

    // ---- block ids of a unit. BIG: lane l holds that of 16-key tile l % NT. Else each lane
    // those of its K rows and V row groups. Indexes stop at the row's end: what stands behind a
    // context's last block is never used.
    const int64_t* table = p.tables + (int64_t)seq * p.table_stride;
    const int last = (int)p.table_width - 1, in_block = p.block_size - 1;
    int64_t raw_ids[NI];
    auto load_ids = [&](int u) {
        auto id = [&](int key) {
            const int at = key >> p.block_shift;
            return table[at < last ? at : last];
        };
        if constexpr (BIG) {
            raw_ids[0] = id(kUnit * u + 16 * (lane & (NT - 1)));
        } else {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                raw_ids[t] = id(kUnit * u + 16 * t + n);
                raw_ids[NT + t] = id(kUnit * u + 16 * t + 4 * kb);
            }
        }
    };
    // The first unit's ids go out before the context's length is known.
    if (last >= 0) load_ids(x);

    const int ctx = __builtin_amdgcn_readfirstlane(decode_ctx(p, seq));
    const int64_t q_first = p.qsl ? p.qsl[seq] : seq;
    const int q_len = __builtin_amdgcn_readfirstlane(p.qsl ? (int)(p.qsl[seq + 1] - q_first) : 1);
    const int rows = q_len * G < p.decode_rows ? q_len * G : p.decode_rows;
    const int pos0 = ctx - q_len;               // of the first token
    const int row = n < rows ? n : rows - 1;
    const int limit = pos0 + row / G;           // last key that the row sees
    auto row_token = [&](int r) { return q_first + r / G; };
    auto row_head = [&](int r) { return (int64_t)kvh * G + r % G; };

    if (whole) b = (int)(((uint32_t)ctx + kUnit - 1) / kUnit);
    const uint8_t* kc = reinterpret_cast<const uint8_t*>(p.k) + kvh * p.sh;
    const uint8_t* vc = reinterpret_cast<const uint8_t*>(p.v) + kvh * p.sh;
    const uint8_t* ksb = p.ks + kvh * p.ssh;
    const uint8_t* vsb = p.vs + kvh * p.ssh;
    // Lane offsets: K row n of a tile, a quarter of it; V rows 4 kb .. 4 kb + 3, dims from n (past
    // head_dim: some others, never stored).
    // K: dims [kb D / 4, + D / 4), at head_dim 128 two pieces of 16, 64 dims apart.
    constexpr int KP = D == 128 ? 2 : 1, KW = KD / KP;      // pieces, dwords of one
    // At head_dim 128 a row is a 128-byte line, and loads that take it whole (8 lanes a row, 8 rows a
    // load) reach 6.1 TB/s where 64 bytes of 16 rows reach 5.5: the rows then pass through LDS (a
    // wave's own, its part of lds.o) on their way to the lanes that want them. 16-byte chunk c of
    // row r is at c ^ (r & 7), which keeps both the writes and the reads free of bank conflicts.
    constexpr bool LINES = D == 128 && BIG;
    const uint32_t k_off = LINES ? (uint32_t)((lane >> 3) * p.ss + (lane & 7) * 16)
                                 : (uint32_t)(kb * 4 * KW) + (BIG ? (uint32_t)(n * p.ss) : 0u);
    char* k_lds = reinterpret_cast<char*>(lds.o[wave]);
    const uint32_t k_put = (uint32_t)((lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3 & 7)) << 4));
    const uint32_t k_get[2] = {(uint32_t)(n * 128 + ((kb ^ (n & 7)) << 4)), (uint32_t)(n * 128 + (((kb + 4) ^ (n & 7)) << 4))};
    uint32_t v_off[VD];
#pragma unroll
    for (int c = 0; c < VD; ++c) {
        const int d = D == 128 ? 8 * n : 64 * c + 4 * n;
        v_off[c] = (uint32_t)(d < D ? d : 0) + (BIG ? (uint32_t)(4 * kb * p.ss) : 0u);
    }
    const uint32_t s_off = BIG ? (uint32_t)(4 * kb) : 0u;

    // K of a unit: rows 16 t + n; its scales, and V: rows 16 t + 4 kb + r.
    uint32_t kw[NT][KD], vw[NT][4][VD], ksw[NT], vsw[NT];
    uint64_t v_row[NT], s_row[NT];
    auto load_k = [&](int u) {
        uint32_t ids[NI];                       // none is followed out of the cache
#pragma unroll
        for (int i = 0; i < NI; ++i) ids[i] = (uint64_t)raw_ids[i] < (uint64_t)p.num_blocks ? (uint32_t)raw_ids[i] : 0u;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint32_t k_id = BIG ? (uint32_t)__builtin_amdgcn_readlane((int)ids[0], t) : ids[BIG ? 0 : t];
            const uint32_t v_id = BIG ? k_id : ids[BIG ? 0 : NT + t];
            const int k_at = (kUnit * u + 16 * t + (BIG ? 0 : n)) & in_block;
            const int v_at = (kUnit * u + 16 * t + (BIG ? 0 : 4 * kb)) & in_block;
            // Strides of a block and offsets inside it fit 32 bits.
            const uint64_t k_row = (uint64_t)k_id * (uint32_t)p.sb + (uint32_t)(k_at * (int)p.ss);
            v_row[t] = BIG ? k_row : (uint64_t)v_id * (uint32_t)p.sb + (uint32_t)(v_at * (int)p.ss);
            s_row[t] = (uint64_t)v_id * (uint32_t)p.ssb + (uint32_t)v_at;
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                uint32_t w[KW];
                if constexpr (BIG) load_dwords<kNt<D>>(Uniform(kc + k_row), k_off, LINES ? 8 * i * (int)p.ss : 64 * i, w);
                else load_dwords<KW>(kc + k_row + k_off + 64 * i, w);
#pragma unroll
                for (int e = 0; e < KW; ++e) kw[t][KW * i + e] = w[e];
            }
            if constexpr (BIG) {
                ksw[t] = __builtin_amdgcn_raw_buffer_load_b32(Uniform(ksb + s_row[t]).r, (int)s_off, 0, 0);
            } else {
                ksw[t] = *reinterpret_cast<const uint32_t*>(ksb + s_row[t]);
            }
        }
    };
    auto load_v = [&]() {
        constexpr int VL = D == 128 ? 1 : VD, VN = VD / VL;     // loads a row, dwords a load
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < VL; ++c) {
                    uint32_t w[VN];
                    if constexpr (BIG) load_dwords<kNt<D>>(Uniform(vc + v_row[t]), v_off[c], r * (int)p.ss, w);
                    else load_dwords<VN>(vc + v_row[t] + r * p.ss + v_off[c], w);
#pragma unroll
                    for (int i = 0; i < VN; ++i) vw[t][r][c + i] = w[i];
                }
            if constexpr (BIG) vsw[t] = __builtin_amdgcn_raw_buffer_load_b32(Uniform(vsb + s_row[t]).r, (int)s_off, 0, 0);
            else vsw[t] = *reinterpret_cast<const uint32_t*>(vsb + s_row[t]);
        }
    };

    const bool any = ctx > 0 && x < b;
    // Q^T: the lane's row, the dims that it has of K, 8 a step.
    constexpr int QW = D / 4 * (int)sizeof(T) / 8;
    uint2 qraw[QW];
    {
        const T* q = reinterpret_cast<const T*>(p.q) + row_token(row) * p.q_st + row_head(row) * p.q_sh + kb * (4 * KW);
#pragma unroll
        for (int i = 0; i < QW; ++i) qraw[i] = reinterpret_cast<const uint2*>(q + (i / (QW / KP)) * 64)[i % (QW / KP)];
    }
    if (any) {
        load_k(x);
        load_v();
        load_ids(x + NW);
    }
    u32x4 qf[NQ][KS];
#pragma unroll
    for (int j = 0; j < KS; ++j) {
        uint32_t w[NQ][4] = {};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (8 * j + 4 * half >= D / 4) continue;
            if constexpr (sizeof(T) == 2) {
                w[0][2 * half] = qraw[2 * j + half].x;
                w[0][2 * half + 1] = qraw[2 * j + half].y;
            } else {
                const uint2 u = qraw[4 * j + 2 * half], v = qraw[4 * j + 2 * half + 1];
                float r[4] = {__builtin_bit_cast(float, u.x), __builtin_bit_cast(float, u.y),
                              __builtin_bit_cast(float, v.x), __builtin_bit_cast(float, v.y)};
#pragma unroll
                for (int i = 0; i < NQ; ++i) {
                    w[i][2 * half] = pack_bf16(r[0], r[1]);
                    w[i][2 * half + 1] = pack_bf16(r[2], r[3]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) r[e] -= (float)(__bf16)r[e];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NQ; ++i) qf[i][j] = u32x4{w[i][0], w[i][1], w[i][2], w[i][3]};
    }

    f32x4 o[4 * VD];
#pragma unroll
    for (int i = 0; i < 4 * VD; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = kNegInf, l_run = 0.f;         // l: this lane's keys only, until the end

    while (any) {
        const int key0 = kUnit * x;
        const bool masked = key0 + kUnit - 1 > pos0;         // some row does not see some key
        const bool more = x + NW < b;
        if constexpr (LINES) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < KP; ++i)
                    store16(k_lds + 2048 * t + 1024 * i + k_put,
                            Vec16{{kw[t][4 * i], kw[t][4 * i + 1], kw[t][4 * i + 2], kw[t][4 * i + 3]}});
            wave_lds_sync();
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < KP; ++i) {
                    const Vec16 v = load16(k_lds + 2048 * t + k_get[i]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) kw[t][4 * i + e] = v.w[e];
                }
            wave_lds_sync();
        }
        float s[4 * NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f32x4 st = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                const u32x4 kf = Qk<T>::keys(kw[t][2 * j], 2 * j + 1 < KD ? kw[t][2 * j + 1 < KD ? 2 * j + 1 : 0] : 0u);
#pragma unroll
                for (int i = 0; i < NQ; ++i) st = Qk<T>::run(kf, qf[i][j], st);
            }
            float ks4[4];
            scales4(ksw[t], ks4);
#pragma unroll
            for (int r = 0; r < 4; ++r) s[4 * t + r] = st[r] * ks4[r] * p.scale_log2;
        }
        // K's registers are free: the next unit's, under this one's softmax and second product. V's
        // follow below, under the next one's first product.
        if (more) load_k(x + NW);
        if (masked) {
            asm volatile("");                   // a branch, not selects in every unit
#pragma unroll
            for (int e = 0; e < 4 * NT; ++e) {
                const int key = key0 + 16 * (e >> 2) + 4 * kb + (e & 3);
                if (key > limit) s[e] = kNegInf;
                // Slots behind the context hold anything: 0 times a NaN would be NaN.
                if (key >= ctx)
#pragma unroll
                    for (int c = 0; c < VD; ++c) vw[e >> 2][e & 3][c] = 0;
            }
        }
        float mt = s[0];
#pragma unroll
        for (int e = 1; e < 4 * NT; ++e) mt = fmaxf(mt, s[e]);
        mt = max_across32(max_across16(mt));
        const bool raise = mt > m_run + kLazy;
        if (__builtin_amdgcn_ballot_w64(raise)) {
            const float alpha = raise ? fast_exp2(m_run - mt) : 1.f;
#pragma unroll
            for (int i = 0; i < 4 * VD; ++i) o[i] *= alpha;
            l_run *= alpha;
            m_run = raise ? mt : m_run;
        }
        const float m_off = m_run == kNegInf ? 0.f : m_run;
        float w[4 * NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float vs4[4];
            scales4(vsw[t], vs4);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float pe = fast_exp2(s[4 * t + r] - m_off);
                l_run += pe;
                w[4 * t + r] = pe * vs4[r];
            }
        }
        if (masked) {
            asm volatile("");
#pragma unroll
            for (int e = 0; e < 4 * NT; ++e)
                if (key0 + 16 * (e >> 2) + 4 * kb + (e & 3) > limit) w[e] = 0.f;
        }
        // 32 keys a step: tiles 2 h and 2 h + 1.
#pragma unroll
        for (int h = 0; h < NT / 2; ++h) {
            float* wh = w + 8 * h;
            u32x4 pf[NP];
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                pf[i] = u32x4{pack_bf16(wh[0], wh[1]), pack_bf16(wh[2], wh[3]), pack_bf16(wh[4], wh[5]),
                              pack_bf16(wh[6], wh[7])};
                if (i + 1 < NP)
#pragma unroll
                    for (int e = 0; e < 8; ++e) wh[e] -= (float)(__bf16)wh[e];
            }
#pragma unroll
            for (int c = 0; c < VD; ++c) {
                uint32_t d0[4], d1[4];
                const uint32_t r0[4] = {vw[2 * h][0][c], vw[2 * h][1][c], vw[2 * h][2][c], vw[2 * h][3][c]};
                const uint32_t r1[4] = {vw[2 * h + 1][0][c], vw[2 * h + 1][1][c], vw[2 * h + 1][2][c], vw[2 * h + 1][3][c]};
                transpose4(r0, d0);
                transpose4(r1, d1);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const u32x4 vf = u32x4{codes_bf16<false>(d0[j]), codes_bf16<true>(d0[j]), codes_bf16<false>(d1[j]),
                                           codes_bf16<true>(d1[j])};
#pragma unroll
                    for (int i = 0; i < NP; ++i) o[4 * c + j] = mfma_bf16(vf, pf[i], o[4 * c + j]);
                }
            }
        }
        if (!more) break;
        load_v();
        x += NW;
        load_ids(x + NW);
    }

    // ---- the waves' parts meet in LDS, row by row.
    l_run = sum_across32(sum_across16(l_run));
    if (n < rows) {
#pragma unroll
        for (int c = 0; c < VD; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = D == 128 ? 8 * (4 * kb + r) + 4 * c : 64 * c + 4 * (4 * kb + r);
                if (d < D)
                    *reinterpret_cast<float4*>(&lds.o[wave][n * D + d]) =
                        make_float4(o[4 * c][r], o[4 * c + 1][r], o[4 * c + 2][r], o[4 * c + 3][r]);
            }
        if (kb == 0) lds.ml[wave][n] = make_float2(m_run, l_run);
    }
    run_sync<NW>();
    constexpr int nthr = 64 * NW;
    const int thr = NW > 1 ? (int)threadIdx.x : lane, wave0 = NW > 1 ? 0 : wave;
    const int items = rows * (D / 4);           // 4 elements of a row each
    auto out4 = [&](int e, const Part& x4) {
        const int r = e / (D / 4), d = e % (D / 4) * 4;
        store4<T>(reinterpret_cast<T*>(p.out) + row_token(r) * p.out_st + row_head(r) * p.out_sh + d, x4.result());
    };
    auto partial = [&](int64_t number, int r) { return (number * heads + kvh) * p.decode_rows + r; };
    for (int e = thr; e < items; e += nthr) {
        const int r = e / (D / 4);
        Part acc = {kNegInf, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
        // All reads and exponentials side by side, as in Part::add.
        float2 ml[NW];
        float4 po[NW];
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            ml[w] = lds.ml[wave0 + w][r];
            po[w] = *reinterpret_cast<const float4*>(&lds.o[wave0 + w][e * 4]);
            acc.m = fmaxf(acc.m, ml[w].x);
        }
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float a = ml[w].y == 0.f ? 0.f : fast_exp2(ml[w].x - acc.m);
            acc.l += a * ml[w].y;
            acc.o.x += a * po[w].x;
            acc.o.y += a * po[w].y;
            acc.o.z += a * po[w].z;
            acc.o.w += a * po[w].w;
        }
        if (whole) {
            out4(e, acc);
        } else {
            const int64_t at = partial(own(), r);
            uint64_t* po = reinterpret_cast<uint64_t*>(p.ws_o + at * D + e % (D / 4) * 4);
            agent_store(po, pair_bits(acc.o.x, acc.o.y));
            agent_store(po + 1, pair_bits(acc.o.z, acc.o.w));
            if (e % (D / 4) == 0) agent_store(reinterpret_cast<uint64_t*>(p.ws_ml + at * 2), pair_bits(acc.m, acc.l));
        }
    }
    if (!whole) {
        // The stores have reached the agent's coherence point before the counter moves (a
        // release fence would write back the XCD's whole L2 instead).
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        run_sync<NW>();
        uint32_t* cnt = p.ws_cnt + ((int64_t)seq * heads + kvh);
        if (thr == 0) lds.arrived[wave0] = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        run_sync<NW>();
        if (__builtin_amdgcn_readfirstlane(lds.arrived[wave0]) == (uint32_t)(parts - 1)) {
            if (thr == 0) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            // Threads beyond the items share the parts: group g takes g, g + groups, ...; group 0
            // then adds the groups up, in order.
            int groups = 1;
            while (groups * 2 * items <= nthr && groups < parts) groups *= 2;
            const int g = groups > 1 ? thr / items : 0;
            float* so = lds.o[wave0];           // the parts are out: free (8 floats a thread)
            constexpr int CH = 4;               // partials whose loads are in flight together
            for (int e0 = 0; e0 < items; e0 += nthr) {
                const int e = e0 + thr - g * items, r = e / (D / 4);
                const bool mine = g < groups && e < items;
                Part acc = {kNegInf, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
                for (int s = g; mine && s < parts; s += CH * groups) {
                    uint64_t ml[CH], oa[CH], ob[CH];
#pragma unroll
                    for (int j = 0; j < CH; ++j) {
                        const int64_t at = partial(part_of(s + j * groups < parts ? s + j * groups : parts - 1), r);
                        const uint64_t* po = reinterpret_cast<const uint64_t*>(p.ws_o + at * D + e % (D / 4) * 4);
                        ml[j] = agent_load(reinterpret_cast<const uint64_t*>(p.ws_ml + at * 2));
                        oa[j] = agent_load(po);
                        ob[j] = agent_load(po + 1);
                    }
#pragma unroll
                    for (int j = 0; j < CH; ++j)
                        if (s + j * groups < parts)
                            acc.add(lo_of(ml[j]), hi_of(ml[j]),
                                    make_float4(lo_of(oa[j]), hi_of(oa[j]), lo_of(ob[j]), hi_of(ob[j])));
                }
                if (groups > 1) {
                    if (mine && g > 0) {
                        float* to = so + ((g - 1) * items + e) * 8;
                        *reinterpret_cast<float4*>(to) = acc.o;
                        *reinterpret_cast<float2*>(to + 4) = make_float2(acc.m, acc.l);
                    }
                    run_sync<NW>();
                    for (int k = 0; mine && g == 0 && k < groups - 1; ++k) {
                        const float* from = so + (k * items + e) * 8;
                        const float2 ml = *reinterpret_cast<const float2*>(from + 4);
                        acc.add(ml.x, ml.y, *reinterpret_cast<const float4*>(from));
                    }
                }
                if (mine && g == 0) out4(e, acc);
            }
        }
    }
}

// (Slot, KV head) of a workgroup or wave: the heads of 8 slots take 8 * heads of them, one slot an
// XCD (workgroup L runs on XCD L % 8).
template <int NW>
__device__ __forceinline__ void decode_place(const Kv8Params& p, int wave, int& slot, int& kvh) {
    const int id = NW > 1 ? (int)blockIdx.x : ((int)blockIdx.x >> 3) * 32 + (int)(blockIdx.x & 7) + 8 * wave;
    const int set = id / (8 * p.num_kv_heads), in = id - set * (8 * p.num_kv_heads);
    slot = set * 8 + (in & 7);
    kvh = in >> 3;
}

// Exclusive running sums of v over the workgroup's W waves, and their total.
template <int W>
__device__ __forceinline__ int block_scan(int v, int* s_wave, int& total) {
    const int lane = lane_id(), wave = (int)(threadIdx.x >> 6);
    int run = wave_scan(v);
    lds_barrier();                              // s_wave's last readers are done
    if (lane == 63) s_wave[wave] = run;
    lds_barrier();
    total = 0;
    for (int w = 0; w < W; ++w) total += s_wave[w];
    run -= v;
    for (int w = 0; w < wave; ++w) run += s_wave[w];
    return run;
}
// Waves a SIMD that registers are held to (128, 168 or 256 a lane): what fits without spills.
template <typename T, int D, bool LEAN>
constexpr int kDecodeWaves = sizeof(T) == 2 ? (D <= 64 && LEAN ? 4 : 3) : (D <= 80 && (LEAN || D == 80) ? 3 : 2);
// Waves of a workgroup that has one run: as many workgroups as registers have room for, so that
// 8 waves only where two of them fit.
template <typename T, int D, bool BIG>
constexpr int kRunWaves = kDecodeWaves<T, D, BIG> == 4 ? 8 : 4;
constexpr int kDecodePer = kDecodeMaxSeqs / 256;    // sequences per thread, at most

// Even runs: the batch's units, sequence after sequence, cut into equal slots.
template <typename T, int D, bool BIG>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kDecodeWaves<T, D, false>))) void kv8_decode_even_kernel(const Kv8Params p) {
    __shared__ int s_before[kDecodeMaxSeqs + 1];
    __shared__ int s_wave[4];
    __shared__ DecodeLds<D, 4> lds;
    const int per = (p.num_seqs + 255) / 256, first = (int)threadIdx.x * per;
    int total;
    {
        int own = 0, u[kDecodePer];
#pragma unroll
        for (int j = 0; j < kDecodePer; ++j) {
            u[j] = j < per && first + j < p.num_seqs ? decode_units<D>(p, first + j) : 0;
            own += u[j];
        }
        int run = block_scan<4>(own, s_wave, total);
#pragma unroll
        for (int j = 0; j < kDecodePer; ++j)
            if (j < per && first + j < p.num_seqs) {
                s_before[first + j] = run;
                run += u[j];
            }
        if (threadIdx.x == 0) s_before[p.num_seqs] = total;
        lds_barrier();
    }
    total = __builtin_amdgcn_readfirstlane(total);
    int slots = total / p.decode_min_units, slot, kvh;
    slots = slots < 1 ? 1 : slots < p.decode_slots ? slots : p.decode_slots;
    decode_place<4>(p, 0, slot, kvh);
    if (slot >= slots) return;
    // Slots [0, more) have len + 1 units, the others len.
    const int len = total / slots, more = total - len * slots;
    auto start_of = [&](int s) { return s * len + (s < more ? s : more); };
    auto slot_of = [&](int u) { return u < more * (len + 1) ? u / (len + 1) : (u - more) / len; };
    const int u0 = start_of(slot), u1 = start_of(slot + 1);
    int seq = 0;
    for (int hi = p.num_seqs; hi - seq > 1;) {      // the last sequence with s_before <= u0
        const int mid = (seq + hi) >> 1;
        if (s_before[mid] <= u0) seq = mid; else hi = mid;
    }
    seq = __builtin_amdgcn_readfirstlane(seq);
    for (; seq < p.num_seqs; ++seq) {
        const int before = __builtin_amdgcn_readfirstlane(s_before[seq]);
        const int after = __builtin_amdgcn_readfirstlane(s_before[seq + 1]);
        if (before >= u1) break;
        if (after == before) continue;
        const int a = before < u0 ? u0 - before : 0, b = after > u1 ? u1 - before : after - before;
        // A slot's partials: number 2 s of the sequence that it begins in, 2 s + 1 of the one that
        // it ends in.
        const int s0 = slot_of(before), s1 = slot_of(after - 1);
        decode_segment<T, D, BIG, 4>(
            p, lds, seq, kvh, a, b, s1 - s0 + 1, [&]() { return 2 * slot + (before <= u0 ? 0 : 1); },
            [&](int k) { return 2 * (s0 + k) + (start_of(s0 + k) < before ? 1 : 0); });
        lds_barrier();                              // lds is free again
    }
}

// Runs that stay inside a sequence: the shortest, no less than decode_min_units, with which all of
// them are at most decode_slots (twice the sequences if that is more); a sequence's are of even
// lengths. A workgroup of NW waves has one; NW = 1: each of four waves. decode_whole: no sequence
// is cut, so that a run's sequence is its number and there is nothing to sum up.
template <typename T, int D, bool BIG, int NW>
__global__ __launch_bounds__(NW > 1 ? 64 * NW : 256) __attribute__((amdgpu_waves_per_eu(kDecodeWaves<T, D, BIG>)))
void kv8_decode_runs_kernel(const Kv8Params p) {
    constexpr int W = NW > 1 ? NW : 4;
    __shared__ int s_wave[W];
    __shared__ int s_found[4][4];                   // by run of the workgroup
    __shared__ DecodeLds<D, W> lds;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    int slot, kvh;
    decode_place<NW>(p, wave, slot, kvh);
    if (p.decode_whole) {
        if (slot >= p.num_seqs || (p.qsl && p.qsl[slot + 1] <= p.qsl[slot])) return;
        decode_segment<T, D, BIG, NW>(p, lds, slot, kvh, 0, 0, 1, [&]() { return 0; }, [&](int) { return 0; });
        return;
    }
    constexpr int kWhole = 1 << 30;                 // units: no sequence has more
    int seq, runs, number, units;                   // a sequence, its runs, this one's number, its units
    auto run_length = [&](int total) {
        const int room = p.decode_slots > 2 * p.num_seqs ? p.decode_slots - p.num_seqs : p.num_seqs;
        const int even = (total + room - 1) / room;
        return p.decode_min_units > even ? p.decode_min_units : even;
    };
    if (p.num_seqs <= 64) {
        // Every wave for itself: lane i has sequence i.
        const int lane = lane_id();
        const int u = lane < p.num_seqs ? decode_units<D>(p, lane) : 0;
        int run = wave_scan(u);
        int len = run_length(__builtin_amdgcn_readlane(run, 63)), mine;
        while (true) {
            mine = (u + len - 1) / len;
            run = wave_scan(mine);
            if (__builtin_amdgcn_readlane(run, 63) <= p.decode_grid || len == kWhole) break;
            len = kWhole;                           // longer contexts than the grid was sized for
        }
        const uint64_t after = __builtin_amdgcn_ballot_w64(run > slot);
        if (!after) return;
        seq = __builtin_ctzll(after);
        runs = __builtin_amdgcn_readlane(mine, seq);
        number = slot - (__builtin_amdgcn_readlane(run, seq) - runs);
        units = __builtin_amdgcn_readlane(u, seq);
    } else {
        const int per = (p.num_seqs + 255) / 256, first = (int)threadIdx.x * per;   // of the first 256 threads
        int own = 0, u[kDecodePer], total;
#pragma unroll
        for (int j = 0; j < kDecodePer; ++j) {
            u[j] = j < per && first + j < p.num_seqs ? decode_units<D>(p, first + j) : 0;
            own += u[j];
        }
        block_scan<W>(own, s_wave, total);
        int len = run_length(total), run;
        while (true) {
            own = 0;
#pragma unroll
            for (int j = 0; j < kDecodePer; ++j) own += (u[j] + len - 1) / len;
            run = block_scan<W>(own, s_wave, total);
            if (total <= p.decode_grid || len == kWhole) break;
            len = kWhole;
        }
        // The thread that has a run's sequence says so.
        if (threadIdx.x < 4) s_found[threadIdx.x][0] = -1;
        lds_barrier();
#pragma unroll
        for (int j = 0; j < kDecodePer; ++j) {
            const int mine = (u[j] + len - 1) / len;
            for (int w = 0; w < (NW > 1 ? 1 : 4); ++w) {
                int ws, head;
                decode_place<NW>(p, w, ws, head);
                if (mine && ws >= run && ws < run + mine) {
                    s_found[w][0] = first + j;
                    s_found[w][1] = mine;
                    s_found[w][2] = ws - run;
                    s_found[w][3] = u[j];
                }
            }
            run += mine;
        }
        lds_barrier();
        const int w = NW > 1 ? 0 : wave;
        seq = __builtin_amdgcn_readfirstlane(s_found[w][0]);
        if (seq < 0) return;
        runs = __builtin_amdgcn_readfirstlane(s_found[w][1]);
        number = __builtin_amdgcn_readfirstlane(s_found[w][2]);
        units = __builtin_amdgcn_readfirstlane(s_found[w][3]);
    }
    const int each = units / runs, more = units - each * runs;      // runs [0, more) have one more
    const int a = number * each + (number < more ? number : more), b = a + each + (number < more ? 1 : 0);
    decode_segment<T, D, BIG, NW>(p, lds, seq, kvh, a, b, runs, [&]() { return slot; },
                                  [&](int k) { return slot - number + k; });
}

template <typename T, int D, bool BIG>
int launch_kv8_decode_d(const Kv8Params& p, hipStream_t stream) {
    const int64_t places = ceil_div(p.decode_grid, 8) * 8 * p.num_kv_heads;   // of (slot, KV head)
    const int64_t wgs = p.decode_mode == kKv8WaveRuns ? ceil_div(places, 32) * 8 : places;
    if (wgs > 0x7fffffff) return fail(PKV_EUNSUPPORTED, "kv8 decode attention: grid too large");
    const dim3 grid((unsigned)wgs);
    if (p.decode_mode == kKv8Even) kv8_decode_even_kernel<T, D, BIG><<<grid, 256, 0, stream>>>(p);
    else if (p.decode_mode == kKv8Runs)
        kv8_decode_runs_kernel<T, D, BIG, kRunWaves<T, D, BIG>><<<grid, 64 * kRunWaves<T, D, BIG>, 0, stream>>>(p);
    else kv8_decode_runs_kernel<T, D, BIG, 1><<<grid, 256, 0, stream>>>(p);
    return check_launch("kv8 decode attention");
}

template <typename T, bool BIG>
int launch_kv8_decode_b(const Kv8Params& p, hipStream_t stream) {
    switch (p.head_dim) {
        case 32: return launch_kv8_decode_d<T, 32, BIG>(p, stream);
        case 48: return launch_kv8_decode_d<T, 48, BIG>(p, stream);
        case 64: return launch_kv8_decode_d<T, 64, BIG>(p, stream);
        case 80: return launch_kv8_decode_d<T, 80, BIG>(p, stream);
        case 96: return launch_kv8_decode_d<T, 96, BIG>(p, stream);
        case 112: return launch_kv8_decode_d<T, 112, BIG>(p, stream);
        default: return launch_kv8_decode_d<T, 128, BIG>(p, stream);
    }
}

}  // namespace

template <typename T>
int launch_kv8_decode(const Kv8Params& p, hipStream_t stream) {
    return p.block_size >= 16 ? launch_kv8_decode_b<T, true>(p, stream) : launch_kv8_decode_b<T, false>(p, stream);
}

}  // namespace pkv
