// Decode attention over the 8-bit paged cache on MFMA (gfx950): the kernel, instantiated by
// type in attn_kv8_decode_*.hip. Head_dim a multiple of 16 from 32 to 128, at most 16 rows
// ((token, query head) pairs) per (sequence, KV head), block sizes that are powers of two from
// 4 up, codes in 4-byte steps, queries and output in 8-byte ones.
//
// Bound: HBM for batches of tens of MB (head_dim + 1 bytes a cached row), latency below that.
//
//  * Split: the batch's keys, in units of 32, sequence after sequence, are cut into `slots` even
//    runs per KV head, whatever the lengths: a prefix sum over the sequences, which every
//    workgroup takes by itself, tells it its own. A run is a workgroup's (its four waves take
//    turns at the units) or, where sequences are short and many, a single wave's. A sequence
//    that a run's end cuts leaves fp32 partials; the last workgroup to finish it merges them,
//    in key order, so results do not depend on timing.
//  * No LDS in the loop: S^T = K Q^T on 16x16x32 takes K rows as they lie in memory (a lane
//    holds a quarter of a row; the order of a contraction is free as long as Q's is the
//    same). Its result leaves a lane with 8 keys of one query row, which are the B operand of
//    O^T += V^T P^T as they stand. V^T's operand is 8 keys of one dim a lane: the lane loads 4
//    (or 8) neighbouring dims of those 8 keys, and byte permutes turn 4 x 4 blocks.
//  * Codes are converted in pairs (v_cvt_scalef32_pk): exact. Key scales multiply the scores,
//    value scales the weights, both in fp32.
//  * Weights enter the second product as bf16 pieces (two for 16-bit types: 16 bits of them,
//    three for fp32), fp32 queries the first one as three: the product is then as exact as its
//    fp32 accumulation, and the matrix unit has time to spare (12-40 MFMAs a unit of 8 KiB).
//  * Loads of the next unit are in flight while one is computed (16 KiB a wave at head_dim 128),
//    nontemporal, block ids one unit further ahead.
//  * Heads of one run share an XCD (workgroup L runs on XCD L % 8): a line of scale bytes holds
//    several heads.
#pragma once

#include "kv8.h"

namespace pkv {
namespace {

constexpr int kUnit = 32;                       // keys
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

// N dwords at a 4-byte aligned address.
template <int N>
__device__ __forceinline__ void load_dwords(const uint8_t* p, uint32_t (&w)[N]) {
    int i = 0;
#pragma unroll
    for (; i + 4 <= N; i += 4) {
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

// BIG: block sizes from 16 up, where 16 keys share a block and addresses are uniform.
template <typename T, int D, bool BIG>
__global__ __launch_bounds__(256) void kv8_decode_kernel(const Kv8Params p) {
    constexpr int KD = D / 16;                  // dwords of K a lane holds of each row
    constexpr int KS = (D + 31) / 32;           // contraction steps of S^T
    // Neighbouring dims of V that a lane holds: 8 at head_dim 128, else 4 of each 64.
    constexpr int VD = D == 128 ? 2 : (D + 63) / 64;   // dwords
    constexpr int NQ = Qk<T>::kPieces, NP = sizeof(T) == 4 ? 3 : 2;

    __shared__ int s_before[kDecodeMaxSeqs + 1];
    __shared__ int s_wave[4];
    __shared__ __attribute__((aligned(16))) float s_o[4][kDecodeRows * D];
    __shared__ float2 s_ml[4][kDecodeRows];
    __shared__ uint32_t s_arrived[4];

    const int tid = (int)threadIdx.x, lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, kb = lane >> 4;
    const int G = p.group;
    const int64_t cap = p.table_width * (int64_t)p.block_size;

    // ---- units before each sequence. A sequence with queries has one unit at least.
    auto ctx_of = [&](int i) {
        const int64_t c = p.ctx_lens[i];
        return (int)(c < 0 ? 0 : c < cap ? c : cap);
    };
    auto units_of = [&](int i) {
        if (p.qsl && p.qsl[i + 1] <= p.qsl[i]) return 0;
        const int u = (int)(((uint32_t)ctx_of(i) + kUnit - 1) / kUnit);
        return u > 0 ? u : 1;
    };
    const int per = (p.num_seqs + 255) / 256, first = tid * per;
    {
        int own = 0, u[8];                      // 2048 sequences over 256 threads
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            u[j] = j < per && first + j < p.num_seqs ? units_of(first + j) : 0;
            own += u[j];
        }
        int run = own;
#pragma unroll
        for (int by = 1; by < 64; by *= 2) {
            const int up = __shfl_up(run, by);
            if (lane >= by) run += up;
        }
        if (lane == 63) s_wave[wave] = run;
        __syncthreads();
        run -= own;
        for (int w = 0; w < wave; ++w) run += s_wave[w];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < per && first + j < p.num_seqs) {
                s_before[first + j] = run;
                run += u[j];
            }
        if (tid == 0) s_before[p.num_seqs] = s_wave[0] + s_wave[1] + s_wave[2] + s_wave[3];
        __syncthreads();
    }
    const int total = __builtin_amdgcn_readfirstlane(s_before[p.num_seqs]);

    // ---- this run: KV head, slot, units [u0, u1).
    const bool coop = p.decode_coop != 0;
    const int heads = p.num_kv_heads;
    int slots = total / p.decode_min_units;
    slots = slots < 1 ? 1 : slots < p.slots ? slots : p.slots;
    int kvh, slot;
    {
        // Workgroup L is on XCD L % 8: the heads of 8 slots take 8 * heads workgroups, one
        // slot an XCD.
        const int id = coop ? (int)blockIdx.x : ((int)blockIdx.x >> 3) * 32 + (int)(blockIdx.x & 7) + 8 * wave;
        const int set = id / (8 * heads), in = id % (8 * heads);
        slot = set * 8 + (in & 7);
        kvh = in >> 3;
    }
    if (slot >= slots) return;                  // uniform in the workgroup where it cooperates
    const int u0 = (int)((int64_t)slot * total / slots), u1 = (int)((int64_t)(slot + 1) * total / slots);
    int seq = 0;
    {
        int lo = 0, hi = p.num_seqs;            // the last sequence with s_before <= u0
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_before[mid] <= u0) lo = mid; else hi = mid;
        }
        seq = __builtin_amdgcn_readfirstlane(lo);
        // Sequences whole (no room for partials): those that begin in this run.
        if (!p.ws_o && s_before[seq] < u0) ++seq;
    }

    const uint8_t* kc = reinterpret_cast<const uint8_t*>(p.k) + kvh * p.sh;
    const uint8_t* vc = reinterpret_cast<const uint8_t*>(p.v) + kvh * p.sh;
    const uint8_t* ksb = p.ks + kvh * p.ssh;
    const uint8_t* vsb = p.vs + kvh * p.ssh;
    const bool scales_together = p.sss == 1 && p.scales4;
    // Lane offsets: K row n of a tile, a quarter of it; V rows 4 kb .. 4 kb + 3, dims from n (past
    // head_dim: some others, never stored).
    const uint32_t k_off = (uint32_t)(kb * (D / 4)) + (BIG ? (uint32_t)(n * p.ss) : 0u);
    uint32_t v_off[VD];
#pragma unroll
    for (int c = 0; c < VD; ++c) {
        const int d = D == 128 ? 8 * n : 64 * c + 4 * n;
        v_off[c] = (uint32_t)(d < D ? d : 0) + (BIG ? (uint32_t)(4 * kb * p.ss) : 0u);
    }
    const uint32_t s_off = BIG ? (uint32_t)(4 * kb * p.sss) : 0u;
    const int step = coop ? 4 : 1, turn = coop ? wave : 0;
    // Among the threads of a run: its workgroup, or its wave.
    auto sync = [&]() {
        if (coop) lds_barrier(); else wave_lds_sync();
    };

    struct Unit {
        uint32_t k[2][KD], v[2][4][VD], ks[2], vs[2];
    };

    for (; seq < p.num_seqs; ++seq) {
        const int before = __builtin_amdgcn_readfirstlane(s_before[seq]);
        const int after = __builtin_amdgcn_readfirstlane(s_before[seq + 1]);
        if (before >= u1) break;
        if (after == before) continue;
        const int a = p.ws_o && before < u0 ? u0 - before : 0;
        const int b = p.ws_o && after > u1 ? u1 - before : after - before;
        const bool whole = a == 0 && b == after - before;

        const int ctx = __builtin_amdgcn_readfirstlane(ctx_of(seq));
        const int64_t q_first = p.qsl ? p.qsl[seq] : seq;
        const int q_len = __builtin_amdgcn_readfirstlane(p.qsl ? (int)(p.qsl[seq + 1] - q_first) : 1);
        const int rows = q_len * G < kDecodeRows ? q_len * G : kDecodeRows;
        const int pos0 = ctx - q_len;           // of the first token
        const int row = n < rows ? n : rows - 1;
        const int limit = pos0 + row / G;       // last key that the row sees
        auto row_token = [&](int r) { return q_first + r / G; };
        auto row_head = [&](int r) { return (int64_t)kvh * G + r % G; };

        // ---- Q^T: elements [kb D / 4, + D / 4) of the lane's row, 8 a step.
        u32x4 qf[NQ][KS];
        {
            const T* q = reinterpret_cast<const T*>(p.q) + row_token(row) * p.q_st + row_head(row) * p.q_sh + kb * (D / 4);
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                uint32_t w[NQ][4] = {};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (8 * j + 4 * half >= D / 4) continue;
                    if constexpr (sizeof(T) == 2) {
                        const u32x2 v = *reinterpret_cast<const u32x2*>(q + 8 * j + 4 * half);
                        w[0][2 * half] = v.x;
                        w[0][2 * half + 1] = v.y;
                    } else {
                        const float2 x = *reinterpret_cast<const float2*>(q + 8 * j + 4 * half);
                        const float2 y = *reinterpret_cast<const float2*>(q + 8 * j + 4 * half + 2);
                        float r[4] = {x.x, x.y, y.x, y.y};
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
        }

        f32x4 o[4 * VD];
#pragma unroll
        for (int i = 0; i < 4 * VD; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m_run = kNegInf, l_run = 0.f;     // l: this lane's keys only, until the end

        // ---- block ids of a unit. BIG: lane l holds that of 16-key tile l % 2. Else each lane
        // those of its K rows and V row groups. Indexes stop at the context's last block.
        const int64_t* table = p.tables + (int64_t)seq * p.table_stride;
        const int last = (ctx - 1) >> p.block_shift;
        constexpr int NI = BIG ? 1 : 4;
        auto load_ids = [&](int x, int64_t (&ids)[NI]) {
            auto id = [&](int key) {
                const int at = key >> p.block_shift;
                const int64_t b = table[at < last ? at : last];
                return (uint64_t)b < (uint64_t)p.num_blocks ? b : 0;   // never followed out of the cache
            };
            if constexpr (BIG) {
                ids[0] = id(kUnit * x + 16 * (lane & 1));
            } else {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    ids[t] = id(kUnit * x + 16 * t + n);
                    ids[2 + t] = id(kUnit * x + 16 * t + 4 * kb);
                }
            }
        };
        const int in_block = p.block_size - 1;
        auto load_unit = [&](int x, const int64_t (&ids)[NI], Unit& f) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int64_t k_id = BIG ? readlane64(ids[0], t) : ids[BIG ? 0 : t];
                const int64_t v_id = BIG ? k_id : ids[BIG ? 0 : 2 + t];
                const int k_at = (kUnit * x + 16 * t + (BIG ? 0 : n)) & in_block;
                const int v_at = (kUnit * x + 16 * t + (BIG ? 0 : 4 * kb)) & in_block;
                const uint8_t* k = kc + (k_id * p.sb + k_at * p.ss);
                const uint8_t* v = vc + (v_id * p.sb + v_at * p.ss);
                load_dwords<KD>(k + k_off, f.k[t]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint8_t* vr = v + r * p.ss;
                    if constexpr (D == 128) {
                        load_dwords<2>(vr + v_off[0], f.v[t][r]);
                    } else {
#pragma unroll
                        for (int c = 0; c < VD; ++c)
                            f.v[t][r][c] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(vr + v_off[c]));
                    }
                }
                const int64_t so = v_id * p.ssb + v_at * p.sss;
                const uint8_t* ks = ksb + so + s_off;
                const uint8_t* vs = vsb + so + s_off;
                if (scales_together) {
                    f.ks[t] = *reinterpret_cast<const uint32_t*>(ks);
                    f.vs[t] = *reinterpret_cast<const uint32_t*>(vs);
                } else {
                    f.ks[t] = f.vs[t] = 0;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        f.ks[t] |= (uint32_t)ks[r * p.sss] << (8 * r);
                        f.vs[t] |= (uint32_t)vs[r * p.sss] << (8 * r);
                    }
                }
            }
        };

        auto compute = [&](int x, Unit& f) {
            const int key0 = kUnit * x;
            const bool masked = key0 + kUnit - 1 > pos0;     // some row does not see some key
            float s[8], vs[8];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f32x4 st = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    const u32x4 kf = Qk<T>::keys(f.k[t][2 * j], 2 * j + 1 < KD ? f.k[t][2 * j + 1 < KD ? 2 * j + 1 : 0] : 0u);
#pragma unroll
                    for (int i = 0; i < NQ; ++i) st = Qk<T>::run(kf, qf[i][j], st);
                }
                float ks4[4], vs4[4];
                scales4(f.ks[t], ks4);
                scales4(f.vs[t], vs4);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[4 * t + r] = st[r] * ks4[r] * p.scale_log2;
                    vs[4 * t + r] = vs4[r];
                }
            }
            if (masked) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = key0 + 16 * (e >> 2) + 4 * kb + (e & 3);
                    if (key > limit) s[e] = kNegInf;
                    // Slots behind the context hold anything: 0 times a NaN would be NaN.
                    if (key >= ctx)
#pragma unroll
                        for (int c = 0; c < VD; ++c) f.v[e >> 2][e & 3][c] = 0;
                }
            }
            float mt = s[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mt = fmaxf(mt, s[e]);
            mt = max_across32(max_across16(mt));
            const bool raise = mt > m_run + kLazy;
            const float m_new = raise ? mt : m_run;
            if (__builtin_amdgcn_ballot_w64(raise)) {
                const float alpha = raise ? fast_exp2(m_run - m_new) : 1.f;
#pragma unroll
                for (int i = 0; i < 4 * VD; ++i) o[i] *= alpha;
                l_run *= alpha;
                m_run = m_new;
            }
            const float m_off = m_run == kNegInf ? 0.f : m_run;
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float pe = fast_exp2(s[e] - m_off);
                l_run += pe;
                w[e] = pe * vs[e];
            }
            if (masked) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (key0 + 16 * (e >> 2) + 4 * kb + (e & 3) > limit) w[e] = 0.f;
            }
            u32x4 pf[NP];
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                pf[i] = u32x4{pack_bf16(w[0], w[1]), pack_bf16(w[2], w[3]), pack_bf16(w[4], w[5]), pack_bf16(w[6], w[7])};
                if (i + 1 < NP)
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] -= (float)(__bf16)w[e];
            }
#pragma unroll
            for (int c = 0; c < VD; ++c) {
                uint32_t d0[4], d1[4];
                const uint32_t r0[4] = {f.v[0][0][c], f.v[0][1][c], f.v[0][2][c], f.v[0][3][c]};
                const uint32_t r1[4] = {f.v[1][0][c], f.v[1][1][c], f.v[1][2][c], f.v[1][3][c]};
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
        };

        int x = a + turn;
        if (ctx > 0 && x < b) {
            Unit f, g;
            int64_t ids[NI];
            load_ids(x, ids);
            load_unit(x, ids, f);
            load_ids(x + step, ids);
            while (true) {
                if (x + step < b) {
                    load_unit(x + step, ids, g);
                    load_ids(x + 2 * step, ids);
                }
                compute(x, f);
                x += step;
                if (x >= b) break;
                if (x + step < b) {
                    load_unit(x + step, ids, f);
                    load_ids(x + 2 * step, ids);
                }
                compute(x, g);
                x += step;
                if (x >= b) break;
            }
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
                        *reinterpret_cast<float4*>(&s_o[wave][n * D + d]) =
                            make_float4(o[4 * c][r], o[4 * c + 1][r], o[4 * c + 2][r], o[4 * c + 3][r]);
                }
            if (kb == 0) s_ml[wave][n] = make_float2(m_run, l_run);
        }
        sync();
        const int nthr = coop ? 256 : 64, thr = coop ? tid : lane;
        const int parts = coop ? 4 : 1, part0 = coop ? 0 : wave;
        const int items = rows * (D / 4);       // 4 elements of a row each
        auto out4 = [&](int e, const Part& x4) {
            const int r = e / (D / 4), d = e % (D / 4) * 4;
            T* to = reinterpret_cast<T*>(p.out) + row_token(r) * p.out_st + row_head(r) * p.out_sh + d;
            store4<T>(to, x4.result());
        };
        // Partials of slot s: side 0 of the sequence that it begins in, side 1 of one that it ends in.
        auto partial = [&](int s, int side) { return ((int64_t)(s * 2 + side) * heads + kvh) * p.decode_rows; };
        for (int e = thr; e < items; e += nthr) {
            const int r = e / (D / 4);
            Part acc = {kNegInf, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
            for (int w = part0; w < part0 + parts; ++w) {
                const float2 ml = s_ml[w][r];
                acc.add(ml.x, ml.y, *reinterpret_cast<const float4*>(&s_o[w][e * 4]));
            }
            if (whole) {
                out4(e, acc);
            } else {
                const int64_t at = partial(slot, before <= u0 ? 0 : 1) + r;
                uint64_t* po = reinterpret_cast<uint64_t*>(p.ws_o + at * D + e % (D / 4) * 4);
                agent_store(po, pair_bits(acc.o.x, acc.o.y));
                agent_store(po + 1, pair_bits(acc.o.z, acc.o.w));
                if (e % (D / 4) == 0) agent_store(reinterpret_cast<uint64_t*>(p.ws_ml + at * 2), pair_bits(acc.m, acc.l));
            }
        }
        if (!whole) {
            // The stores have reached the agent's coherence point before the counter moves
            // (a release fence would write back the XCD's whole L2 instead).
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            sync();
            // Slots that hold a unit of this sequence.
            auto slot_of = [&](int64_t u) { return (int)(((u + 1) * slots - 1) / total); };
            const int s0 = slot_of(before), s1 = slot_of(after - 1);
            uint32_t* cnt = p.ws_cnt + ((int64_t)seq * heads + kvh);
            if (thr == 0) s_arrived[wave] = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            sync();
            const bool merge = __builtin_amdgcn_readfirstlane(s_arrived[coop ? 0 : wave]) == (uint32_t)(s1 - s0);
            if (merge) {
                if (thr == 0) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                // Threads beyond the items share the partials: group g takes s0 + g, s0 + g + groups,
                // ...; group 0 then adds the groups up, in order.
                int groups = 1;
                while (groups * 2 * items <= nthr) groups *= 2;
                const int g = groups > 1 ? thr / items : 0;
                float* so = s_o[part0];         // the parts are out: free (8 floats a thread)
                constexpr int CH = 4;           // partials whose loads are in flight together
                for (int e0 = 0; e0 < items; e0 += nthr) {
                    const int e = e0 + thr - g * items, r = e / (D / 4);
                    const bool mine = g < groups && e < items;
                    Part acc = {kNegInf, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
                    for (int s = s0 + g; mine && s <= s1; s += CH * groups) {
                        uint64_t ml[CH], oa[CH], ob[CH];
#pragma unroll
                        for (int j = 0; j < CH; ++j) {
                            const int sj = s + j * groups <= s1 ? s + j * groups : s1;
                            // Side 1 where the slot began before this sequence: the first one only.
                            const int64_t at = partial(sj, (int64_t)sj * total / slots < before ? 1 : 0) + r;
                            const uint64_t* po = reinterpret_cast<const uint64_t*>(p.ws_o + at * D + e % (D / 4) * 4);
                            ml[j] = agent_load(reinterpret_cast<const uint64_t*>(p.ws_ml + at * 2));
                            oa[j] = agent_load(po);
                            ob[j] = agent_load(po + 1);
                        }
#pragma unroll
                        for (int j = 0; j < CH; ++j)
                            if (s + j * groups <= s1)
                                acc.add(lo_of(ml[j]), hi_of(ml[j]),
                                        make_float4(lo_of(oa[j]), hi_of(oa[j]), lo_of(ob[j]), hi_of(ob[j])));
                    }
                    if (groups > 1) {
                        if (mine && g > 0) {
                            float* to = so + ((g - 1) * items + e) * 8;
                            *reinterpret_cast<float4*>(to) = acc.o;
                            *reinterpret_cast<float2*>(to + 4) = make_float2(acc.m, acc.l);
                        }
                        sync();
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
        sync();                                 // s_o, s_ml are free again
    }
}

template <typename T, int D>
int launch_kv8_decode_d(const Kv8Params& p, hipStream_t stream) {
    const int64_t sets = ceil_div(p.slots, 8) * 8 * p.num_kv_heads;   // (slot, head) pairs
    const int64_t wgs = p.decode_coop ? sets : ceil_div(sets, 32) * 8;
    if (wgs > 0x7fffffff) return fail(PKV_EUNSUPPORTED, "kv8 decode attention: grid too large");
    if (p.block_size >= 16) kv8_decode_kernel<T, D, true><<<dim3((unsigned)wgs), 256, 0, stream>>>(p);
    else kv8_decode_kernel<T, D, false><<<dim3((unsigned)wgs), 256, 0, stream>>>(p);
    return check_launch("kv8 decode attention");
}

}  // namespace

template <typename T>
int launch_kv8_decode(const Kv8Params& p, hipStream_t stream) {
    switch (p.head_dim) {
        case 32: return launch_kv8_decode_d<T, 32>(p, stream);
        case 48: return launch_kv8_decode_d<T, 48>(p, stream);
        case 64: return launch_kv8_decode_d<T, 64>(p, stream);
        case 80: return launch_kv8_decode_d<T, 80>(p, stream);
        case 96: return launch_kv8_decode_d<T, 96>(p, stream);
        case 112: return launch_kv8_decode_d<T, 112>(p, stream);
        default: return launch_kv8_decode_d<T, 128>(p, stream);
    }
}

}  // namespace pkv
