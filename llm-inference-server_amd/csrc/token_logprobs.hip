// Log probabilities of given tokens over rows of logits, their ranks, the rows' entropies and the
// `top` likeliest tokens of each row, in one pass over the logits.
//
//   y = x log2(e),  c = a whole number near the row's largest y,  s = sum 2^(y - c),  t = sum 2^(y - c) (y - c)
//   log p(i) = ln2 (y_i - c - log2 s),   entropy = ln2 (log2 s - t / s),   rank = 1 + #{x > x_i}
//
// A workgroup has one row, or one of `parts` pieces of it where there are few rows; the last piece
// of a row to finish merges them. A lane keeps (c, s, t) of its own in fp32 and raises c only when a
// tile exceeds it by more than 4; c is whole so that y - c is one fma, rounded once, in every lane. Logits
// are read once, 16 bytes a lane, whatever a row's alignment: its first and last 16 bytes are taken apart.
//
// Such references need |y| below 2^30. Logits far below it are nothing beside others; rows (pieces) that
// have a larger one, or only smaller ones, are summed again, against their largest logit itself.
//
// Top: the k-th largest of 64 maxima, of each lane over the waves, is a lower bound tau of the row's k-th
// largest logit so far, found by 16 ballots on the maxima's bits. A tile that holds something above it (most do
// not, after a few) raises it and appends what reaches it to the wave's list in LDS. Of logits equal to tau a
// wave takes k: of equal ones the lowest indices count, and a wave's indices rise. At the end the waves'
// lists, cut by the last tau, hold little more than k entries, which rank themselves by counting. Masked
// logits (-inf) never enter a list; if a row has fewer others than k, the lowest masked ids follow.
//
// Bound: HBM and, for 16-bit logits, the vector unit (an exponential takes four slots of the nine that a logit
// costs).
#include "pkv_common.h"

#include "attention.h"

namespace pkv {
namespace {

constexpr int kWaves = 4;
constexpr int kMaxTop = 64;             // a list's entries are ranked against one another; one lane max each
constexpr int kList = 640;              // a wave's: kMaxTop after a cut and a load of 512 logits
constexpr int kMerged = 1024;
constexpr float kRaise = 4.f;           // weights of up to 2^5: larger ones lose digits in their exponents' rounding
constexpr float kFar = 536870912.f;     // 2^29
constexpr float kLeast = -300.f;        // 2^kLeast and e^kLeast are 0 in fp32
constexpr float kLn2 = 0.6931471805599453f;

struct LogprobArgs {
    const void* logits;
    int64_t stride;                     // elements
    int vocab, parts, top;
    const int64_t* ids;
    float* logprobs;
    int64_t* ranks;
    float* entropy;
    float* top_logprobs;
    int64_t* top_ids;
    uint32_t* counters;                 // one a row, zero between calls
    uint64_t* partials;                 // [row][part][3 + top]: (m, s), (t, above), entries, keys
};

// Larger for larger logits, of equal ones for lower ids.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);       // one zero
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float x, int id) { return (uint64_t)order_of(x) << 32 | (uint32_t)~id; }
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, u >> 31 ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int id_of(uint64_t key) { return (int)~(uint32_t)key; }

__device__ __forceinline__ int lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// A lower bound of the k-th largest of the lanes' x (k <= 64), itself one of them.
__device__ __forceinline__ float kth_of_lanes(float x, int k) {
    const uint32_t u = order_of(x);
    uint32_t t = 0;
    for (uint32_t bit = 0x80000000u; bit > 0x8000u; bit >>= 1)
        if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(u >= (t | bit))) >= k) t |= bit;
    return -wave_max(u >= t ? -x : kNegInf);
}

// Of a lane, wave, piece or row. c, and t, in units of ln 2 for kNear, else of 1. The rows' levels:
enum { kBelow = 0, kNear = 1, kBeyond = 2, kNone = 3 };      // nothing above -2^29; the rule; above 2^29; NaN
struct Stat {
    float c, s, t;                      // s = 0: nothing yet
};

// BASE2: weights are 2^(y - c), else e^(x - c).
template <bool BASE2>
__device__ __forceinline__ Stat merge(Stat a, Stat b) {
    const float c = fmaxf(a.c, b.c);
    // (Bounded: c of -inf, and logits of the type's lowest value, are nothing and not 0 * -inf.)
    const float da = fmaxf(a.c - c, kLeast), db = fmaxf(b.c - c, kLeast);
    const float fa = fast_exp2(BASE2 ? da : da * kLog2e), fb = fast_exp2(BASE2 ? db : db * kLog2e);
    return Stat{c, a.s * fa + b.s * fb, fmaf(da, a.s, a.t) * fa + fmaf(db, b.s, b.t) * fb};
}

template <bool BASE2>
__device__ __forceinline__ Stat wave_merge(Stat x) {
#pragma unroll
    for (int off = 1; off < 64; off *= 2)
        x = merge<BASE2>(x, Stat{__shfl_xor(x.c, off), __shfl_xor(x.s, off), __shfl_xor(x.t, off)});
    return x;
}

// The largest float below x (-inf stays).
__device__ __forceinline__ float below(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    if (x == kNegInf) return x;
    return __builtin_bit_cast(float, x == 0.f ? 0x80000001u : u >> 31 ? u + 1 : u - 1);
}

// The k largest of list[0 .. n), in order, to list2[0 .. min(n, k)); threads `id` of `count`.
__device__ __forceinline__ void rank_keys(const uint64_t* list, int n, int k, uint64_t* list2, int id, int count) {
    for (int i = id; i < n; i += count) {
        const uint64_t mine = list[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += list[j] > mine ? 1 : 0;
        if (above < k) list2[above] = mine;
    }
}

template <typename T>
struct Vec;                             // 16 bytes of logits
template <>
struct Vec<float> {
    static constexpr int N = 4;
    __device__ __forceinline__ static void get(const Vec16& v, float* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __builtin_bit_cast(float, v.w[i]);
    }
};
template <typename T>
struct Vec {
    static constexpr int N = 8;
    __device__ __forceinline__ static void get(const Vec16& v, float* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = Pair<T>::lo(v.w[i]);
            x[2 * i + 1] = Pair<T>::hi(v.w[i]);
        }
    }
};

// U: 16-byte loads of a lane and tile.
template <typename T, int U>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4))) void token_logprobs_kernel(const LogprobArgs a) {
    constexpr int N = Vec<T>::N;
    __shared__ uint64_t s_list[kWaves][kList];
    __shared__ uint64_t s_merged[kMerged], s_top[kMaxTop];
    __shared__ float s_max[kWaves][64];
    __shared__ Stat s_stat[kWaves];
    __shared__ int s_above[kWaves], s_far[kWaves], s_n, s_entries[64];
    __shared__ uint32_t s_arrived;
    const int tid = (int)threadIdx.x, lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = blockIdx.x / (unsigned)a.parts;
    const int part = (int)(blockIdx.x % (unsigned)a.parts);
    const T* x0 = reinterpret_cast<const T*>(a.logits) + row * a.stride;
    const int64_t id = a.ids ? a.ids[row] : -1;
    const bool asked = (uint64_t)id < (uint64_t)a.vocab;
    const float own = to_f32(x0[asked ? id : 0]);
    const float limit = asked ? own : __builtin_huge_valf();     // ranks count what is above it

    // The row in 16-byte pieces from the 16-byte boundary at or below its start; `head` elements of
    // the first one are not the row's.
    const int head = (int)(((uintptr_t)x0 & 15) / sizeof(T));
    const T* base = x0 - head;
    const int pieces = (head + a.vocab + N - 1) / N;
    const int per_part = ((pieces + a.parts - 1) / a.parts + 63) & ~63;
    const int q_begin = part * per_part < pieces ? part * per_part : pieces;
    const int q_end = pieces - q_begin < per_part ? pieces : q_begin + per_part;

    Stat st = {kNegInf, 0.f, 0.f};
    float ref = 0.f;                    // st.c where it is above -inf
    bool far = false;                   // a logit above 2^29
    int above = 0;                      // of the wave
    // The wave's list of the likeliest, their bound, how many equal to it are listed, what a tile has to
    // exceed to be looked at, the lane's largest logit.
    uint64_t* list = s_list[wave];
    int listed = 0, equal = 0;
    float tau = kNegInf, limit_top = a.top > 0 ? kNegInf : __builtin_huge_valf(), lane_max = kNegInf;
    s_max[wave][lane] = kNegInf;
    if (a.top > 0) __syncthreads();

    auto load = [&](int q0, Vec16* raw) {
        // q0: the wave's first piece.
        const int q = q0 + lane;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (q + 64 * u < q_end && q + 64 * u > 0 && q + 64 * u < pieces - 1)
                raw[u] = load16_stream(base + (int64_t)(q + 64 * u) * N);
    };
    auto values = [&](int q0, int u, const Vec16& raw, float* x) {
        const int q = q0 + lane + 64 * u;
        if (q > 0 && q < pieces - 1 && q < q_end) {
            Vec<T>::get(raw, x);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int i = q * N + e - head;
                x[e] = q < q_end && i >= 0 && i < a.vocab ? to_f32(x0[i]) : kNegInf;
            }
        }
    };
    // Drops what is below tau from the list; if that leaves too much for `more`, all but the k largest.
    auto shorten = [&](int more) {
        int kept = 0;
        const uint32_t least = order_of(tau);
        for (int i = 0; i < listed; i += 64) {
            const uint64_t key = i + lane < listed ? list[i + lane] : 0;
            const uint64_t keep = __builtin_amdgcn_ballot_w64(i + lane < listed && (uint32_t)(key >> 32) >= least);
            wave_lds_sync();
            if (keep >> lane & 1) list[kept + lanes_below(keep)] = key;
            wave_lds_sync();
            kept += __builtin_popcountll(keep);
        }
        listed = kept;
        if (listed + more <= kList) return;
        // Ranks first, then the moves: lists of 64 entries a round.
        uint64_t mine[kList / 64];
        int rank[kList / 64];
#pragma unroll
        for (int r = 0; r < kList / 64; ++r) {
            mine[r] = 64 * r + lane < listed ? list[64 * r + lane] : 0;
            rank[r] = 0;
        }
        for (int j = 0; j < listed; ++j) {
            const uint64_t key = list[j];
#pragma unroll
            for (int r = 0; r < kList / 64; ++r) rank[r] += key > mine[r] ? 1 : 0;
        }
        wave_lds_sync();
#pragma unroll
        for (int r = 0; r < kList / 64; ++r)
            if (64 * r + lane < listed && rank[r] < a.top) list[rank[r]] = mine[r];
        wave_lds_sync();
        listed = listed < a.top ? listed : a.top;
    };

    constexpr int kTile = kWaves * 64 * U;
    Vec16 raw[U];
    const int q_first = q_begin + wave * 64 * U;
    if (q_first < q_end) load(q_first, raw);
    for (int q0 = q_first; q0 < q_end; q0 += kTile) {
        float x[U][N], um[U], tm = kNegInf;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            values(q0, u, raw[u], x[u]);
            um[u] = x[u][0];
#pragma unroll
            for (int e = 1; e < N; ++e) um[u] = fmaxf(um[u], x[u][e]);
            tm = fmaxf(tm, um[u]);
        }
        if (q0 + kTile < q_end) load(q0 + kTile, raw);
        const float ym = tm * kLog2e;
        if (__builtin_amdgcn_ballot_w64(ym > st.c + kRaise)) {
            far |= ym > kFar;
            if (ym > st.c + kRaise && ym > -kFar) {
                const float c = rintf(ym), d = fmaxf(st.c - c, kLeast), f = fast_exp2(d);
                st = Stat{c, st.s * f, fmaf(d, st.s, st.t) * f};
                ref = c;
            }
        }
        float s = 0.f, t = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float d = fmaf(x[u][e], kLog2e, -ref);
                const float w = fast_exp2(d);               // NaN stays NaN; -inf: 0
                s += w;
                t = fmaf(w, fmaxf(d, kLeast), t);           // 0 * kLeast, not 0 * -inf
            }
        st.s += s;
        st.t += t;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (__builtin_amdgcn_ballot_w64(um[u] > limit)) {
#pragma unroll
                for (int e = 0; e < N; ++e) above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(x[u][e] > limit));
            }
        if (__builtin_amdgcn_ballot_w64(tm > limit_top)) {
            lane_max = fmaxf(lane_max, tm);
            // What the other waves have found by now: any of it bounds the row's k-th.
            float both = lane_max;
            __hip_atomic_store(&s_max[wave][lane], lane_max, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
#pragma unroll
            for (int w = 0; w < kWaves; ++w)
                both = fmaxf(both, __hip_atomic_load(&s_max[w][lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
            const float raised = kth_of_lanes(both, a.top);
            if (raised > tau) {
                tau = raised;
                equal = 0;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool more_equal = equal < a.top;
                auto takes = [&](float v) { return v > tau || (more_equal && v == tau && v > kNegInf); };
                if (!__builtin_amdgcn_ballot_w64(takes(um[u]))) continue;
                int more = 0;
#pragma unroll
                for (int e = 0; e < N; ++e) more += __builtin_popcountll(__builtin_amdgcn_ballot_w64(takes(x[u][e])));
                if (listed + more > kList) shorten(more);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const uint64_t lanes = __builtin_amdgcn_ballot_w64(takes(x[u][e]));
                    if (takes(x[u][e]))
                        list[listed + lanes_below(lanes)] = key_of(x[u][e], (q0 + lane + 64 * u) * N + e - head);
                    listed += __builtin_popcountll(lanes);
                    equal += __builtin_popcountll(__builtin_amdgcn_ballot_w64(x[u][e] == tau));
                }
            }
            limit_top = equal < a.top ? below(tau) : tau;
        }
    }

    // ---- the workgroup's.
    st = wave_merge<true>(st);
    const bool any_far = __builtin_amdgcn_ballot_w64(far) != 0;
    if (lane == 0) {
        s_stat[wave] = st;
        s_above[wave] = above;
        s_far[wave] = any_far;
    }
    if (tid == 0) s_n = 0;
    s_max[wave][lane] = lane_max;
    __syncthreads();
    Stat all = s_stat[0];
    int more = s_above[0], level = s_far[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
        all = merge<true>(all, s_stat[w]);
        more += s_above[w];
        level |= s_far[w];
    }
    level = level ? kBeyond : all.s > 0.f ? kNear : all.s == 0.f ? kBelow : kNone;
    if (level == kBeyond || level == kBelow) {
        // Once more, against the piece's largest logit.
        float m = kNegInf;
        auto each = [&](auto f) {
            for (int q = q_begin + tid; q < q_end; q += 256)
                for (int e = 0; e < N; ++e) {
                    const int i = q * N + e - head;
                    if (i >= 0 && i < a.vocab) f(to_f32(x0[i]));
                }
        };
        each([&](float v) { m = fmaxf(m, v); });
        m = wave_max(m);
        __syncthreads();                               // s_stat has been read
        if (lane == 0) s_stat[wave].c = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, s_stat[w].c);
        Stat x = {m, 0.f, 0.f};
        if (m > kNegInf)
            each([&](float v) {
                const float d = v - m, w = fast_exp2(d * kLog2e);
                x.s += w;
                x.t = fmaf(w, fmaxf(d, kLeast), x.t);
            });
        x = wave_merge<false>(x);
        __syncthreads();
        if (lane == 0) s_stat[wave] = x;
        __syncthreads();
        all = s_stat[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) all = merge<false>(all, s_stat[w]);
        if (all.s != all.s) level = kNone;
    }
    int n = 0;
    // The lists, cut by the row's bound, into one.
    if (a.top > 0) {
        float both = s_max[0][lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) both = fmaxf(both, s_max[w][lane]);
        tau = fmaxf(tau, kth_of_lanes(both, a.top));
        shorten(kList - kMerged / kWaves);          // a wave's share of s_merged at most
        wave_lds_sync();
        int at = 0;
        if (lane == 0) at = atomicAdd(&s_n, listed);
        at = __builtin_amdgcn_readfirstlane(at);
        for (int i = lane; i < listed; i += 64) s_merged[at + i] = list[i];
        __syncthreads();
        n = s_n;
        rank_keys(s_merged, n, a.top, s_top, tid, 256);
        n = n < a.top ? n : a.top;
        __syncthreads();
    }
    if (a.parts > 1) {
        // Out to where every XCD sees it; the stores have arrived there before the count moves.
        const int words = 3 + a.top;
        uint64_t* mine = a.partials + (row * a.parts + part) * words;
        auto put = [&](int i, uint64_t v) { __hip_atomic_store(mine + i, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
        auto two = [](float lo, uint32_t hi) { return (uint64_t)hi << 32 | __builtin_bit_cast(uint32_t, lo); };
        if (tid == 0) {
            put(0, two(all.c, __builtin_bit_cast(uint32_t, all.s)));
            put(1, two(all.t, (uint32_t)more));
            put(2, (uint64_t)n | (uint64_t)level << 32);
        }
        if (tid < n) put(3 + tid, s_top[tid]);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) s_arrived = __hip_atomic_fetch_add(a.counters + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (s_arrived != (uint32_t)a.parts - 1) return;
        if (tid == 0) __hip_atomic_store(a.counters + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        auto get = [&](int p, int i) {
            return __hip_atomic_load(a.partials + (row * a.parts + p) * words + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        };
        // Parts in a fixed order: lane p of every wave has part p, merged across the wave. Those of the highest
        // level are the row's; the others are nothing beside them.
        Stat x = {kNegInf, 0.f, 0.f};
        int count = 0, its = 0;
        uint64_t entries = 0;
        if (lane < a.parts) {
            const uint64_t ms = get(lane, 0), tn = get(lane, 1);
            entries = get(lane, 2);
            its = (int)(entries >> 32);
            x = Stat{__builtin_bit_cast(float, (uint32_t)ms), __builtin_bit_cast(float, (uint32_t)(ms >> 32)),
                     __builtin_bit_cast(float, (uint32_t)tn)};
            count = (int)(tn >> 32);
        }
        level = kBelow;
        for (int l = kNear; l <= kNone; ++l)
            if (__builtin_amdgcn_ballot_w64(its == l)) level = l;
        if (its != level) x = Stat{kNegInf, 0.f, 0.f};
        all = level == kNear ? wave_merge<true>(x) : wave_merge<false>(x);
        for (int off = 1; off < 64; off *= 2) count += __shfl_xor(count, off);
        more = count;
        if (a.top > 0) {
            if (tid == 0) s_n = 0;
            if (tid < 64) s_entries[tid] = (int)entries;
            __syncthreads();
            uint64_t* joined = &s_list[0][0];      // parts * top <= 32 * 64 of kWaves * kList
            // A part's list holds its k largest, in order. The largest last entry of a full list bounds
            // the row's k-th from below.
            uint64_t least = lane < a.parts && (int)(uint32_t)entries == a.top ? get(lane, 2 + a.top) : 0;
            for (int off = 1; off < 64; off *= 2) {
                const uint64_t o = __shfl_xor((unsigned long long)least, off);
                least = o > least ? o : least;
            }
            for (int i = tid; i < a.parts * a.top; i += 256) {
                const int p = i / a.top, e = i - p * a.top;
                const uint64_t key = get(p, 3 + e);
                if (e < s_entries[p] && key >= least) joined[atomicAdd(&s_n, 1)] = key;
            }
            __syncthreads();
            n = s_n;
            rank_keys(joined, n, a.top, s_top, tid, 256);
            n = n < a.top ? n : a.top;
            __syncthreads();
        }
    }

    // ---- out. A row whose sum is NaN, or 0, has no distribution.
    const bool proper = all.s > 0.f && level != kNone;
    const bool near = level == kNear;
    const float nan = __builtin_nanf("");
    const float log_s = near ? log2f(all.s) : logf(all.s);
    auto log_p = [&](float v) {
        if (!near) return v - all.c - log_s;
        // (The product overflows at the type's lowest value.)
        return v < -kFar ? v - kLn2 * (all.c + log_s) : kLn2 * (fmaf(v, kLog2e, -all.c) - log_s);
    };
    if (tid == 0) {
        a.logprobs[row] = proper && asked ? log_p(own) : nan;
        a.ranks[row] = proper && asked ? more + 1 : 0;
        const float h = log_s - all.t / all.s;
        a.entropy[row] = proper ? fmaxf(near ? kLn2 * h : h, 0.f) : nan;
    }
    float* out = a.top_logprobs + row * a.top;
    int64_t* out_ids = a.top_ids + row * a.top;
    if (tid < a.top && (tid < n || !proper)) {
        out[tid] = proper ? log_p(logit_of(s_top[tid])) : nan;
        out_ids[tid] = proper ? id_of(s_top[tid]) : -1;
    }
    if (proper && n < a.top && tid == 0) {
        // The rest of the row is -inf: its lowest ids.
        int next = 0;
        for (int i = n; i < a.top; ++i, ++next) {
            for (bool again = true; again;) {
                again = false;
                for (int j = 0; j < n; ++j)
                    if (id_of(s_top[j]) == next) {
                        again = true;
                        ++next;
                    }
            }
            out[i] = kNegInf;
            out_ids[i] = next;
        }
    }
}

// Pieces of a row, none shorter than a load of every lane.
int parts_of(int64_t rows, int64_t vocab, int itemsize) {
    const int64_t longest = ceil_div(vocab * itemsize, 16 * 256);
    int64_t parts = rows > 0 ? 512 / rows : 1;
    parts = parts < longest ? parts : longest;
    return (int)(parts < 1 ? 1 : parts > 32 ? 32 : parts);
}

template <typename T>
int launch_t(const LogprobArgs& a, int64_t rows, hipStream_t stream) {
    const dim3 grid((unsigned)(rows * a.parts));
    const int64_t per = ceil_div(ceil_div((int64_t)a.vocab * sizeof(T), 16), a.parts);
    if (per <= 512) token_logprobs_kernel<T, 1><<<grid, 256, 0, stream>>>(a);
    else token_logprobs_kernel<T, 4><<<grid, 256, 0, stream>>>(a);
    return check_launch("token_logprobs");
}

}  // namespace
}  // namespace pkv

using namespace pkv;

static int itemsize_of(int dtype) { return dtype == PKV_FLOAT32 ? 4 : 2; }

extern "C" int64_t pkv_token_logprobs_workspace_bytes(int64_t num_rows, int64_t vocab_size, int64_t top, int dtype) {
    if (num_rows <= 0 || vocab_size <= 0 || top < 0 || top > kMaxTop) return 0;
    const int parts = parts_of(num_rows, vocab_size, itemsize_of(dtype));
    return parts == 1 ? 0 : kMergeCounterBytes + num_rows * parts * (3 + top) * 8;
}

extern "C" int pkv_token_logprobs(const void* logits, int64_t logits_stride, int64_t num_rows, int64_t vocab_size,
                                  int dtype, const int64_t* ids, int64_t top, float* logprobs, int64_t* ranks,
                                  float* entropy, float* top_logprobs, int64_t* top_ids, void* workspace,
                                  int64_t workspace_bytes, hipStream_t stream) {
    clear_error();
    if (dtype != PKV_FLOAT32 && dtype != PKV_FLOAT16 && dtype != PKV_BFLOAT16)
        return fail(PKV_EINVAL, "token_logprobs: unknown dtype %d", dtype);
    if (num_rows < 0 || vocab_size < 1 || top < 0) return fail(PKV_EINVAL, "token_logprobs: bad sizes");
    if (top > vocab_size) return fail(PKV_EINVAL, "token_logprobs: top %lld of %lld logits", (long long)top, (long long)vocab_size);
    if (num_rows > 0x3fffffff || vocab_size > 0x3fffffff || top > kMaxTop)
        return fail(PKV_EUNSUPPORTED, "token_logprobs: top above %d, or sizes beyond int32", kMaxTop);
    if (num_rows == 0) return PKV_OK;
    if (!logits || !ids || !logprobs || !ranks || !entropy || (top > 0 && (!top_logprobs || !top_ids)))
        return fail(PKV_EINVAL, "token_logprobs: null pointer");
    LogprobArgs a = {};
    a.logits = logits;
    a.stride = logits_stride;
    a.vocab = (int)vocab_size;
    a.top = (int)top;
    a.ids = ids;
    a.logprobs = logprobs;
    a.ranks = ranks;
    a.entropy = entropy;
    a.top_logprobs = top_logprobs;
    a.top_ids = top_ids;
    a.parts = parts_of(num_rows, vocab_size, itemsize_of(dtype));
    if (a.parts > 1) {
        const int64_t need = pkv_token_logprobs_workspace_bytes(num_rows, vocab_size, top, dtype);
        if (!workspace || workspace_bytes < need)
            return fail(PKV_EWORKSPACE, "token_logprobs: workspace of %lld bytes, need %lld",
                        (long long)(workspace ? workspace_bytes : 0), (long long)need);
        a.counters = reinterpret_cast<uint32_t*>(workspace);
        a.partials = reinterpret_cast<uint64_t*>(reinterpret_cast<char*>(workspace) + kMergeCounterBytes);
    }
    switch (dtype) {
        case PKV_FLOAT32: return launch_t<float>(a, num_rows, stream);
        case PKV_FLOAT16: return launch_t<_Float16>(a, num_rows, stream);
        default: return launch_t<bf16_t>(a, num_rows, stream);
    }
}
