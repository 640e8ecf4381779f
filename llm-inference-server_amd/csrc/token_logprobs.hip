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
// Top: of a tile, lanes keep only whether it holds their largest logit so far, and the second largest of
// their tiles' largest. The k-th largest of the 256 lanes' largest logits, found by ballots on their bits, is a lower bound tau
// of the row's k-th largest. Lanes that reach it, hardly more than k, read that one tile's logits again (64 bytes of 16-bit
// ones; all their tiles where the second reaches tau too) and list what reaches tau. The entries, hardly more
// than k, rank themselves by counting. A wave with more to list than there is room for (rows of many equal logits)
// walks all its tiles again instead, in the order of the ids, and takes of logits equal to tau only the first k.
// Masked logits (-inf) never enter a list; if a row has fewer others than k, the lowest masked ids follow.
// (Lists grown while the logits stream by, against a bound that rises, cost 66 of 192 us of 2048 rows of 128000
// at k = 20.)
//
// Bound: HBM and, for 16-bit logits, the vector unit (an exponential takes four slots of the nine that a logit
// costs).
#include "pkv_common.h"

#include "attention.h"

namespace pkv {
namespace {

constexpr int kWaves = 4;
constexpr int kMaxTop = 64;             // a list's entries are ranked against one another; one lane max each
constexpr int kList = 640;              // of a wave: kMaxTop after a cut, and a load of 512 logits
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

// A lower bound of the k-th largest of the lanes' W values x (k <= 64), itself one of them.
template <int W>
__device__ __forceinline__ float kth_of_lanes(const float* x, int k) {
    uint32_t u[W], t = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) u[w] = order_of(x[w]);
    for (uint32_t bit = 0x80000000u; bit > 0x8000u; bit >>= 1) {
        int n = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(u[w] >= (t | bit)));
        if (n >= k) t |= bit;
        if (n == k) break;                    // the k-th itself bounds them
    }
    float least = kNegInf;
#pragma unroll
    for (int w = 0; w < W; ++w) least = fmaxf(least, u[w] >= t ? -x[w] : kNegInf);
    return -wave_max(least);
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
    __shared__ int s_at[kWaves][64];
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
    // The lane's largest logit and its tile's first piece, the second largest of its tiles' largest.
    float best = kNegInf, second = kNegInf, tau = kNegInf;
    int best_at = 0;
    uint64_t* list = s_list[wave];      // of the wave's likeliest
    int listed = 0;

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
    // Leaves the k largest of the list.
    auto shorten = [&]() {
        uint64_t mine[kList / 64];
        int rank[kList / 64];
        wave_lds_sync();
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
        second = fmaxf(second, fminf(best, tm));
        best_at = tm > best ? q0 : best_at;
        best = fmaxf(best, tm);
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
    s_max[wave][lane] = best;
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
        // Once more, against the piece's largest logit (without any: nothing).
        float m = fmaxf(fmaxf(s_max[0][lane], s_max[1][lane]), fmaxf(s_max[2][lane], s_max[3][lane]));
        m = wave_max(m);
        Stat x = {m, 0.f, 0.f};
        for (int q = q_begin + tid; q < q_end && m > kNegInf; q += 256)
            for (int e = 0; e < N; ++e) {
                const int i = q * N + e - head;
                if (i < 0 || i >= a.vocab) continue;
                const float d = to_f32(x0[i]) - m, w = fast_exp2(d * kLog2e);
                x.s += w;
                x.t = fmaf(w, fmaxf(d, kLeast), x.t);
            }
        x = wave_merge<false>(x);
        __syncthreads();                               // s_stat has been read
        if (lane == 0) s_stat[wave] = x;
        __syncthreads();
        all = s_stat[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) all = merge<false>(all, s_stat[w]);
        if (all.s != all.s) level = kNone;
    }
    int n = 0;
    if (a.top > 0) {
        float max_of[kWaves];
#pragma unroll
        for (int w = 0; w < kWaves; ++w) max_of[w] = s_max[w][lane];
        tau = kth_of_lanes<kWaves>(max_of, a.top);
        // Of one piece a lane, of q's values or raw's, those that reach tau; false where the list has no room.
        auto inner = [&](int q, bool live) { return live && q > 0 && q < pieces - 1; };
        auto push = [&](int q, bool live, const Vec16& raw) {
            float v[N];
            if (inner(q, live)) {
                Vec<T>::get(raw, v);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const int i = q * N + e - head;
                    v[e] = live && i >= 0 && i < a.vocab ? to_f32(x0[i]) : kNegInf;
                }
            }
            int more = 0;
            auto takes = [&](int e) { return v[e] >= tau && v[e] > kNegInf; };
#pragma unroll
            for (int e = 0; e < N; ++e) more += __builtin_popcountll(__builtin_amdgcn_ballot_w64(takes(e)));
            if (listed + more > kList) return false;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const uint64_t lanes = __builtin_amdgcn_ballot_w64(takes(e));
                if (takes(e)) list[listed + lanes_below(lanes)] = key_of(v[e], q * N + e - head);
                listed += __builtin_popcountll(lanes);
            }
            return true;
        };
        const uint64_t wide = __builtin_amdgcn_ballot_w64(second >= tau && second > kNegInf);
        const uint64_t narrow = __builtin_amdgcn_ballot_w64(best >= tau && best > kNegInf) & ~wide;
        const int n_wide = __builtin_popcountll(wide), n_narrow = __builtin_popcountll(narrow);
        const int tiles = q_first < q_end ? (q_end - q_first + kTile - 1) / kTile : 0;
        bool fits = true;
        if (narrow >> lane & 1) s_at[wave][lanes_below(narrow)] = best_at + lane;
        if (wide >> lane & 1) s_at[wave][n_narrow + lanes_below(wide)] = q_first + lane;
        wave_lds_sync();
        // Lane's piece in round r: first one tile of each narrow lane, U pieces of it side by side, then all tiles
        // of each wide one, 64 pieces a round. Rounds load kAhead at a time.
        constexpr int kAhead = 4;
        const int first_wide = (n_narrow * U + 63) / 64, per_wide = (tiles * U + 63) / 64;
        const int rounds = first_wide + n_wide * per_wide;
        auto piece = [&](int r, bool& live) {
            if (r < first_wide) {
                const int mine = (64 * r + lane) / U;
                live = mine < n_narrow;
                return s_at[wave][live ? mine : 0] + 64 * (lane % U);
            }
            const int j = (r - first_wide) % per_wide * 64 + lane;
            live = j < tiles * U;
            return s_at[wave][n_narrow + (r - first_wide) / per_wide] + j / U * kTile + 64 * (j % U);
        };
        // (Of a lone tile every lane still has its piece.)
        const bool lone = U == 1 && tiles == 1;
        if (lone) fits = push(q_first + lane, q_first + lane < q_end, raw[0]);
        for (int r0 = 0; fits && !lone && r0 < rounds; r0 += kAhead) {
            Vec16 ahead[kAhead];
            int q[kAhead];
            bool live[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                live[i] = false;
                q[i] = r0 + i < rounds ? piece(r0 + i, live[i]) : 0;
                live[i] = live[i] && q[i] < q_end;
                if (inner(q[i], live[i])) ahead[i] = load16(base + (int64_t)q[i] * N);
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (fits && r0 + i < rounds) fits = push(q[i], live[i], ahead[i]);
        }
        if (!fits) {
            // Everything once more, of what equals tau the first k.
            listed = 0;
            int equal = 0;
            for (int q0 = q_first; q0 < q_end; q0 += kTile) {
                load(q0, raw);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float v[N];
                    values(q0, u, raw[u], v);
                    const bool more_equal = equal < a.top;
                    auto takes = [&](int e) { return v[e] > tau || (more_equal && v[e] == tau && v[e] > kNegInf); };
                    int more = 0;
#pragma unroll
                    for (int e = 0; e < N; ++e) more += __builtin_popcountll(__builtin_amdgcn_ballot_w64(takes(e)));
                    if (more == 0) continue;
                    if (listed + more > kList) shorten();
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const uint64_t lanes = __builtin_amdgcn_ballot_w64(takes(e));
                        if (takes(e)) list[listed + lanes_below(lanes)] = key_of(v[e], (q0 + lane + 64 * u) * N + e - head);
                        listed += __builtin_popcountll(lanes);
                        equal += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v[e] == tau));
                    }
                }
            }
        }
        // A wave's share of s_merged at most.
        if (listed > kMerged / kWaves) shorten();
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
            // A part's list holds its k largest, in order. Where the m-th entries of k / m lists reach a value, k
            // logits do: with m for half of the lists that there are, a bound that lets hardly more than twice
            // k pass.
            const int its_n = (int)(uint32_t)entries, lists = __builtin_popcountll(__builtin_amdgcn_ballot_w64(its_n > 0));
            const int half = lists > 0 ? (2 * a.top + lists - 1) / lists : 1, m = half < a.top ? half : a.top;
            const float mth = lane < a.parts && its_n >= m ? logit_of(get(lane, 2 + m)) : kNegInf;
            const float bound = kth_of_lanes<1>(&mth, (a.top + m - 1) / m);
            const uint64_t least = bound > kNegInf ? (uint64_t)order_of(bound) << 32 : 0;
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
