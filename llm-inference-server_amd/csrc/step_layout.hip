// Block tables and slot maps of a step, built on the GPU from request lengths: one launch.
//
// For sequence i with context c_i (its new tokens included), q_i new tokens and h_i held
// blocks: it needs ceil(c_i / bs) blocks, takes the missing ones from the free list in
// sequence order, and its token t sits at position c_i - q_i + t, in slot
// table[position / bs] * bs + position % bs. All of it is two running sums over the sequences
// (new blocks, new tokens) and gathers.
//
// Bound: latency (a decode step moves some hundred bytes): 8 sequences 3.4 us, 256 4.6, 1,024
// 6.0, the last two loads behind one another (lengths, then table entries or free blocks) and an
// empty launch 2. So there is one launch and no
// workgroup waits for another: each sums over all sequences by itself (24 bytes a sequence,
// from L2 but for the first reader) and writes its own share of the tokens and of the new
// table entries. A token in a new block reads the free list, not the table entry that some
// other workgroup writes; table entries below h_i are only read, those from h_i on only
// written. All or nothing: every workgroup reaches the same verdict from the same sums.
#include "pkv_common.h"

namespace pkv {
namespace {

struct LayoutArgs {
    int64_t* tables;
    int64_t table_stride, width;
    const int64_t* held;
    const int64_t* ctx;
    const int64_t* qlen;
    const int64_t* free_blocks;
    int64_t num_free, num_tokens;
    int num_seqs, block_size, block_shift;
    int64_t* held_out;
    int64_t* slots;
    int64_t* positions;
    int64_t* starts;
    int64_t* counts;                 // blocks taken, blocks needed, impossible lengths
};

// Inclusive running sums over the wave's lanes of values below 2^40, in 20-bit halves (DPP moves
// 32 bits).
__device__ __forceinline__ int64_t wave_scan64(int64_t v) {
    const int lo = wave_scan((int)(v & 0xfffff)), hi = wave_scan((int)(v >> 20));
    return ((int64_t)hi << 20) + lo;
}

struct Sums {
    int64_t tokens, blocks, bad;
};

// N threads: one sequence each, N sequences a pass.
template <int N>
__global__ __launch_bounds__(N) void step_layout_kernel(const LayoutArgs a) {
    constexpr int W = N / 64;
    __shared__ int64_t s_tokens[W], s_blocks[W];
    __shared__ int s_bad[W];
    __shared__ int64_t s_token0[N], s_block0[N];   // running sums before each sequence of the pass
    __shared__ int64_t s_shift[N];                 // token number -> position
    __shared__ int64_t s_held[N];
    const int tid = (int)threadIdx.x, lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    auto div = [&](int64_t x) { return a.block_shift >= 0 ? x >> a.block_shift : x / a.block_size; };

    int64_t ctx = 0, q = 0, held = 0;              // this thread's sequence of the pass
    auto load = [&](int first) {
        const int i = first + tid;
        ctx = q = held = 0;
        if (i < a.num_seqs) {
            ctx = a.ctx[i];
            q = a.qlen[i];
            held = a.held[i];
        }
        const int64_t need = ctx > 0 ? div(ctx - 1) + 1 : 0;
        const bool bad = q < 0 || q > ctx || held < 0 || held > a.width || need > a.width;
        // An impossible sequence counts for nothing else. Sums stay below 2^40: of blocks because the
        // tables hold them, of tokens because none is counted past what the step has room for.
        const int64_t most = a.num_tokens + 1;
        return Sums{bad ? 0 : q < most ? q : most, bad || need <= held ? 0 : need - held, bad ? 1 : 0};
    };
    // Sums over the threads below this one; all of them in `total`.
    auto scan = [&](const Sums& own, Sums& total) {
        Sums run{wave_scan64(own.tokens), wave_scan64(own.blocks), 0};
        const int bad = wave_scan((int)own.bad);
        __syncthreads();                           // the last pass's readers are done
        if (lane == 63) {
            s_tokens[wave] = run.tokens;
            s_blocks[wave] = run.blocks;
            s_bad[wave] = bad;
        }
        __syncthreads();
        // Every wave sums up the waves: lane w has wave w.
        const int64_t tw = lane < W ? s_tokens[lane] : 0, bw = lane < W ? s_blocks[lane] : 0;
        const int64_t ts = wave_scan64(tw), bs = wave_scan64(bw);
        total = Sums{readlane64(ts, W - 1), readlane64(bs, W - 1),
                     __builtin_amdgcn_readlane(wave_scan(lane < W ? s_bad[lane] : 0), W - 1)};
        return Sums{run.tokens - own.tokens + readlane64(ts - tw, wave), run.blocks - own.blocks + readlane64(bs - bw, wave), 0};
    };

    // The verdict, over all sequences.
    Sums own = load(0), all{0, 0, 0};
    Sums before = scan(own, all);
    const bool one_pass = a.num_seqs <= N;
    if (!one_pass) {
        Sums part = own;
        for (int first = N; first < a.num_seqs; first += N) {
            const Sums next = load(first);
            const int64_t t = part.tokens + next.tokens, most = a.num_tokens + 1;
            part = Sums{t < most ? t : most, part.blocks + next.blocks, part.bad + next.bad};
        }
        scan(part, all);
    }
    if (all.tokens > a.num_tokens) ++all.bad;
    const bool ok = all.bad == 0 && all.blocks <= a.num_free;
    if (blockIdx.x == 0 && tid == 0) {
        a.counts[0] = ok ? all.blocks : 0;
        a.counts[1] = all.blocks;
        a.counts[2] = all.bad;
        a.starts[0] = 0;
    }

    // This workgroup's tokens and new blocks.
    const int64_t wgs = gridDim.x, at = blockIdx.x;
    const int64_t per_t = (a.num_tokens + wgs - 1) / wgs, per_b = (all.blocks + wgs - 1) / wgs;
    const int64_t t0 = at * per_t, t1 = t0 + per_t < a.num_tokens ? t0 + per_t : a.num_tokens;
    const int64_t b0 = at * per_b, b1 = b0 + per_b < all.blocks ? b0 + per_b : all.blocks;
    Sums base{0, 0, 0};
    for (int first = 0; first < a.num_seqs; first += N) {
        Sums sum = all;
        if (!one_pass) {
            own = load(first);
            before = scan(own, sum);
        }
        const int n = a.num_seqs - first < N ? a.num_seqs - first : N;
        const int64_t tok = base.tokens + before.tokens, blk = base.blocks + before.blocks;
        if (tid < n && (int64_t)(first / N) % wgs == at) {
            a.held_out[first + tid] = ok ? held + own.blocks : held;
            a.starts[first + tid + 1] = ok ? tok + own.tokens : 0;
        }
        if (ok) {
            s_token0[tid] = tok;
            s_block0[tid] = blk;
            s_shift[tid] = ctx - q - tok;
            s_held[tid] = held;
            __syncthreads();
            // The last sequence of the pass whose running sum is at most x: the one that x is in
            // (sequences without any share their sum with their successor).
            auto owner = [&](const int64_t* s, int64_t x) {
                int lo = 0, hi = n;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (s[mid] <= x) lo = mid; else hi = mid;
                }
                return lo;
            };
            const int64_t te = base.tokens + sum.tokens, be = base.blocks + sum.blocks;
            for (int64_t t = (t0 > base.tokens ? t0 : base.tokens) + tid; t < (t1 < te ? t1 : te); t += N) {
                const int s = owner(s_token0, t);
                const int64_t pos = t + s_shift[s], j = div(pos), h = s_held[s];
                const int64_t id = j < h ? a.tables[(int64_t)(first + s) * a.table_stride + j]
                                         : a.free_blocks[s_block0[s] + j - h];
                a.slots[t] = id * a.block_size + (pos - j * a.block_size);
                a.positions[t] = pos;
            }
            for (int64_t e = (b0 > base.blocks ? b0 : base.blocks) + tid; e < (b1 < be ? b1 : be); e += N) {
                const int s = owner(s_block0, e);
                a.tables[(int64_t)(first + s) * a.table_stride + s_held[s] + (e - s_block0[s])] = a.free_blocks[e];
            }
        }
        base = Sums{base.tokens + sum.tokens, base.blocks + sum.blocks, 0};
    }
    // Rows of no sequence.
    const int64_t real = ok ? all.tokens : 0;
    for (int64_t t = (t0 > real ? t0 : real) + tid; t < t1; t += N) {
        a.slots[t] = -1;
        a.positions[t] = 0;
    }
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int pkv_step_layout(int64_t* block_tables, int64_t table_stride, int64_t table_width, const int64_t* held,
                               const int64_t* context_lens, const int64_t* query_lens, int64_t num_seqs,
                               const int64_t* free_blocks, int64_t num_free, int64_t block_size, int64_t num_tokens,
                               int64_t* held_out, int64_t* slots, int64_t* positions, int64_t* query_start_loc,
                               int64_t* counts, hipStream_t stream) {
    clear_error();
    if (num_seqs < 0 || num_tokens < 0 || num_free < 0 || table_width < 0 || block_size <= 0)
        return fail(PKV_EINVAL, "step_layout: bad sizes");
    if (num_seqs > 0x7fffffff - 1024 || num_tokens > 0x7fffffff || block_size > 0x7fffffff || table_width > 0x7fffffff)
        return fail(PKV_EUNSUPPORTED, "step_layout: sizes beyond int32");
    if (num_seqs > 1 && table_stride < table_width)
        return fail(PKV_EINVAL, "step_layout: rows of %lld blocks overlap at a stride of %lld", (long long)table_width,
                    (long long)table_stride);
    if (!query_start_loc || !counts ||
        (num_seqs > 0 && (!held || !context_lens || !query_lens || !held_out || (!block_tables && table_width > 0))) ||
        (num_tokens > 0 && (!slots || !positions)) || (num_free > 0 && !free_blocks))
        return fail(PKV_EINVAL, "step_layout: null pointer");
    LayoutArgs a = {};
    a.tables = block_tables;
    a.table_stride = table_stride;
    a.width = table_width;
    a.held = held;
    a.ctx = context_lens;
    a.qlen = query_lens;
    a.free_blocks = free_blocks;
    a.num_free = num_free;
    a.num_tokens = num_tokens;
    a.num_seqs = (int)num_seqs;
    a.block_size = (int)block_size;
    a.block_shift = block_size & (block_size - 1) ? -1 : 63 - __builtin_clzll((unsigned long long)block_size);
    a.held_out = held_out;
    a.slots = slots;
    a.positions = positions;
    a.starts = query_start_loc;
    a.counts = counts;
    const int threads = num_seqs <= 256 ? 256 : 1024;
    int64_t wgs = ceil_div(num_tokens > num_seqs ? num_tokens : num_seqs, threads);
    wgs = wgs < 1 ? 1 : wgs < 512 ? wgs : 512;
    if (threads == 256) step_layout_kernel<256><<<dim3((unsigned)wgs), 256, 0, stream>>>(a);
    else step_layout_kernel<1024><<<dim3((unsigned)wgs), 1024, 0, stream>>>(a);
    return check_launch("step_layout");
}
