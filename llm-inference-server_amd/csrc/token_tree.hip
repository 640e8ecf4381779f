// Drafted token trees: what each node sees and where it stands, and the path that the target
// model accepts.
//
// A sequence's nodes are its rows query_start_loc[i] .. query_start_loc[i + 1] of the packed step, in
// an order in which parents come first; `parents` holds a node's parent as its number in the
// sequence, -1 for a root.
//
//  * Layout. seen(i) = seen(parent(i)) + {i}, depth(i) = depth(parent(i)) + 1. A workgroup has one
//    sequence and its parents in LDS; a thread walks from its node to the root. The numbers fall
//    along the walk (a parent that is not below its child ends it: impossible), so that the mask
//    words are finished one by one, from the last to the first, in a register.
//  * Accept. Node c fits if its token is the target's token at its parent; of a node's children that
//    fit, the first goes on. All nodes find that out side by side (an LDS minimum at the parent),
//    then one thread follows the links.
//
// Both are bound by latency: launch, the sequence's bounds, one load of each input. 8 sequences of 8-32 nodes
// take 2.8 (layout) and 2.9 us (walk), 256 of 16-256 nodes 3.6 both, calls back to back in a graph.
#include "pkv_common.h"

namespace pkv {
namespace {

constexpr int kMaxNodes = 8192;         // of a sequence: links of 4 bytes in LDS
constexpr int kStaged = 2048;           // nodes whose targets are in LDS too

struct Nodes {
    int64_t first;
    int count;                          // 0 where the bounds are impossible
};

// Rows of sequence i; bounds that do not fit the step have no nodes.
__device__ __forceinline__ Nodes nodes_of(const int64_t* starts, int i, int64_t num_tokens, int64_t most) {
    const int64_t a = starts[i], b = starts[i + 1];
    if (a < 0 || b < a || b > num_tokens || b - a > most) return Nodes{0, 0};
    return Nodes{a, (int)(b - a)};
}

__global__ __launch_bounds__(256) void tree_layout_kernel(const int64_t* __restrict__ parents,
                                                          const int64_t* __restrict__ starts,
                                                          const int64_t* __restrict__ ctx, int num_seqs,
                                                          int64_t num_tokens, int max_nodes, int words,
                                                          uint64_t* __restrict__ masks,
                                                          int64_t* __restrict__ positions) {
    extern __shared__ int s_up[];
    const int tid = (int)threadIdx.x, n_threads = (int)blockDim.x;
    auto none = [&](int64_t row) {
        for (int w = 0; w < words; ++w) masks[row * words + w] = 0;
        positions[row] = 0;
    };
    if ((int)blockIdx.x >= num_seqs) {
        // Rows of no sequence: before the first one and past the last.
        auto in_step = [&](int64_t r) { return r < 0 ? 0 : r < num_tokens ? r : num_tokens; };
        const int64_t before = num_seqs > 0 ? in_step(starts[0]) : 0, from = num_seqs > 0 ? in_step(starts[num_seqs]) : 0;
        const int64_t step = (int64_t)(gridDim.x - num_seqs) * n_threads;
        for (int64_t i = (int64_t)(blockIdx.x - num_seqs) * n_threads + tid; i < before + num_tokens - from; i += step)
            none(i < before ? i : from + i - before);
        return;
    }
    const int seq = (int)blockIdx.x;
    const Nodes at = nodes_of(starts, seq, num_tokens, num_tokens);
    if (at.count == 0) {
        // (Bounds outside the step: what of its rows are inside.)
        const int64_t a = starts[seq], b = starts[seq + 1];
        for (int64_t r = (a < 0 ? 0 : a) + tid; r < (b < num_tokens ? b : num_tokens); r += n_threads) none(r);
        return;
    }
    const int64_t cached = ctx[seq] - at.count;
    if (at.count > max_nodes || cached < 0) {
        for (int i = tid; i < at.count; i += n_threads) none(at.first + i);
        return;
    }
    for (int i = tid; i < at.count; i += n_threads) {
        const int64_t p = parents[at.first + i];
        s_up[i] = p >= -1 && p < i ? (int)p : -2;
    }
    __syncthreads();
    for (int i = tid; i < at.count; i += n_threads) {
        const int64_t row = at.first + i;
        uint64_t* out = masks + row * words;
        for (int w = words - 1; w > i >> 6; --w) out[w] = 0;
        int j = i, word = i >> 6, depth = -1;
        uint64_t bits = 0;
        while (j >= 0) {
            for (; word > j >> 6; --word) {
                out[word] = bits;
                bits = 0;
            }
            bits |= 1ull << (j & 63);
            ++depth;
            j = s_up[j];
        }
        if (j == -2) {                  // an impossible parent on the way
            none(row);
            continue;
        }
        for (; word >= 0; --word) {
            out[word] = bits;
            bits = 0;
        }
        positions[row] = cached + depth;
    }
}

__global__ __launch_bounds__(256) void tree_accept_kernel(const int64_t* __restrict__ tokens,
                                                          const int64_t* __restrict__ parents,
                                                          const int64_t* __restrict__ targets,
                                                          const int64_t* __restrict__ starts, int64_t num_tokens,
                                                          int64_t max_depth, int64_t* __restrict__ paths,
                                                          int64_t* __restrict__ counts,
                                                          int64_t* __restrict__ next_tokens) {
    __shared__ int s_next[kMaxNodes];   // of a node: its first child that fits
    __shared__ int64_t s_target[kStaged];
    const int tid = (int)threadIdx.x, seq = (int)blockIdx.x;
    const Nodes at = nodes_of(starts, seq, num_tokens, kMaxNodes);
    const int n = at.count;
    int64_t* path = paths + seq * max_depth;
    const bool staged = n <= kStaged;
    for (int i = tid; i < n; i += 256) {
        s_next[i] = 0x7fffffff;
        if (staged) s_target[i] = targets[at.first + i];
    }
    __syncthreads();
    for (int i = tid; i < n; i += 256) {
        const int64_t p = parents[at.first + i], token = tokens[at.first + i];
        if (p >= 0 && p < i && token == (staged ? s_target[p] : targets[at.first + p])) atomicMin(&s_next[p], i);
    }
    __syncthreads();
    if (tid < 64) {
        // Every lane walks; lane d stores node d.
        int node = n > 0 ? 0 : -1, last = -1;
        int64_t kept = 0;
        for (int64_t d = 0; d < max_depth; d += 64) {
            int mine = -1;
            for (int e = 0; e < 64 && d + e < max_depth && node >= 0; ++e) {
                if (e == tid) mine = node;
                last = node;
                ++kept;
                const int next = s_next[node];
                node = next < n ? next : -1;
            }
            if (d + tid < max_depth) path[d + tid] = mine;
        }
        if (tid == 0) {
            counts[seq] = kept;
            next_tokens[seq] = last >= 0 ? targets[at.first + last] : -1;
        }
    }
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int pkv_tree_layout(const int64_t* parents, const int64_t* query_start_loc, const int64_t* context_lens,
                               int64_t num_seqs, int64_t num_tokens, int64_t max_nodes, int64_t* masks,
                               int64_t* positions, hipStream_t stream) {
    clear_error();
    if (num_seqs < 0 || num_tokens < 0 || max_nodes < 0) return fail(PKV_EINVAL, "tree_layout: bad sizes");
    if (num_seqs > 0x3fffffff || num_tokens > 0x7fffffff || max_nodes > kMaxNodes)
        return fail(PKV_EUNSUPPORTED, "tree_layout: more than %d nodes a sequence, or sizes beyond int32", kMaxNodes);
    if (num_tokens == 0) return PKV_OK;
    if (!parents || (!masks && max_nodes > 0) || !positions || !query_start_loc || (num_seqs > 0 && !context_lens))
        return fail(PKV_EINVAL, "tree_layout: null pointer");
    const int words = (int)ceil_div(max_nodes, 64);
    const int threads = max_nodes <= 64 ? 64 : 256;
    // Behind the sequences' workgroups, those of the rows past them.
    const int64_t more = ceil_div(num_tokens, threads);
    const dim3 grid((unsigned)(num_seqs + (more < 16 ? more : 16)));
    tree_layout_kernel<<<grid, threads, max_nodes * sizeof(int), stream>>>(
        parents, query_start_loc, context_lens, (int)num_seqs, num_tokens, (int)max_nodes, words,
        reinterpret_cast<uint64_t*>(masks), positions);
    return check_launch("tree_layout");
}

extern "C" int pkv_tree_accept(const int64_t* tokens, const int64_t* parents, const int64_t* targets,
                               const int64_t* query_start_loc, int64_t num_seqs, int64_t num_tokens, int64_t max_depth,
                               int64_t* paths, int64_t* counts, int64_t* next_tokens, hipStream_t stream) {
    clear_error();
    if (num_seqs < 0 || num_tokens < 0 || max_depth < 1) return fail(PKV_EINVAL, "tree_accept: bad sizes");
    if (num_seqs > 0x7fffffff || num_tokens > 0x7fffffff || max_depth > kMaxNodes)
        return fail(PKV_EUNSUPPORTED, "tree_accept: paths of more than %d nodes, or sizes beyond int32", kMaxNodes);
    if (num_seqs == 0) return PKV_OK;
    if (!query_start_loc || !paths || !counts || !next_tokens || (num_tokens > 0 && (!tokens || !parents || !targets)))
        return fail(PKV_EINVAL, "tree_accept: null pointer");
    tree_accept_kernel<<<dim3((unsigned)num_seqs), 256, 0, stream>>>(tokens, parents, targets, query_start_loc,
                                                                     num_tokens, max_depth, paths, counts, next_tokens);
    return check_launch("tree_accept");
}
