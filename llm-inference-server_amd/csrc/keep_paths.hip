// The accepted paths' K/V rows move behind their sequences' cached ones, in every layer of K and V in
// one launch: path node d of a sequence with c cached tokens goes from position c + path[d] to
// position c + d.
//
// In place, without a copy in between: paths ascend, so path[d] >= d, a row is read no later than
// another is written over it, and no row is written that a later node is still to be read from
// (path[e] > path[d] >= d for e > d). A thread has C columns (of 16 bytes at most) of the rows of one
// sequence, of any pool tensors, and takes the nodes in order, kBatch of each column's loads in flight and
// then their stores; threads have nothing to do with one another's bytes.
//
// Bound by latency: a workgroup finds bounds and path, then table entries, before the first row. With
// enough workgroups for the GPU a thread has four columns, so that fewer of them do (64 sequences, 64
// tensors of 2 KiB rows, 54 MB: 14.4 us, of which the rows' way is 11; one column 25).
#include "pkv_common.h"

namespace pkv {
namespace {

constexpr int kBatch = 8;

// A pool's address comes from memory: said to be a global one, or its loads would count as LDS reads too and
// wait for them.
template <typename T>
using global = __attribute__((address_space(1))) T;

struct KeepArgs {
    char* const* tensors;
    int64_t num_tensors, num_blocks, block_bytes, row_bytes;
    int block_size;
    int scales;                  // bytes a slot behind the rows of a block, at [scale][slot]
    const int64_t* tables;
    int64_t table_stride, table_width;
    const int64_t* ctx;
    const int64_t* starts;
    const int64_t* paths;
    int64_t max_depth;
    int64_t columns;             // of a row
};

template <typename U, int C>
__global__ __launch_bounds__(256) void keep_paths_kernel(const KeepArgs a) {
    // Of the nodes that move: byte offsets of their rows in a pool tensor, and of their first scale.
    __shared__ int64_t s_from[64], s_to[64], s_scale_from[64], s_scale_to[64];
    __shared__ int s_count, s_ends;
    const int seq = (int)blockIdx.y, tid = (int)threadIdx.x;
    const int64_t nodes = a.starts[seq + 1] - a.starts[seq];
    const int64_t cached = a.ctx[seq] - nodes;
    if (nodes <= 0 || cached < 0) return;
    const int64_t per_tensor = a.columns + a.scales;
    global<char>* base[C];
    int64_t column[C];                             // -1: none
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int64_t item = ((int64_t)blockIdx.x * C + c) * 256 + tid;
        const int64_t tensor = item / per_tensor;
        const bool live = tensor < a.num_tensors;
        column[c] = live ? item - tensor * per_tensor : -1;
        base[c] = (global<char>*)(live ? a.tensors[tensor] : nullptr);
    }
    const int64_t* path = a.paths + seq * a.max_depth;
    int64_t before = -1;                           // the node ahead of the 64 at hand
    for (int64_t d0 = 0; d0 < a.max_depth; d0 += 64) {
        if (tid < 64) {
            // A path ends where it no longer ascends inside the tree.
            const int64_t d = d0 + tid;
            const int64_t node = d < a.max_depth ? path[d] : -1;
            const int64_t left = tid > 0 ? path[d - 1 < a.max_depth ? d - 1 : 0] : before;
            const uint64_t ends = __builtin_amdgcn_ballot_w64(!(node > left && node < nodes));
            const int count = ends ? __builtin_ctzll(ends) : 64;
            bool moves = false;
            int64_t block_from = 0, block_to = 0;
            int off_from = 0, off_to = 0;
            if (tid < count && node != d) {
                const int64_t pf = cached + node, pt = cached + d;
                const int64_t bf = pf / a.block_size, bt = pt / a.block_size;
                if (bf < a.table_width) {
                    block_from = a.tables[seq * a.table_stride + bf];
                    block_to = a.tables[seq * a.table_stride + bt];
                    off_from = (int)(pf - bf * a.block_size);
                    off_to = (int)(pt - bt * a.block_size);
                    moves = (uint64_t)block_from < (uint64_t)a.num_blocks && (uint64_t)block_to < (uint64_t)a.num_blocks;
                }
            }
            // Those that move, side by side.
            const uint64_t all = __builtin_amdgcn_ballot_w64(moves);
            if (moves) {
                const int at = __builtin_popcountll(all & ((1ull << tid) - 1));
                const int64_t scales = a.row_bytes * a.block_size;
                s_from[at] = block_from * a.block_bytes + off_from * a.row_bytes;
                s_to[at] = block_to * a.block_bytes + off_to * a.row_bytes;
                s_scale_from[at] = block_from * a.block_bytes + scales + off_from;
                s_scale_to[at] = block_to * a.block_bytes + scales + off_to;
            }
            if (tid == 0) {
                s_count = __builtin_popcountll(all);
                s_ends = count < 64;
            }
        }
        __syncthreads();
        const int count = s_count;
        for (int d = 0; d < count; d += kBatch) {
            int64_t from[kBatch], to[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                // Past the last one: it once more, not stored.
                const int e = d + i < count ? d + i : count - 1;
                from[i] = s_from[e];
                to[i] = s_to[e];
            }
            U row[C][kBatch];
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (column[c] >= 0 && column[c] < a.columns)
#pragma unroll
                    for (int i = 0; i < kBatch; ++i)
                        row[c][i] = *reinterpret_cast<global<const U>*>(base[c] + from[i] + column[c] * sizeof(U));
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (column[c] >= 0 && column[c] < a.columns)
#pragma unroll
                    for (int i = 0; i < kBatch; ++i)
                        if (d + i < count) *reinterpret_cast<global<U>*>(base[c] + to[i] + column[c] * sizeof(U)) = row[c][i];
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (column[c] < a.columns) continue;
            const int64_t at = (column[c] - a.columns) * a.block_size;
            for (int d = 0; d < count; ++d) base[c][s_scale_to[d] + at] = base[c][s_scale_from[d] + at];
        }
        if (s_ends || d0 + 64 >= a.max_depth) return;
        before = path[d0 + 63];
        __syncthreads();
    }
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int pkv_keep_paths(void* const* tensors, int64_t num_tensors, int64_t num_blocks, int64_t block_size,
                              int64_t block_bytes, int64_t row_bytes, int64_t scales, const int64_t* block_tables,
                              int64_t table_stride, int64_t table_width, const int64_t* context_lens,
                              const int64_t* query_start_loc, int64_t num_seqs, const int64_t* paths,
                              int64_t max_depth, hipStream_t stream) {
    clear_error();
    if (num_tensors < 0 || num_blocks < 0 || block_size <= 0 || row_bytes <= 0 || scales < 0 || table_width < 0 ||
        num_seqs < 0 || max_depth < 0 || block_bytes < block_size * (row_bytes + scales))
        return fail(PKV_EINVAL, "keep_paths: bad sizes");
    if (block_size > 0x7fffffff || scales > 0x7fffffff || num_seqs > 65535)
        return fail(PKV_EUNSUPPORTED, "keep_paths: sizes beyond what the kernel indexes");
    if (num_tensors == 0 || num_seqs == 0 || max_depth == 0 || num_blocks == 0 || table_width == 0) return PKV_OK;
    if (!tensors || !block_tables || !context_lens || !query_start_loc || !paths)
        return fail(PKV_EINVAL, "keep_paths: null pointer");
    KeepArgs a = {};
    a.tensors = reinterpret_cast<char* const*>(tensors);
    a.num_tensors = num_tensors;
    a.num_blocks = num_blocks;
    a.block_bytes = block_bytes;
    a.row_bytes = row_bytes;
    a.block_size = (int)block_size;
    a.scales = (int)scales;
    a.tables = block_tables;
    a.table_stride = table_stride;
    a.table_width = table_width;
    a.ctx = context_lens;
    a.starts = query_start_loc;
    a.paths = paths;
    a.max_depth = max_depth;
    const uint64_t sizes = (uint64_t)block_bytes | (uint64_t)row_bytes;
    const int unit = sizes % 16 == 0 ? 16 : sizes % 4 == 0 ? 4 : 1;
    a.columns = row_bytes / unit;
    const int64_t items = (a.columns + scales) * num_tensors;
    const bool many = ceil_div(items, 256) * num_seqs >= 1024;
    const int64_t gx = ceil_div(items, many ? 1024 : 256);
    if (gx > 0x7fffffff) return fail(PKV_EUNSUPPORTED, "keep_paths: grid too large");
    const dim3 grid((unsigned)gx, (unsigned)num_seqs);
    auto launch = [&](auto unit_of) {
        typedef decltype(unit_of) U;
        if (many) keep_paths_kernel<U, 4><<<grid, 256, 0, stream>>>(a);
        else keep_paths_kernel<U, 1><<<grid, 256, 0, stream>>>(a);
    };
    if (unit == 16) launch(u32x4_t{});
    else if (unit == 4) launch(uint32_t{});
    else launch(uint8_t{});
    return check_launch("keep_paths");
}
