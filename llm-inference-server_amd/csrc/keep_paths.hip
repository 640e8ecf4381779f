// The accepted paths' K/V rows move behind their sequences' cached ones, in every layer of K and V in
// one launch: path node d of a sequence with c cached tokens goes from position c + path[d] to
// position c + d.
//
// In place, without a copy in between: paths ascend, so path[d] >= d, a row is read no later than
// another is written over it, and no row is written that a later node is still to be read from
// (path[e] > path[d] >= d for e > d). A thread has one column (16 bytes at most) of the rows of one
// (sequence, pool tensor) and takes the nodes in order, kBatch loads in flight and then their stores;
// threads have nothing to do with one another's bytes.
//
// Bound by latency (bounds and path, then table entries, then rows) up to a full batch of a deep
// model, by HBM behind that.
#include "pkv_common.h"

namespace pkv {
namespace {

constexpr int kBatch = 8;

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

template <typename U>
__global__ __launch_bounds__(256) void keep_paths_kernel(const KeepArgs a) {
    __shared__ int64_t s_from[64], s_to[64];       // byte offsets in a pool tensor; -1: stays
    __shared__ int s_off[64][2];                   // slots inside their blocks
    __shared__ int s_count;
    const int seq = (int)blockIdx.y, tid = (int)threadIdx.x;
    const int64_t nodes = a.starts[seq + 1] - a.starts[seq];
    const int64_t cached = a.ctx[seq] - nodes;
    if (nodes <= 0 || cached < 0) return;
    const int64_t per_tensor = a.columns + a.scales;
    const int64_t item = (int64_t)blockIdx.x * 256 + tid;
    const bool live = item < per_tensor * a.num_tensors;
    const int64_t tensor = live ? item / per_tensor : 0;
    const int64_t column = item - tensor * per_tensor;
    char* base = live ? a.tensors[tensor] : nullptr;
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
            if (tid == 0) s_count = count;
            int64_t from = -1, to = -1;
            if (tid < count && node != d) {
                const int64_t pf = cached + node, pt = cached + d;
                const int64_t bf = pf / a.block_size, bt = pt / a.block_size;
                if (bf < a.table_width) {
                    const int64_t idf = a.tables[seq * a.table_stride + bf], idt = a.tables[seq * a.table_stride + bt];
                    const int of = (int)(pf - bf * a.block_size), ot = (int)(pt - bt * a.block_size);
                    if ((uint64_t)idf < (uint64_t)a.num_blocks && (uint64_t)idt < (uint64_t)a.num_blocks) {
                        from = idf * a.block_bytes;
                        to = idt * a.block_bytes;
                        s_off[tid][0] = of;
                        s_off[tid][1] = ot;
                    }
                }
            }
            s_from[tid] = from;
            s_to[tid] = to;
        }
        __syncthreads();
        const int count = s_count;
        if (live && column < a.columns) {
            for (int d = 0; d < count; d += kBatch) {
                U row[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    if (d + i < count && s_from[d + i] >= 0)
                        row[i] = *reinterpret_cast<const U*>(base + s_from[d + i] + s_off[d + i][0] * a.row_bytes +
                                                             column * sizeof(U));
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    if (d + i < count && s_from[d + i] >= 0)
                        *reinterpret_cast<U*>(base + s_to[d + i] + s_off[d + i][1] * a.row_bytes + column * sizeof(U)) =
                            row[i];
            }
        } else if (live) {
            const int64_t at = a.row_bytes * a.block_size + (column - a.columns) * a.block_size;
            for (int d = 0; d < count; ++d)
                if (s_from[d] >= 0) base[s_to[d] + at + s_off[d][1]] = base[s_from[d] + at + s_off[d][0]];
        }
        if (count < 64 || d0 + 64 >= a.max_depth) return;
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
    const int64_t gx = ceil_div((a.columns + scales) * num_tensors, 256);
    if (gx > 0x7fffffff) return fail(PKV_EUNSUPPORTED, "keep_paths: grid too large");
    const dim3 grid((unsigned)gx, (unsigned)num_seqs);
    if (unit == 16) keep_paths_kernel<uint4><<<grid, 256, 0, stream>>>(a);
    else if (unit == 4) keep_paths_kernel<uint32_t><<<grid, 256, 0, stream>>>(a);
    else keep_paths_kernel<uint8_t><<<grid, 256, 0, stream>>>(a);
    return check_launch("keep_paths");
}
