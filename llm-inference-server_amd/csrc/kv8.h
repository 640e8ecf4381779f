// The 8-bit paged cache: its format, and what its kernels share (internal to libpagedkv).
//
// A cached row (one token, one KV head, K or V) is head_dim e4m3 codes (OCP: bias 7, largest
// magnitude 448, NaN but no infinity) and one scale byte b: value = code * 2^(b - 127). b is
// the least with which the row's largest magnitude is at most 448. A row holding a value that
// is not finite is the NaN row: b = 255, codes 0.
//
// Why a power of two: e4m3 has an exponent of its own, so a finer scale would buy no relative
// precision; code * 2^k is exact in bf16 and fp32 (8 exponent bits) wherever it is a normal number
// of theirs, so the matrix instructions run on the cache's exact values; and quantising
// x * 2^(127 - b) rounds once. (Not 2^128, code 256 at b = 247, to which |x| of 1.9375 * 2^127 and
// more round up, as they do in other conversions to few bits; nor what is below 2^-126.)
// Why NaN in the scale: codes stay finite, so 0 * V is 0 where a key is masked.
#pragma once

#include "attention.h"

namespace pkv {

constexpr float kE4m3Max = 448.f;
constexpr int kScaleBias = 127;
constexpr int kScaleNan = 255;

// AttnParams with the codes as k / v (strides sb, ss, sh in bytes) and their scale bytes.
struct Kv8Params : AttnParams {
    const uint8_t* ks;
    const uint8_t* vs;
    int64_t ssb, sss, ssh;           // scale strides (bytes): block, slot, head
    int64_t max_context_len;
    // Decode: how the batch's keys are cut (kKv8Even ...), into how many runs per KV head at most,
    // the grid's room for them, the units that a run has at least, whether no sequence is cut,
    // and the rows of a partial (ws_o, ws_ml by [number][KV head][row]).
    int decode_mode, decode_slots, decode_grid, decode_min_units, decode_whole, decode_rows;
};

// Whether block strides, offsets inside a block and block numbers fit the 32-bit factors of the
// kernels that compute uniform addresses from them.
inline bool kv8_offsets_fit(const Kv8Params& p) {
    auto small = [&](int64_t slot) { return slot >= 0 && slot <= (1 << 26) && slot * p.block_size <= (1 << 30); };
    return small(p.ss) && small(p.sss) && p.sb >= 0 && p.sb <= 0x7fffffff && p.ssb >= 0 && p.ssb <= 0x7fffffff &&
           p.num_blocks <= 0x7fffffff;
}

// 2^(b - 127), NaN for 255.
__device__ __forceinline__ float scale_of(uint32_t b) {
    const uint32_t w = b << 23;
    return __builtin_bit_cast(float, (b == 0u || b == 255u) ? w | 0x00400000u : w);
}

// The scale byte of a row whose largest |x| has these fp32 bits: 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return kScaleNan;
    const int b = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return b < 0 ? 0u : (uint32_t)b;
}

// Decode (kv8_decode.h): at most 16 (token, query head) pairs per (sequence, KV head). What it
// asks of the shape, strides and addresses; its plan; its launch, by type.
enum { kKv8Even, kKv8Runs, kKv8WaveRuns };
constexpr int kKv8DecodeRows = 16, kKv8DecodeMaxSeqs = 2048;
bool kv8_decode_applies(const Kv8Params& p, int dtype);
// Sets p's decode fields but the pointers; returns the bytes of partials that cutting takes.
int64_t kv8_decode_plan(Kv8Params& p, const int64_t* host_ctx, const int64_t* host_qlen);
template <typename T>
int launch_kv8_decode(const Kv8Params& p, hipStream_t stream);

// Chunks (kv8_chunk.h): 128 rows a workgroup. What it asks likewise; contexts are cut by
// prefill_split_plan. Its launch returns PKV_EUNSUPPORTED, without an error, for grids that
// are too large.
bool kv8_chunk_applies(const Kv8Params& p, int dtype);
template <typename T>
int launch_kv8_chunk(const Kv8Params& p, hipStream_t stream);

// The rest: any shape.
int launch_kv8_generic(const Kv8Params& p, int dtype, hipStream_t stream);

}  // namespace pkv
