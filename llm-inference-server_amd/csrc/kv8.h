// The 8-bit paged cache: its format, and what its kernels share (internal to libpagedkv).
//
// A cached row (one token, one KV head, K or V) is head_dim e4m3 codes (OCP: bias 7, largest
// magnitude 448, NaN but no infinity) and one scale byte b: value = code * 2^(b - 127). b is
// the least with which the row's largest magnitude is at most 448. A row holding a value that
// is not finite is the NaN row: b = 255, codes 0.
//
// Why a power of two: e4m3 has an exponent of its own, so a finer scale would buy no relative
// precision; code * 2^k is exact in bf16 and fp32 (8 exponent bits), so the matrix
// instructions run on the cache's exact values; and quantising x * 2^(127 - b) rounds once.
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
    int slots;                       // decode: runs that the batch's keys are cut into, per KV head
};

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

// Decode (attn_kv8_decode.hip): rows of at most 16 (token, query head) pairs per (sequence,
// KV head). Chunks (attn_kv8_chunk.hip): 128 rows a workgroup. Both return PKV_EUNSUPPORTED
// without an error for what they do not take; the generic kernel takes the rest.
int launch_kv8_generic(const Kv8Params& p, int dtype, hipStream_t stream);

}  // namespace pkv
