// Append to the 8-bit paged cache: new K/V rows are quantised (kv8.h) into their slots.
//
// Bound: HBM for prompts (a bf16 row of 128 is 256 bytes read, 129 written: 8,192 tokens of 8 KV
// heads, 50.5 MB, in 12.0 us, 4.2 TB/s, where a large copy reaches 4.9), latency for decode steps
// (32 tokens 2.8-3.8 us). A row is held by the fewest lanes that load it in 16-byte pieces (8
// elements a lane; fp32 two such pieces), so its largest magnitude is a reduction over 4 to 16
// neighbouring lanes (DPP) for head_dims up to 128, with no LDS. Two or four rows a lane, their
// loads in flight together, were slower (12.8 and 13.2 us), nontemporal loads too (14.1). The
// magnitude is taken on the bit patterns as integers: above 0x7f7fffff is a value that is not
// finite.
#include <type_traits>

#include "kv8.h"

namespace pkv {
namespace {

struct Kv8AppendArgs {
    uint8_t* codes[2];
    uint8_t* scales[2];
    const char* rows[2];
    const int64_t* slots;
    int64_t cb, cs, ch, sb, ss, sh;   // cache strides (bytes)
    int64_t st, sth;                  // row strides (elements): token, head
    int64_t num_slots, num_rows;      // num_rows = tokens * heads
    int block_size, block_shift, num_kv_heads, head_dim;
};

// Largest value over each aligned group of L lanes.
template <int L>
__device__ __forceinline__ uint32_t group_max(uint32_t x) {
    auto dpp = [](uint32_t v, auto ctrl) {
        return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, decltype(ctrl)::value, 0xf, 0xf, true);
    };
    auto mx = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    if constexpr (L >= 2) x = mx(x, dpp(x, std::integral_constant<int, kDppQuadXor1>()));
    if constexpr (L >= 4) x = mx(x, dpp(x, std::integral_constant<int, kDppQuadXor2>()));
    if constexpr (L >= 8) x = mx(x, dpp(x, std::integral_constant<int, kDppRowHalfMirror>()));
    if constexpr (L >= 16) x = mx(x, dpp(x, std::integral_constant<int, kDppRowMirror>()));
    if constexpr (L >= 32) {
        auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        x = mx((uint32_t)r[0], (uint32_t)r[1]);
    }
    if constexpr (L >= 64) {
        auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        x = mx((uint32_t)r[0], (uint32_t)r[1]);
    }
    return x;
}

// 8 elements of a row from element d, `n` of them inside it.
template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T* p, int n, float (&x)[8]) {
    if constexpr (WIDE) {
        if constexpr (sizeof(T) == 4) {
            const Vec16 a = load16(p), b = load16(p + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = __builtin_bit_cast(float, a.w[i]);
                x[4 + i] = __builtin_bit_cast(float, b.w[i]);
            }
        } else {
            const Vec16 a = load16(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = Pair<T>::lo(a.w[i]);
                x[2 * i + 1] = Pair<T>::hi(a.w[i]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i < n ? to_f32(p[i]) : 0.f;
    }
}

// L lanes a row, 8 elements a lane.
// WIDE: rows are 16-byte aligned multiples of 8 elements and codes 8-byte aligned.
template <typename T, int L, bool WIDE>
__global__ __launch_bounds__(256) void kv8_append_kernel(const Kv8AppendArgs a) {
    const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / L;
    const int sub = (int)threadIdx.x % L;
    const int which = (int)blockIdx.y;
    const bool live = row < a.num_rows;
    const int64_t r = live ? row : a.num_rows - 1;
    const int64_t tok = r / a.num_kv_heads;
    const int head = (int)(r - tok * a.num_kv_heads);
    const T* src = reinterpret_cast<const T*>(a.rows[which]) + tok * a.st + head * a.sth;
    const int64_t slot = a.slots[tok];
    const int d = sub * 8, n = a.head_dim - d;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (n > 0) load8<T, WIDE>(src + d, n, x);
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu;
        big = big > b ? big : b;
    }
    big = group_max<L>(big);
    if (!live || (uint64_t)slot >= (uint64_t)a.num_slots || n <= 0) return;   // outside the cache: skipped
    const uint32_t b = scale_byte(big);
    const int64_t blk = a.block_shift >= 0 ? slot >> a.block_shift : slot / a.block_size;
    const int64_t at = slot - blk * a.block_size;
    uint8_t* dst = a.codes[which] + blk * a.cb + at * a.cs + head * a.ch + d;
    const int shift = kScaleBias - (int)b;
    uint32_t w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float y[4];
#pragma unroll
        // Exact: within 448, and what falls below fp32 is far below e4m3's least step.
        for (int i = 0; i < 4; ++i) y[i] = __builtin_ldexpf(x[4 * j + i], shift);
        // Rounds to nearest, ties to even.
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        c = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
        w[j] = b == kScaleNan ? 0u : (uint32_t)c;
    }
    if constexpr (WIDE) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) dst[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
    if (sub == 0) a.scales[which][blk * a.sb + at * a.ss + head * a.sh] = (uint8_t)b;
}

template <typename T, bool WIDE>
int launch_kv8_append(const Kv8AppendArgs& a, hipStream_t stream) {
    int lanes = 4;
    while (lanes * 8 < a.head_dim) lanes *= 2;
    const int64_t gx = ceil_div(a.num_rows * lanes, 256);
    if (gx > 0x7fffffff) return fail(PKV_EUNSUPPORTED, "kv8_append: grid too large");
    const dim3 grid((unsigned)gx, 2);
    switch (lanes) {
        case 4: kv8_append_kernel<T, 4, WIDE><<<grid, 256, 0, stream>>>(a); break;
        case 8: kv8_append_kernel<T, 8, WIDE><<<grid, 256, 0, stream>>>(a); break;
        case 16: kv8_append_kernel<T, 16, WIDE><<<grid, 256, 0, stream>>>(a); break;
        case 32: kv8_append_kernel<T, 32, WIDE><<<grid, 256, 0, stream>>>(a); break;
        case 64: kv8_append_kernel<T, 64, WIDE><<<grid, 256, 0, stream>>>(a); break;
        default: return fail(PKV_EUNSUPPORTED, "kv8_append: head_dim %d > 512", a.head_dim);
    }
    return check_launch("kv8_append");
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int pkv_kv8_append(void* k_codes, void* v_codes, int64_t code_stride_block, int64_t code_stride_slot,
                              int64_t code_stride_head, void* k_scales, void* v_scales, int64_t scale_stride_block,
                              int64_t scale_stride_slot, int64_t scale_stride_head, int64_t num_blocks,
                              int64_t block_size, int64_t num_kv_heads, int64_t head_dim, const void* k_new,
                              const void* v_new, int64_t new_stride_t, int64_t new_stride_h, const int64_t* slots,
                              const int64_t* host_slots, int64_t num_tokens, int dtype, hipStream_t stream) {
    clear_error();
    if (dtype != PKV_FLOAT32 && dtype != PKV_FLOAT16 && dtype != PKV_BFLOAT16)
        return fail(PKV_EINVAL, "kv8_append: unknown dtype %d", dtype);
    if (num_tokens < 0 || num_blocks <= 0 || block_size <= 0 || num_kv_heads <= 0 || head_dim <= 0)
        return fail(PKV_EINVAL, "kv8_append: bad sizes");
    if (num_tokens > 0x7fffffff || num_kv_heads > 0x7fffffff || head_dim > 512 || block_size > 0x7fffffff)
        return fail(PKV_EUNSUPPORTED, "kv8_append: head_dim %lld > 512, or sizes beyond int32", (long long)head_dim);
    if (num_blocks > 0x7fffffffffffffff / block_size || num_tokens > ((int64_t)1 << 48) / num_kv_heads)
        return fail(PKV_EUNSUPPORTED, "kv8_append: slots or rows beyond what the kernel counts");
    if (num_tokens == 0) return PKV_OK;
    if (!k_codes || !v_codes || !k_scales || !v_scales || !k_new || !v_new || !slots)
        return fail(PKV_EINVAL, "kv8_append: null pointer");
    if (host_slots) {
        uint64_t high = 0;                      // a negative slot is above all others
        for (int64_t i = 0; i < num_tokens; ++i) high = high > (uint64_t)host_slots[i] ? high : (uint64_t)host_slots[i];
        if (high >= (uint64_t)(num_blocks * block_size))
            return fail(PKV_ERANGE, "slot index outside [0, %lld)", (long long)(num_blocks * block_size));
    }
    Kv8AppendArgs a = {};
    a.codes[0] = (uint8_t*)k_codes;
    a.codes[1] = (uint8_t*)v_codes;
    a.scales[0] = (uint8_t*)k_scales;
    a.scales[1] = (uint8_t*)v_scales;
    a.rows[0] = (const char*)k_new;
    a.rows[1] = (const char*)v_new;
    a.slots = slots;
    a.cb = code_stride_block;
    a.cs = code_stride_slot;
    a.ch = code_stride_head;
    a.sb = scale_stride_block;
    a.ss = scale_stride_slot;
    a.sh = scale_stride_head;
    a.st = new_stride_t;
    a.sth = new_stride_h;
    a.num_slots = num_blocks * block_size;
    a.num_rows = num_tokens * num_kv_heads;
    a.block_size = (int)block_size;
    a.block_shift = block_size & (block_size - 1) ? -1 : 63 - __builtin_clzll((unsigned long long)block_size);
    a.num_kv_heads = (int)num_kv_heads;
    a.head_dim = (int)head_dim;
    const int64_t isz = dtype == PKV_FLOAT32 ? 4 : 2;
    const uint64_t rows = (uint64_t)(uintptr_t)k_new | (uint64_t)(uintptr_t)v_new | (uint64_t)(new_stride_t * isz) |
                          (uint64_t)(new_stride_h * isz);
    const uint64_t codes = (uint64_t)(uintptr_t)k_codes | (uint64_t)(uintptr_t)v_codes |
                           (uint64_t)code_stride_block | (uint64_t)code_stride_slot | (uint64_t)code_stride_head;
    const bool wide = head_dim % 8 == 0 && rows % 16 == 0 && codes % 8 == 0;
    switch (dtype) {
        case PKV_FLOAT32: return wide ? launch_kv8_append<float, true>(a, stream) : launch_kv8_append<float, false>(a, stream);
        case PKV_FLOAT16:
            return wide ? launch_kv8_append<_Float16, true>(a, stream) : launch_kv8_append<_Float16, false>(a, stream);
        default: return wide ? launch_kv8_append<bf16_t, true>(a, stream) : launch_kv8_append<bf16_t, false>(a, stream);
    }
}
