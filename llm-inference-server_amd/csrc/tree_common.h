// What the matrix kernels of tree attention share on the device: LDS DMA, windows of the masks, what is not
// finite in V. (Internal to libpagedkv; every file that includes it has its own copies.)
#pragma once

#include <type_traits>

#include "prefill_common.h"
#include "tree.h"

namespace pkv {
namespace {

__device__ __forceinline__ uint32_t lds_u32(const void* p) {
    return (uint32_t)(uintptr_t)((const __attribute__((address_space(3))) char*)p);
}
// 16 bytes per lane by LDS DMA to LDS address lds + 16 lane (M0 = lds), from the uniform base sbase plus
// the lane's 32-bit offset, or from the lane's own 64-bit address; inline asm, hidden from the
// compiler's wait counting, which would wait for it before every LDS read. M0 is reserved to the
// compiler (a clobber of it is not honoured): all LDS DMAs of these kernels go through these helpers.
__device__ __forceinline__ void dma16(const char* sbase, uint32_t voff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds), "v"(voff), "s"(sbase)
                 : "memory");
}
__device__ __forceinline__ void dma16(const char* addr, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"(lds), "v"(addr)
                 : "memory");
}

// A 32-bit word of the pool (two elements of a 16-bit type) with those elements that are not finite, whose
// exponent bits are all set, as zeros.
template <typename T>
__device__ __forceinline__ uint32_t finite_of(uint32_t w) {
    if constexpr (sizeof(T) == 4) {
        return (w & 0x7f800000u) == 0x7f800000u ? 0u : w;
    } else {
        constexpr uint32_t E = sizeof(T) == 2 && __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
        const uint32_t lo = (w & E) == E ? 0u : 0xffffu, hi = (w >> 16 & E) == E ? 0u : 0xffff0000u;
        return w & (lo | hi);
    }
}

// Four elements of a pool row.
template <typename T>
struct Four {
    uint32_t w[sizeof(T)];
    __device__ __forceinline__ static Four load(const T* p) {
        Four f;
        if constexpr (sizeof(T) == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            f.w[0] = v.x; f.w[1] = v.y; f.w[2] = v.z; f.w[3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            f.w[0] = v.x; f.w[1] = v.y;
        }
        return f;
    }
    // x + its elements that are not finite.
    __device__ __forceinline__ float4 add_rest(float4 x) const {
        uint32_t r[sizeof(T)];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); ++i) r[i] = w[i] ^ finite_of<T>(w[i]);
        if constexpr (sizeof(T) == 4) {
            auto f = [](uint32_t b) { return __builtin_bit_cast(float, b); };
            return make_float4(x.x + f(r[0]), x.y + f(r[1]), x.z + f(r[2]), x.w + f(r[3]));
        } else {
            return make_float4(x.x + Pair<T>::lo(r[0]), x.y + Pair<T>::hi(r[0]), x.z + Pair<T>::lo(r[1]),
                               x.w + Pair<T>::hi(r[1]));
        }
    }
};

// What a row sees. Its first two mask words, all there are up to 128 nodes, are in registers: read in the
// tile that needs them they hold it up by a memory round trip, and with it by the next tile's loads.
struct TreeRow {
    const uint64_t* mask;
    uint64_t first, second;
    __device__ __forceinline__ TreeRow(const uint64_t* m, int words)
        : mask(m), first(words > 0 ? m[0] : 0), second(words > 1 ? m[1] : 0) {}
    __device__ __forceinline__ uint64_t word(int i, int words) const {
        return i == 0 ? first : i == 1 ? second : i < words ? mask[i] : 0;
    }
    // Of the 32 keys from key0 on, those that it sees: all before pos0, and nodes by their bits, up to kmax.
    __device__ __forceinline__ uint32_t window(int words, int key0, int pos0, int kmax) const {
        const int node = key0 - pos0, left = kmax - key0;
        uint32_t w = ~0u;
        if (node >= 0) {
            const int sh = node & 63;
            const uint64_t lo = word(node >> 6, words) >> sh;
            w = (uint32_t)(sh > 32 ? lo | word((node >> 6) + 1, words) << (64 - sh) : lo);
        } else if (node > -32) {
            w = (uint32_t)(first << -node) | ((1u << -node) - 1);
        }
        return left >= 32 ? w : left <= 0 ? 0u : w & ((1u << left) - 1);
    }
};

// From a staged V tile of KEYS keys, key0 the first, of CPR 16-byte chunks each (in any order inside their
// row): keys past the last one and, of drafted keys, elements that are not finite, out (zeros; `taken` set).
// Cached keys are seen by all rows and stay. All 256 threads.
template <typename T, int KEYS, int CPR>
__device__ __forceinline__ void tree_take_out(char* tile_v, int key0, int pos0, int kmax, int& taken) {
    for (int c = (int)threadIdx.x; c < KEYS * CPR; c += 256) {
        const int key = key0 + c / CPR;
        if (key < pos0) continue;
        uint4* at = reinterpret_cast<uint4*>(tile_v) + c;
        const uint4 v = *at;
        const uint4 f = key < kmax ? make_uint4(finite_of<T>(v.x), finite_of<T>(v.y), finite_of<T>(v.z), finite_of<T>(v.w))
                                   : make_uint4(0, 0, 0, 0);
        if (f.x == v.x && f.y == v.y && f.z == v.z && f.w == v.w) continue;
        *at = f;
        if (key < kmax) taken = 1;
    }
}

}  // namespace
}  // namespace pkv
