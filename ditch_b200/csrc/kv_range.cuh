// What the kernels that read the 8-bit cache share: the tiles of tokens that
// a run of rows sees, and 8-bit codes to f16 pairs.
#pragma once

#include "kvcache.cuh"

namespace ditch {
namespace kv {

// The tiles of `size` tokens that rows at positions lo .. hi see: the sinks'
// tiles, then those from the first row's window to the last row.
struct Range {
    int n, sink_tiles, first;
    __device__ __forceinline__ int token(int i, int size) const { return (i < sink_tiles ? i : i - sink_tiles + first) * size; }
};

__device__ __forceinline__ Range range_of(int lo, int hi, int window, int sinks, int size) {
    Range r;
    r.sink_tiles = 0;
    r.first = 0;
    if (window && lo - window + 1 > 0) {
        r.first = (lo - window + 1) / size;
        r.sink_tiles = min((sinks + size - 1) / size, r.first);
    }
    r.n = r.sink_tiles + hi / size + 1 - r.first;
    return r;
}

// Codes to f16, exactly. int8: the code + 128 goes into the mantissa of 1024,
// and 1152 is taken off again (to leave that to the products' f32 sums cost
// the digits of sums far smaller than the weights, and saved less than 2 %).
// E4M3 by cvt, a pair at a time.
__device__ __forceinline__ uint32_t int8_pair(uint32_t plus128, uint32_t select) {
    const uint32_t u = __byte_perm(plus128, 0x64646464u, select);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ void e4m3_pairs(uint32_t w, uint32_t &a, uint32_t &b) {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(a), "=r"(b)
        : "r"(w));
}

// Codes 2 half and 2 half + 1 of two tokens' four, each as a pair over the
// tokens.
template <bool FP8>
__device__ __forceinline__ void value_pairs(uint32_t w0, uint32_t w1, int half, uint32_t &a, uint32_t &b) {
    uint32_t u = __byte_perm(w0, w1, half ? 0x7362 : 0x5140);  // 0 of both, 1 of both
    if (FP8) {
        e4m3_pairs(u, a, b);
    } else {
        u ^= 0x80808080u;
        a = int8_pair(u, 0x4140);
        b = int8_pair(u, 0x4342);
    }
}

}  // namespace kv
}  // namespace ditch
