// The paged key / value cache's storage, shared by the kernels that write it, read it back and attend over it.
//
// A page holds page_size tokens of every head. K: [layers, pages, heads, page_size, D]; V: [layers, pages, heads,
// page_size / 4, D, 4], four tokens side by side, so that the four values of one dimension that a lane of a
// probability x value product needs are one word (8-bit kinds) or two (bf16). The 8-bit kinds keep for each
// (token, head) of K and of V a scale byte b: value = code * 2^(b - 127); b = 255 stands for a row that held a NaN or
// an infinity, which reads back as NaN throughout. A scale that is a power of two makes x / scale and code * scale
// exact, so the code is the correctly rounded one whatever the input's type and a row that was read back, written again,
// reads as the same values; the price is up to one bit of int8's range (e4m3, a floating type, loses none).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "noise_b200.h"

namespace noise {
namespace kv {

// The least scale byte with max|x| <= 2^(b - 127) * (largest code), from the bits of max|x|; [1, 254].
template <int KIND>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  constexpr int TOP = KIND == NOISE_KV_E4M3 ? 8 : 6;                        // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
  constexpr uint32_t FRACTION = KIND == NOISE_KV_E4M3 ? 0x600000u : 0x7e0000u;
  const int b = static_cast<int>(amax_bits >> 23) - TOP + ((amax_bits & 0x7fffffu) > FRACTION ? 1 : 0);
  return static_cast<uint32_t>(b < 1 ? 1 : b);
}

__device__ __forceinline__ float power(int biased) { return __uint_as_float(static_cast<uint32_t>(biased) << 23); }

// Four codes in a word, from x scaled to the codes' range.
template <int KIND>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if constexpr (KIND == NOISE_KV_E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  } else {
    const auto whole = [](float x) { return __float_as_uint(x + 12582912.f); };  // 1.5 * 2^23: rounds to the last bit
    return __byte_perm(__byte_perm(whole(a), whole(b), 0x0040), __byte_perm(whole(c), whole(d), 0x0040), 0x5410);
  }
}

// The four codes of a word as two pairs of fp16 (exact).
template <int KIND>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (KIND == NOISE_KV_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {  // 1024 + (code + 128) has the byte code ^ 0x80 as its last 8 bits
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}

}  // namespace kv
}  // namespace noise
