// 8-bit key/value cache: element formats and block scales shared by the cache and attention
// kernels.
//
// Data (B, Hkv, cap, D) in e4m3 or int8; one scale byte per (sequence, head, block of T
// tokens), E8M0: scale = 2^(byte - 127).  The scale is the smallest power of two with
// amax <= QMAX * scale (QMAX 448 / 127), so dividing by it is exact and quantising is one
// rounding (to nearest even); for int8 that gives up half a bit on average against an
// arbitrary scale, and buys that a block whose maximum rises while it fills can be moved to
// the new scale by an exact shift, and that scales fold into exponents in the attention.
// Byte 255 marks a block that was given a NaN or an infinity: it reads back as NaN.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace mykb {
namespace kv8 {

typedef __nv_bfloat16 bf16;
constexpr int kMinScale = 27;   // 2^-100: keeps every scale, its inverse and their products normal in fp32
constexpr int kBadScale = 255;

// Scale byte for the largest magnitude of a block, given as bf16 bits without the sign.
template <bool INT8>
__device__ __forceinline__ int scale_byte(uint32_t amax16) {
  const int e = (int)(amax16 >> 7), m = (int)(amax16 & 127u);
  if (e == 255) return kBadScale;
  // amax = (1 + m / 128) 2^(e - 127); 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
  return max(kMinScale, INT8 ? e - 6 + (m > 126) : e - 8 + (m > 96));
}

__device__ __forceinline__ float scale_value(int byte) {  // 2^(byte - 127), NaN for kBadScale
  return byte == kBadScale ? __int_as_float(0x7fffffff) : __int_as_float(byte << 23);
}
__device__ __forceinline__ float scale_inverse(int byte) { return __int_as_float((254 - byte) << 23); }

// Two fp32 values -> two 8-bit values (low byte first), round to nearest even.
template <bool INT8>
__device__ __forceinline__ uint32_t quant2(float a, float b) {
  if constexpr (INT8) {
    const int x = max(-127, min(127, __float2int_rn(a))), y = max(-127, min(127, __float2int_rn(b)));
    return (uint32_t)(x & 255) | ((uint32_t)(y & 255) << 8);
  } else {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  }
}

// Four 8-bit values (a register, low byte first) -> two f16x2 registers, exactly.
template <bool INT8>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (INT8) {
    // the f16 with bits 0x6400 | u is 1024 + u; u = value + 128
    const uint32_t u = w ^ 0x80808080u;
    uint32_t l = __byte_perm(u, 0x64646464u, 0x4140), h = __byte_perm(u, 0x64646464u, 0x4342);
    const uint32_t off = 0x64806480u;  // 1152
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(l), "r"(off));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(h), "r"(off));
  } else {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

}  // namespace kv8
}  // namespace mykb
