// What the two kernels of the 4-bit products share: how packed weights become
// 16-bit values, and the kernel for a few rows.
#pragma once

#include "common.cuh"

namespace tv {
namespace w4 {

template <typename T> __device__ __forceinline__ T bits_as(uint32_t u) { return *reinterpret_cast<T*>(&u); }
template <typename T> __device__ __forceinline__ uint32_t as_bits(T v) { return *reinterpret_cast<uint32_t*>(&v); }

// Eight packed weights -> four pairs of 16-bit values in k order.
//
// bf16: the bits 0 .. 255 read as a bf16 are that integer times 2^-133 (the
// subnormal range and the first binade share a spacing), so a nibble masked at
// bits 0-3 is u * 2^-133 and one at bits 4-7 is u * 2^-129, and ONE fused
// multiply-add, (u * 2^-133) * (s * 2^(133 - 40)) - 8 s * 2^-40, gives
// (u - 8) * s * 2^-40 rounded once: both factors and the addend are exact.
// The accumulator is multiplied by 2^40 at the end.  Scales from 2^-80 to
// 2^30 stay inside the exponent range.  9 instructions for 8 weights; the
// usual 128 + u form needs a subtraction and a product, 15.
//
// fp16's exponents are too few for that.  It takes the form that 4-bit kernels
// commonly have: 1024 + u (or 1024 + 16 u), made by OR, loses its offset in one
// exact operation, then the product rounds once.
template <typename T> struct Unpack;
template <> struct Unpack<__nv_bfloat16> {
  __nv_bfloat162 sa, sb, off;
  __device__ __forceinline__ void scale(uint32_t twice) {      // the scale's bits in both halves
    const __nv_bfloat162 s2 = bits_as<__nv_bfloat162>(twice);
    sa = __hmul2(s2, __float2bfloat162_rn(9.903520314283042e27f));      // 2^93
    sb = __hmul2(s2, __float2bfloat162_rn(6.189700196426902e26f));      // 2^89
    off = __hmul2(s2, __float2bfloat162_rn(-7.275957614183426e-12f));   // -2^-37
  }
  __device__ __forceinline__ void word(uint32_t w, uint32_t* o) const {
    const uint32_t v = w >> 8;
    o[0] = as_bits(__hfma2(bits_as<__nv_bfloat162>(w & 0x000F000Fu), sa, off));
    o[1] = as_bits(__hfma2(bits_as<__nv_bfloat162>(w & 0x00F000F0u), sb, off));
    o[2] = as_bits(__hfma2(bits_as<__nv_bfloat162>(v & 0x000F000Fu), sa, off));
    o[3] = as_bits(__hfma2(bits_as<__nv_bfloat162>(v & 0x00F000F0u), sb, off));
  }
  static __device__ __forceinline__ float unscale() { return 1099511627776.0f; }   // 2^40
};
template <> struct Unpack<__half> {
  __half2 s2;
  __device__ __forceinline__ void scale(uint32_t twice) { s2 = bits_as<__half2>(twice); }
  __device__ __forceinline__ void word(uint32_t w, uint32_t* o) const {
    const uint32_t v = w >> 8;
    const __half2 lo = __float2half2_rn(-1032.f), sixteenth = __float2half2_rn(0.0625f), hi = __float2half2_rn(-72.f);
    o[0] = as_bits(__hmul2(__hadd2(bits_as<__half2>((w & 0x000F000Fu) | 0x64006400u), lo), s2));
    o[1] = as_bits(__hmul2(__hfma2(bits_as<__half2>((w & 0x00F000F0u) | 0x64006400u), sixteenth, hi), s2));
    o[2] = as_bits(__hmul2(__hadd2(bits_as<__half2>((v & 0x000F000Fu) | 0x64006400u), lo), s2));
    o[3] = as_bits(__hmul2(__hfma2(bits_as<__half2>((v & 0x00F000F0u) | 0x64006400u), sixteenth, hi), s2));
  }
  static __device__ __forceinline__ float unscale() { return 1.0f; }
};

// Index of the scale of 32-k unit u of a row: u / (group / 32) by
// multiplication; magic 0 stands for group 32.
__host__ __device__ inline uint32_t group_magic(int group) {
  const uint32_t g32 = (uint32_t)group / 32;
  return g32 == 1 ? 0 : (uint32_t)(((1ull << 32) + g32 - 1) / g32);
}

}  // namespace w4

// Whether the kernel for a few rows takes a request, and its launch.
bool w4_rows_fit(const tv_w4_args* a);
int launch_w4_rows(const tv_w4_args* a, cudaStream_t st);

}  // namespace tv
