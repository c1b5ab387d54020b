// li4_int4_pages.cuh -- rows of a cache in 4 bits: codes to values and back (sm_100a).
//
// A word of codes holds dims 0, 2, 4, 6 in the nibbles of its low half and dims 1, 3, 5, 7 in those of its high half, so a
// mask leaves a pair of neighbouring dims in the two halves of a register.  OR-ing a nibble into the mantissa of a
// power of two gives that power plus the code exactly (see li4_common.cuh); taking the power off and one fused
// multiply-add give c s + m rounded once.
#pragma once

#include "li4_common.cuh"

namespace li4 {

constexpr int kGroup4 = 32;  // LI4_KV_GROUP

template <typename T>
struct Codes4;
template <>
struct Codes4<__half> {
  static constexpr uint32_t NaN2 = 0x7fff7fffu;
  // The codes of nibble I of both halves of w as values.
  template <int I>
  static __device__ __forceinline__ uint32_t codes(uint32_t w) {
    // odd nibbles stand at bits 4 .. 7: 64 + c with the exponent of 64, where a unit is 16 of the last place
    const __half2 x = u32_as_h2(lop3_and_or(I >= 2 ? w >> 8 : w, I & 1 ? 0x00F000F0u : 0x000F000Fu,
                                            I & 1 ? 0x54005400u : 0x64006400u));
    const __half b = __ushort_as_half(I & 1 ? 0x5400 : 0x6400);
    return h2_as_u32(__hsub2(x, __halves2half2(b, b)));
  }
  static __device__ __forceinline__ uint32_t fma(uint32_t c, uint32_t s, uint32_t m) {
    return h2_as_u32(__hfma2(u32_as_h2(c), u32_as_h2(s), u32_as_h2(m)));
  }
  static __device__ __forceinline__ float value(uint16_t x) { return __half2float(__ushort_as_half(x)); }
  static __device__ __forceinline__ uint16_t nearest(double x) {
    return __half_as_ushort(__float2half_rn(__double2float_rn(x)));  // (by way of 32 bits)
  }
  static __device__ __forceinline__ uint16_t cut(float x) { return __half_as_ushort(__float2half_rz(x)); }  // towards zero
  static __device__ __forceinline__ uint16_t down(double x) { return cut(__double2float_rz(x)); }          // x >= 0
};
template <>
struct Codes4<__nv_bfloat16> {
  static constexpr uint32_t NaN2 = 0x7fff7fffu;
  template <int I>
  static __device__ __forceinline__ uint32_t codes(uint32_t w) {
    const uint32_t x = lop3_and_or(I ? w >> (4 * I) : w, 0x000F000Fu, 0x43004300u);  // 128 + c
    const __nv_bfloat16 b = __ushort_as_bfloat16(0x4300);
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), __halves2bfloat162(b, b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint32_t fma(uint32_t c, uint32_t s, uint32_t m) {
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&c),
                                     *reinterpret_cast<const __nv_bfloat162*>(&s),
                                     *reinterpret_cast<const __nv_bfloat162*>(&m));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float value(uint16_t x) { return __bfloat162float(__ushort_as_bfloat16(x)); }
  static __device__ __forceinline__ uint16_t nearest(double x) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(__double2float_rn(x)));
  }
  static __device__ __forceinline__ uint16_t cut(float x) { return __bfloat16_as_ushort(__float2bfloat16_rz(x)); }
  static __device__ __forceinline__ uint16_t down(double x) { return cut(__double2float_rz(x)); }
};

// (s, s) and (m, m) of a pair of parameters.
__device__ __forceinline__ uint32_t both_low(uint32_t p) { return __byte_perm(p, p, 0x1010); }
__device__ __forceinline__ uint32_t both_high(uint32_t p) { return __byte_perm(p, p, 0x3232); }

// The eight values of a word, dims in order: u[i] = (dim 2 i, dim 2 i + 1).
template <typename T>
__device__ __forceinline__ void values8(uint32_t w, uint32_t s2, uint32_t m2, uint32_t u[4]) {
  u[0] = Codes4<T>::fma(Codes4<T>::template codes<0>(w), s2, m2);
  u[1] = Codes4<T>::fma(Codes4<T>::template codes<1>(w), s2, m2);
  u[2] = Codes4<T>::fma(Codes4<T>::template codes<2>(w), s2, m2);
  u[3] = Codes4<T>::fma(Codes4<T>::template codes<3>(w), s2, m2);
}

}  // namespace li4
