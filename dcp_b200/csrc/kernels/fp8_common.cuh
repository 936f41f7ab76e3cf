// 8-bit codes with a power-of-two scale per block, shared by the kernels that make and read them.
//
// A block of values x is kept as codes c = round(x / s) in e4m3 or e5m2 and one byte for the scale s = 2^(e - 127)
// (e8m0): the smallest power of two with max|x| <= largest code * s.  Both formats' largest code is 1.75 * 2^b (448 and
// 57344), so the exponent comes from the exponent field of max|x| and one comparison of its mantissa, without a
// logarithm.  A block with a value that is not finite gets the byte 255, which stands for NaN: all of it reads back as
// NaN.  Zeros get the byte 0.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace dcpk {

enum : int { kTypeF32 = 0, kTypeF16 = 1, kTypeBf16 = 2 };      // of values, as in the attention kernels
enum : int { kCodeE4m3 = 0, kCodeE5m2 = 1 };

// exponent byte of the scale of a block whose largest magnitude has the bits `amax`; kTop: 8 for e4m3, 15 for e5m2
template <int kTop>
__device__ __forceinline__ int scale_byte(uint32_t amax) {
  if (amax >= 0x7f800000u) return 255;
  const int e = int(amax >> 23) - kTop + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < 0 ? 0 : e;   // at most 254 - kTop + 1
}
// 1 / s and s themselves; both are exact (2^127's reciprocal and 2^-127 are denormal)
__device__ __forceinline__ float scale_inverse(int byte) {
  return __uint_as_float(byte == 255 ? 0x7fffffffu : byte == 254 ? 0x00400000u : uint32_t(254 - byte) << 23);
}
__device__ __forceinline__ float scale_value(int byte) {
  return __uint_as_float(byte == 255 ? 0x7fffffffu : byte == 0 ? 0x00400000u : uint32_t(byte) << 23);
}

// two values to two codes, to nearest even, beyond the largest code to it; NaN stays NaN
template <int kCode>
__device__ __forceinline__ uint32_t to_codes2(float lo, float hi) {
  uint16_t r;
  if (kCode == kCodeE4m3) asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
template <int kCode>
__device__ __forceinline__ uint2 to_codes8(const float (&v)[8], float inv) {
  uint2 r;
  r.x = to_codes2<kCode>(v[0] * inv, v[1] * inv) | (to_codes2<kCode>(v[2] * inv, v[3] * inv) << 16);
  r.y = to_codes2<kCode>(v[4] * inv, v[5] * inv) | (to_codes2<kCode>(v[6] * inv, v[7] * inv) << 16);
  return r;
}
static_assert(kCodeE4m3 == 0 && kCodeE5m2 == 1, "code types are also the operand types of the tensor cores' instruction");

// values of type T, eight at a time or one by one, as fp32
template <typename T> struct Raw8 { uint4 v; };
template <> struct Raw8<float> { uint4 v, w; };

__device__ __forceinline__ void load_raw(Raw8<__nv_bfloat16>& r, const __nv_bfloat16* p) { r.v = *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void load_raw(Raw8<__half>& r, const __half* p) { r.v = *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void load_raw(Raw8<float>& r, const float* p) {
  r.v = reinterpret_cast<const uint4*>(p)[0];
  r.w = reinterpret_cast<const uint4*>(p)[1];
}
__device__ __forceinline__ void widen(const Raw8<__nv_bfloat16>& r, float (&f)[8]) {
  const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void widen(const Raw8<__half>& r, float (&f)[8]) {
  const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x; f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ void widen(const Raw8<float>& r, float (&f)[8]) {
  const uint32_t w[8] = {r.v.x, r.v.y, r.v.z, r.v.w, r.w.x, r.w.y, r.w.z, r.w.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_float(float v) { return v; }
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) {
  uint4 r;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = r;
}
__device__ __forceinline__ void store8(__half* p, const float (&f)[8]) {
  uint4 r;
  __half2* h = reinterpret_cast<__half2*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = r;
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

// largest magnitude as bits: non-negative floats order like their bits, and NaN and infinity come above all finite ones
__device__ __forceinline__ uint32_t amax_bits(uint32_t m, float v) { return max(m, __float_as_uint(v) & 0x7fffffffu); }

}  // namespace dcpk
