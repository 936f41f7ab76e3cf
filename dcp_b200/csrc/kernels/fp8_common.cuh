// 8-bit codes with a power-of-two scale per block, shared by the kernels that make and read them.
//
// A block of values x is kept as codes c = round(x / s) in e4m3 or e5m2 and one byte for the scale s = 2^(e - 127)
// (e8m0): the smallest power of two with max|x| <= largest code * s.  Both formats' largest code is 1.75 * 2^b (448 and
// 57344), so the exponent comes from the exponent field of max|x| and one comparison of its mantissa, without a
// logarithm.  A block with a value that is not finite gets the byte 255, which stands for NaN: all of it reads back as
// NaN.  Zeros get the byte 0.
//
// The kernels are launched while the one before them ends (launch.cuh) and read what it writes, after grid_wait().  So no pointer
// to global memory is __restrict__ and nothing goes through __ldg: the compiler takes such loads for loads of constants, which
// it may move in front of the wait.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "ptx.cuh"

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
// eight values to codes, times 1 / scale (one, or one each)
template <int kCode>
__device__ __forceinline__ uint2 to_codes8(const uint64_t (&v)[4], const uint64_t (&inv)[4]) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    unpack_f32x2(mul_f32x2(v[i], inv[i]), lo, hi);
    c[i] = to_codes2<kCode>(lo, hi);
  }
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}
template <int kCode>
__device__ __forceinline__ uint2 to_codes8(const uint64_t (&v)[4], float inv) {
  const uint64_t two = pack_f32x2(inv, inv), all[4] = {two, two, two, two};
  return to_codes8<kCode>(v, all);
}
static_assert(kCodeE4m3 == 0 && kCodeE5m2 == 1, "code types are also the operand types of the tensor cores' instruction");

// ---------------------------------------------------------------- eight neighbouring values
// As they lie in memory, and as four pairs of fp32 for packed arithmetic.
template <typename T> struct Raw8 { uint32_t w[4]; };
template <> struct Raw8<float> { uint32_t w[8]; };
template <typename T> static constexpr int kWordsOf = sizeof(Raw8<T>) / 4;

template <typename T>
__device__ __forceinline__ void load_raw(Raw8<T>& r, const T* p) {   // on 16 bytes
#pragma unroll
  for (int i = 0; i < kWordsOf<T>; i += 4) {
    const uint4 v = reinterpret_cast<const uint4*>(p)[i / 4];
    r.w[i] = v.x; r.w[i + 1] = v.y; r.w[i + 2] = v.z; r.w[i + 3] = v.w;
  }
}
template <typename T>
__device__ __forceinline__ void store_raw(T* p, const Raw8<T>& r) {
#pragma unroll
  for (int i = 0; i < kWordsOf<T>; i += 4) reinterpret_cast<uint4*>(p)[i / 4] = make_uint4(r.w[i], r.w[i + 1], r.w[i + 2], r.w[i + 3]);
}
__device__ __forceinline__ float2 widen_word(__nv_bfloat16, uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ float2 widen_word(__half, uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <typename T>
__device__ __forceinline__ void widen(const Raw8<T>& r, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(r.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = widen_word(T(), r.w[i]);
      f[2 * i] = t.x; f[2 * i + 1] = t.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ void widen(const Raw8<T>& r, uint64_t (&f)[4]) {
  float v[8];
  widen(r, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = pack_f32x2(v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ uint32_t narrow_word(__nv_bfloat16, float lo, float hi) { return pack_bf16x2(lo, hi); }
__device__ __forceinline__ uint32_t narrow_word(__half, float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ Raw8<T> narrow(const float (&f)[8]) {
  Raw8<T> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = narrow_word(T(), f[2 * i], f[2 * i + 1]);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ Raw8<T> narrow(const uint64_t (&f)[4]) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack_f32x2(f[i], v[2 * i], v[2 * i + 1]);
  return narrow<T>(v);
}
// a + b in their type.  In 16 bits one rounding of the exact sum, as fp32's sum rounded again gives: a sum that fp32 does not
// hold has an addend too small to reach the middle between two values of the type.
template <typename T>
__device__ __forceinline__ Raw8<T> add_raw(const Raw8<T>& a, const Raw8<T>& b) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < kWordsOf<T>; ++i) {
    if constexpr (sizeof(T) == 4) {
      r.w[i] = __float_as_uint(__uint_as_float(a.w[i]) + __uint_as_float(b.w[i]));
    } else {
      using P = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
      const P v = __hadd2(*reinterpret_cast<const P*>(&a.w[i]), *reinterpret_cast<const P*>(&b.w[i]));
      r.w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  return r;
}

__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_float(float v) { return v; }

__device__ __forceinline__ float max3_abs(float a, float b, float c) {   // NaN if one is
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// largest magnitude of eight values, as bits: non-negative floats order like their bits, and NaN and infinity come above all
// finite ones
__device__ __forceinline__ uint32_t amax_bits(const uint64_t (&f)[4]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    unpack_f32x2(f[i], lo, hi);
    m = max3_abs(m, lo, hi);
  }
  return __float_as_uint(m);
}

// ---------------------------------------------------------------- rows that do not begin on 16 bytes
// The words of a longer piece, `bytes` (a multiple of two, below 16) further on.
template <int kWords>
__device__ __forceinline__ void shift_words(uint32_t (&w)[kWords], uint32_t bytes) {
  if (bytes & 8)
#pragma unroll
    for (int i = 0; i + 2 < kWords; ++i) w[i] = w[i + 2];
  if (bytes & 4)
#pragma unroll
    for (int i = 0; i + 1 < kWords; ++i) w[i] = w[i + 1];
  if (bytes & 2)
#pragma unroll
    for (int i = 0; i + 1 < kWords; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
}
// Values 8 chunk .. 8 chunk + 7 of a row of `width`, zeros behind its end.  Unaligned ones come in the aligned pieces of 16
// bytes that hold some of them (so none lies outside the memory they were allocated in, which begins and ends on more than
// 16), of which neighbouring threads share one: two accesses instead of eight.
template <bool kAligned, typename T>
__device__ __forceinline__ void load_chunk(const T* row, int chunk, int width, Raw8<T>& r) {
  const int n = width - chunk * 8;
  if (n <= 0) {
    r = Raw8<T>{};
    return;
  }
  if (kAligned) {   // rows hold whole chunks
    load_raw(r, row + chunk * 8);
    return;
  }
  constexpr int kWords = kWordsOf<T>;
  const uintptr_t at = reinterpret_cast<uintptr_t>(row + chunk * 8), base = at & ~uintptr_t(15), end = at + (n < 8 ? n : 8) * sizeof(T);
  uint32_t w[kWords + 4];
#pragma unroll
  for (int i = 0; i < kWords + 4; i += 4) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (base + 4 * i < end) v = *reinterpret_cast<const uint4*>(base + 4 * i);
    w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
  }
  shift_words(w, uint32_t(at & 15));
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    constexpr int kPer = 8 / kWords;
    r.w[i] = i * kPer >= n ? 0u : kPer == 2 && i * kPer + 1 >= n ? w[i] & 0xffffu : w[i];
  }
}
// The same for storing, by all 32 lanes of a warp with neighbouring chunks.  An unaligned lane stores the aligned pieces that
// begin inside its chunk, with what the next lane has; what has no such neighbour goes value by value.
template <bool kAligned, typename T>
__device__ __forceinline__ void store_chunk(T* row, int chunk, int width, const Raw8<T>& r) {
  const int n = min(width - chunk * 8, 8);
  T* p = row + chunk * 8;
  if (kAligned) {
    if (n > 0) store_raw(p, r);
    return;
  }
  constexpr int kWords = kWordsOf<T>;
  const int lane = threadIdx.x & 31;
  const uint32_t past = uint32_t(reinterpret_cast<uintptr_t>(p)) & 15;   // the same for all lanes
  uint32_t w[kWords + 4];
#pragma unroll
  for (int i = 0; i < kWords; ++i) w[i] = r.w[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[kWords + i] = __shfl_down_sync(0xffffffffu, r.w[i], 1);
  const int next = __shfl_down_sync(0xffffffffu, n, 1), head = past ? int((16 - past) / sizeof(T)) : 0;   // values before the first piece
  const bool pieces = n == 8 && (past == 0 || (lane < 31 && next >= head));
  const bool before = __shfl_up_sync(0xffffffffu, int(pieces), 1) && lane > 0 && past;   // the head is the lane before's
  if (past) shift_words(w, 16 - past);
  if (pieces) {
    Raw8<T> out;
#pragma unroll
    for (int i = 0; i < kWords; ++i) out.w[i] = w[i];
    store_raw(reinterpret_cast<T*>(reinterpret_cast<char*>(p) + (past ? 16 - past : 0)), out);
  }
  if (!pieces || !before) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t word = r.w[j * kWords / 8];
      if (j < n && (j < head ? !before : !pieces)) {
        if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(p)[j] = word;
        else reinterpret_cast<uint16_t*>(p)[j] = uint16_t(j & 1 ? word >> 16 : word);
      }
    }
  }
}

}  // namespace dcpk
