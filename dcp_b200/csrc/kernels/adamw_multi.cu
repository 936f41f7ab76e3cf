// One AdamW step over many tensors, moments in 32 or 8 bits.
//
//   m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2      w -= lr (m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps) + wd w)
//
// with g the gradient times grad_scale and the clipping coefficient min(1, clip / (norm + 1e-6)).  28 bytes per parameter with
// moments in 32 bits (bf16 parameter and gradient, fp32 master), 16 with moments in 8, and 2 more for the norm.  218M parameters
// in 32 bits: norm 70 us (6.2 TB/s), update 967 (6.3 TB/s), bound by HBM.  In 8 bits: update 648 us (5.3 TB/s), bound by issuing 78
// instructions per parameter (75 % of the slots): hash 9, rounding and packing of two codes 15, the moments 11, root and
// quotient 13, addresses and conversions.
//
// Moments in 8 bits: m and sqrt(v) as e4m3 with a power-of-two scale per 256 values (fp8_common.cuh).  The root, because it
// is what the update divides by and because it halves v's range of exponents.  A moving average does not survive rounding to
// nearest: with b2 = 0.999 a step changes sqrt(v) by 0.05 %, half a step of e4m3 is 3 to 6 %, so it would never decay.  So
// the codes are rounded stochastically: 16 random bits are added behind the code's last place before the cut, which is
// right on average.  The bits are a hash of seed, step, tensor and element, so a step can be repeated to the bit.  A root
// that is not zero keeps the smallest code at least: the update never divides by eps alone where there was a gradient.  A
// moment that is not finite is kept as NaN and leaves its neighbours and the scale alone, as in 32 bits.
//
// A warp works on the 256 values of a scale, eight per lane.  The tensors' addresses are kernel arguments: no table has to
// be brought to the GPU when gradients move, and a captured graph holds its own.  The step counter and the bias corrections
// are on the GPU, so a replayed graph counts on.
#include <algorithm>

#include "entries.h"
#include "fp8_common.cuh"
#include "launch.cuh"
#include "ptx.cuh"

namespace dcpk {

static constexpr int kAdamTensors = 128;   // of a launch
static constexpr int kStateBlock = 256;
static constexpr int kAdamThreads = 256;
static constexpr int kChunk = kAdamThreads * 8;   // values a CTA takes at a time: one block per warp

struct AdamTensor {
  void* param;
  const void* grad;
  float* master;             // null: the parameter is its own master
  void* m;
  void* v;
  uint8_t* m_scale;
  uint8_t* v_scale;
  long n;
};
struct AdamList {
  AdamTensor t[kAdamTensors];
  int first_chunk[kAdamTensors + 1];
  uint8_t aligned[kAdamTensors];
  int n, base;               // base: tensors in launches before
};
struct AdamScalars { float lr, beta1, rest1, beta2, rest2, eps, wd; };   // rest: 1 - beta
static constexpr int kAdamStatus = 4;
struct AdamStatus { const int* word[kAdamStatus]; };   // null: none
// what a step's kernels hand on, in global memory
struct AdamShared { float coef, bc1, root_bc2; uint32_t key; int skip; };

// finaliser of MurmurHash3 (A. Appleby, public domain), and without its last step
__device__ __forceinline__ uint32_t mix32_open(uint32_t x) {
  x ^= x >> 16; x *= 0x85ebca6bu;
  x ^= x >> 13; x *= 0xc2b2ae35u;
  return x;
}
__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x = mix32_open(x);
  return x ^ (x >> 16);
}

// the tensor a chunk belongs to
__device__ __forceinline__ int find_tensor(const AdamList& list, int chunk) {
  int lo = 0, hi = list.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (list.first_chunk[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

// Loads leave L1 alone: nothing is read twice, and with the moments in 8 bits that is worth 4 % (218M parameters 780 -> 750 us).
// Eight neighbours, a 16-byte access in 16-bit types and one of 32 bytes in fp32 (two of 16 bytes, each of which touches all
// sectors of the warp's 1024 bytes: see the kernel's figures); otherwise one by one, every 32nd.
__device__ __forceinline__ void load_near(const float* p, float (&f)[8]) {
  uint32_t r[8];
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "l"(p) : "memory");
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(r[j]);
}
template <typename T>
__device__ __forceinline__ void load_near(const T* p, float (&f)[8]) {
  Raw8<T> raw;
  load_raw(raw, p);
  widen(raw, f);
}
__device__ __forceinline__ void store_near(float* p, const float (&f)[8]) {
  uint32_t r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = __float_as_uint(f[j]);
  st_global_v8(p, r);
}
template <typename T>
__device__ __forceinline__ void store_near(T* p, const float (&f)[8]) { store_raw(p, narrow<T>(f)); }

template <typename T>
__device__ __forceinline__ void load8(const T* p, long e0, int lane, long n, bool vec, float (&f)[8]) {
  if (vec) {
    load_near(p + e0 + lane * 8, f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = e0 + j * 32 + lane < n ? to_float(p[e0 + j * 32 + lane]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, long e0, int lane, long n, bool vec, Raw8<T>& r) {   // as they lie in memory
  if (vec) {
    if constexpr (sizeof(T) == 2)
      asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]) : "l"(p + e0 + lane * 8) : "memory");
    else load_raw(r, p + e0 + lane * 8);
  } else {
    T v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = e0 + j * 32 + lane < n ? p[e0 + j * 32 + lane] : from_float<T>(0.f);
    r = *reinterpret_cast<const Raw8<T>*>(v);
  }
}
template <typename T>
__device__ __forceinline__ void put8(T* p, long e0, int lane, long n, bool vec, const float (&f)[8]) {
  if (vec) {
    store_near(p + e0 + lane * 8, f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (e0 + j * 32 + lane < n) p[e0 + j * 32 + lane] = from_float<T>(f[j]);
  }
}
__device__ __forceinline__ float2 from_codes2(uint32_t c) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(c)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ uint2 load_codes8(const uint8_t* p, long e0, int lane, long n, bool vec) {
  if (vec) {
    uint2 r;
    asm volatile("ld.global.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p + e0 + lane * 8) : "memory");
    return r;
  }
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (e0 + j * 32 + lane < n) w[j >> 2] |= uint32_t(p[e0 + j * 32 + lane]) << (8 * (j & 3));
  return make_uint2(w[0], w[1]);
}
// codes as values, without their scale
__device__ __forceinline__ void widen_codes(uint2 r, float (&f)[8]) {
  const uint32_t w[2] = {r.x, r.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = from_codes2(w[i >> 1] >> (16 * (i & 1)));
    f[2 * i] = t.x; f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ void store_codes8(uint8_t* p, long e0, int lane, long n, bool vec, uint2 r) {
  if (vec) {
    *reinterpret_cast<uint2*>(p + e0 + lane * 8) = r;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (e0 + j * 32 + lane < n) p[e0 + j * 32 + lane] = uint8_t((j < 4 ? r.x : r.y) >> (8 * (j & 3)));
  }
}
// Square root by one step of Newton's iteration with the residual of a fused product: to nearest but for one value in a
// million, without sqrtf's branch for the ends of the range.  Zero for zero; below 2^-126 too small, NaN for infinity: those
// take sqrtf.
__device__ __forceinline__ float root_of(float v) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaxf(v, 1.17549435e-38f)));
  const float r = v * y;
  return fmaf(fmaf(-r, r, v), 0.5f * y, r);
}
__device__ __forceinline__ float inverse_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// Codes of a block's values, at random to one of the two neighbours; `amax` is the block's largest magnitude.  A product
// with 2^-120 / scale takes e4m3's smallest exponent to fp32's: the code is bits 20 to 26 then, for its denormals too, and
// the cut is a shift.  The largest magnitude is at most 448 * scale, whose bits below the code are zero: no sum goes past the
// code 0x7e.
template <bool kRoot>
__device__ __forceinline__ uint2 encode8(float amax, const float (&f)[8], const uint32_t (&random)[8], int& byte) {
  uint32_t top[8];   // the code in the upper byte
  // 16 random bits are added behind the code, the upper ones of the hash or the lower, whose last step (x ^ x >> 16) is done
  // here.  Not as (bits << 4) + __byte_perm(...), which is an instruction less: ptxas of CUDA 12.9 makes codes of zero of that.
  const auto cut = [](uint32_t bits, uint32_t x) { return (bits + ((kRoot ? x >> 12 : (x << 4) ^ (x >> 12)) & 0xffff0u)) << 4; };
  byte = scale_byte<8>(__float_as_uint(amax));
  if (byte <= 156) {   // 2^-120 / scale is a float
    const float inv = byte <= 133 ? __uint_as_float(uint32_t(134 - byte) << 23) : __uint_as_float(0x00400000u >> (byte - 134));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t bits = __float_as_uint(fabsf(f[j]) * inv);
      if (kRoot) bits = max(bits, min(__float_as_uint(f[j]), 0x00100000u));
      top[j] = cut(bits, random[j]);
      if (!kRoot) top[j] |= __float_as_uint(f[j]) & 0x80000000u;
    }
  } else {             // huge, or something that is not finite: those become NaN and do not count for the scale
    uint32_t finite = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = __float_as_uint(f[j]) & 0x7fffffffu;
      finite = max(finite, b < 0x7f800000u ? b : 0u);
    }
    byte = scale_byte<8>(__reduce_max_sync(0xffffffffu, finite));
    const float inv = scale_inverse(byte);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = fabsf(f[j]);
      uint32_t bits = __float_as_uint(a * inv * 0x1p-120f);
      if (kRoot && a > 0.f) bits = max(bits, 0x00100000u);
      top[j] = cut(bits, random[j]);
      if (!(a < INFINITY)) top[j] = 0x7f000000u;
      if (!kRoot) top[j] |= __float_as_uint(f[j]) & 0x80000000u;
    }
  }
  const auto four = [&](int i) {
    return __byte_perm(__byte_perm(top[i], top[i + 1], 0x0073), __byte_perm(top[i + 2], top[i + 3], 0x0073), 0x5410);
  };
  return make_uint2(four(0), four(4));
}

// Sum of squares of 8 kN values, in fp32 for these few and from there on in 64 bits.  fp32 does not hold a square above 2^128 and
// rounds one below 2^-126 to a multiple of 2^-149, so where the sum is not finite or below 2^-100 (against which 32 such
// roundings do not count) it is taken again in 64 bits, from the gradients on: a single gradient of 1e20 would make the norm
// infinite, and what it clips zero.
template <typename G, int kN>
__device__ __forceinline__ double sum_of_squares(const Raw8<G> (&raw)[kN], float scale) {
  float sq[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < kN; ++u) {
    float g[8];
    widen(raw[u], g);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = g[j] * scale;
      sq[j] += x * x;
    }
  }
  const float sum = ((sq[0] + sq[1]) + (sq[2] + sq[3])) + ((sq[4] + sq[5]) + (sq[6] + sq[7]));
  if (sum >= 0x1p-100f && sum < INFINITY) return double(sum);
  double wide = 0.0;
#pragma unroll
  for (int u = 0; u < kN; ++u) {
    float g[8];
    widen(raw[u], g);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double x = double(g[j]) * double(scale);
      wide += x * x;
    }
  }
  return wide;
}

// Sum of squares of a CTA's gradients; `parts` are added up in order.  A CTA has a run of chunks, so that it looks for its tensor
// once and has four loads per thread under way (a chunk at a time from a grid of CTAs: 436 MB in 144 us).
template <typename G>
__global__ void __launch_bounds__(kAdamThreads) adamw_norm_kernel(const __grid_constant__ AdamList list, float grad_scale, double* parts) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_chunks = list.first_chunk[list.n];
  double t = 0.0;
  grid_wait();
  int chunk = int(long(n_chunks) * blockIdx.x / gridDim.x);
  const int stop = int(long(n_chunks) * (blockIdx.x + 1) / gridDim.x);
  for (int i = find_tensor(list, chunk); chunk < stop; ++i) {
    const int last = min(stop, list.first_chunk[i + 1]);   // of this tensor
    const long n = list.t[i].n;
    const G* grad = static_cast<const G*>(list.t[i].grad);
    long e0 = long(chunk - list.first_chunk[i]) * kChunk;
    const long end = min(n, long(last - list.first_chunk[i]) * kChunk);
    if (list.aligned[i])
      for (; e0 + 4 * kChunk <= end; e0 += 4 * kChunk) {
        Raw8<G> raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) load_raw(raw[u], grad + e0 + u * kChunk + threadIdx.x * 8);
        t += sum_of_squares(raw, grad_scale);
      }
    for (; e0 < end; e0 += kChunk) {
      const long at = e0 + warp * kStateBlock;
      Raw8<G> raw[1];
      load8(grad, at, lane, n, list.aligned[i] && at + kStateBlock <= n, raw[0]);
      t += sum_of_squares(raw, grad_scale);
    }
    chunk = last;
  }
  grid_let_next();
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) t += __shfl_xor_sync(0xffffffffu, t, s);
  __shared__ double warps[kAdamThreads / 32];
  if (lane == 0) warps[warp] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kAdamThreads / 32; ++w) t += warps[w];
    parts[blockIdx.x] = t;
  }
}

// step counter, bias corrections, clipping coefficient: one CTA
__global__ void __launch_bounds__(256) adamw_prepare_kernel(const double* parts, int n_parts, int64_t* step, double beta1,
                                                            double beta2, float grad_scale, float clip, const float* factor,
                                                            uint32_t seed, float* norm, const AdamStatus status, AdamShared* shared) {
  __shared__ double sums[8];
  grid_wait();
  grid_let_next();
  double t = 0.0;
  for (int i = threadIdx.x; i < n_parts; i += 256) t += parts[i];
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) t += __shfl_xor_sync(0xffffffffu, t, s);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = t;
  __syncthreads();
  if (threadIdx.x) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) t += sums[w];
  bool skip = false;
#pragma unroll
  for (int i = 0; i < kAdamStatus; ++i) skip |= status.word[i] && *status.word[i] != 0;
  const int64_t now = *step + 1;
  if (!skip) *step = now;
  shared->skip = skip;
  float coef = factor ? grad_scale * *factor : grad_scale;
  if (n_parts > 0) {
    const double length = sqrt(t);
    *norm = float(length);
    const float c = float(double(clip) / (length + 1e-6));
    coef *= c > 1.f ? 1.f : c;   // a NaN norm gives NaN
  }
  shared->coef = coef;
  shared->bc1 = float(1.0 / (1.0 - pow(beta1, double(now))));
  shared->root_bc2 = float(sqrt(1.0 / (1.0 - pow(beta2, double(now)))));
  shared->key = mix32(seed + uint32_t(now) * 0x9e3779b1u);
}

template <typename G>
struct Block8 {   // a lane's part of a block with moments in 8 bits
  Raw8<G> grad;
  float w[8];
  uint2 m, v;
  int m_byte, v_byte;
};

// All CTAs walk the chunks together: neighbours in time are neighbours in memory (a run of chunks for each CTA: 896 -> 979 us
// for 218M parameters in 8 bits).
template <typename P, typename G, bool kMaster, bool kEight>
__global__ void __launch_bounds__(kAdamThreads, kEight ? 3 : 5) adamw_multi_kernel(const __grid_constant__ AdamList list, const AdamScalars s,
                                                                                   const AdamShared* shared) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_chunks = list.first_chunk[list.n];
  grid_wait();
  if (shared->skip) return;
  const float coef = shared->coef, bc1 = shared->bc1, root_bc2 = shared->root_bc2;
  const bool small_numbers = kEight && (s.eps < root_bc2 * 0x1p-37f || s.beta2 < 0x1p-10f);   // see update()
  int chunk = blockIdx.x;
  for (int i = find_tensor(list, chunk); chunk < n_chunks; ++i) {
    const AdamTensor& t = list.t[i];
    const long n = t.n;
    const uint32_t key = kEight ? mix32(shared->key + uint32_t(list.base + i) * 0x85ebca77u) : 0u;
    const bool aligned = list.aligned[i];
    const auto start_of = [&](int c) { return long(c - list.first_chunk[i]) * kChunk + warp * kStateBlock; };
    if constexpr (kEight) {
      Block8<G> next;
      const auto fetch = [&](Block8<G>& b, long e0, bool vec) {
        load8(static_cast<const G*>(t.grad), e0, lane, n, vec, b.grad);
        if (kMaster) load8(static_cast<const float*>(t.master), e0, lane, n, vec, b.w);
        else load8(static_cast<const P*>(t.param), e0, lane, n, vec, b.w);
        b.m = load_codes8(static_cast<const uint8_t*>(t.m), e0, lane, n, vec);
        b.v = load_codes8(static_cast<const uint8_t*>(t.v), e0, lane, n, vec);
        b.m_byte = t.m_scale[e0 / kStateBlock];
        b.v_byte = t.v_scale[e0 / kStateBlock];
      };
      // kWide: for blocks near the ends of fp32's range
      const auto body = [&](const Block8<G>& b, const float (&g)[8], long e0, bool vec, auto wide) {
        constexpr bool kWide = decltype(wide)::value;
        float w[8], m[8], v[8], root[8];
        // the scales are powers of two: they go into the factors the codes are multiplied with anyway
        const float keep_m = s.beta1 * scale_value(b.m_byte), v_scale = scale_value(b.v_byte), keep_v = s.beta2 * v_scale * v_scale;
        widen_codes(b.m, m);
        widen_codes(b.v, v);
        uint32_t random[8];
        float m_max = 0.f, v_max = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          // each rounded by itself: old moments and gradients are short numbers, so blocks whose largest value lies on the
          // very border between two scales are not rare, and a fused product would take them to the other side than the
          // formula
          m[j] = __fadd_rn(__fmul_rn(keep_m, m[j]), __fmul_rn(s.rest1, g[j]));
          const float old = kWide ? v[j] * v_scale : v[j];
          v[j] = __fadd_rn(__fmul_rn(kWide ? s.beta2 : keep_v, __fmul_rn(old, old)), __fmul_rn(__fmul_rn(s.rest2, g[j]), g[j]));
          if (j & 1) {
            m_max = max3_abs(m_max, m[j - 1], m[j]);
            v_max = max3_abs(v_max, v[j - 1], v[j]);
          }
          root[j] = kWide ? sqrtf(v[j]) : root_of(v[j]);
          w[j] = b.w[j] - s.lr * (m[j] * bc1 * inverse_approx(root[j] * root_bc2 + s.eps) + s.wd * b.w[j]);
          random[j] = mix32_open(uint32_t(e0 + (vec ? lane * 8 + j : j * 32 + lane)) * 0x9e3779b1u + key);
        }
        if (kMaster) put8(t.master, e0, lane, n, vec, w);
        put8(static_cast<P*>(t.param), e0, lane, n, vec, w);
        int m_byte, v_byte;
        m_max = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m_max)));
        v_max = sqrtf(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v_max))));
        store_codes8(static_cast<uint8_t*>(t.m), e0, lane, n, vec, encode8<false>(m_max, m, random, m_byte));
        store_codes8(static_cast<uint8_t*>(t.v), e0, lane, n, vec, encode8<true>(v_max, root, random, v_byte));
        if (lane == 0) {
          t.m_scale[e0 / kStateBlock] = uint8_t(m_byte);
          t.v_scale[e0 / kStateBlock] = uint8_t(v_byte);
        }
      };
      // A v may overflow (its root is infinite and moves nothing), lie below 2^-126 (beside a root above 2^-45 in its block such a
      // root has the smallest code whatever it is, and beside eps it does not count, unless that is small), or come of a
      // scale whose square times beta2 leaves fp32's normal range.  The gradients and the old scale tell where none of it can
      // be: v >= beta2 (224 scale)^2 and (1 - beta2) g^2.  Looked for before anything is computed: 218M parameters 763.4 -> 764.6 us;
      // after the fast form, whose weights and roots then wait for the answer, 755.6 -> 789.6.  All blocks in this form (eps =
      // 1e-15) take 1 % longer: update alone 675 -> 680.
      const auto update = [&](const Block8<G>& b, long e0, bool vec) {
        float g[8], g_max = 0.f;
        widen(b.grad, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          g[j] *= coef;
          if (j & 1) g_max = max3_abs(g_max, g[j - 1], g[j]);
        }
        const bool wide = !(g_max < 0x1p60f) || (b.v_byte == 0 && g_max < 0x1p-30f && g_max > 0.f);
        if (__any_sync(0xffffffffu, wide) || uint32_t(b.v_byte - 1) < 79u || b.v_byte > 180 || small_numbers) body(b, g, e0, vec, std::true_type());
        else body(b, g, e0, vec, std::false_type());
      };
      // whole blocks, the next one's loads under way while this one is worked on; then the tensor's end, or all of it where
      // it is not aligned
      const auto whole = [&](int c) { return aligned && c < list.first_chunk[i + 1] && start_of(c) + kStateBlock <= n; };
      if (whole(chunk)) fetch(next, start_of(chunk), true);
      for (; whole(chunk); chunk += gridDim.x) {
        const Block8<G> now = next;
        if (whole(chunk + gridDim.x)) fetch(next, start_of(chunk + gridDim.x), true);
        update(now, start_of(chunk), true);
      }
      for (; chunk < list.first_chunk[i + 1]; chunk += gridDim.x)
        if (start_of(chunk) < n) {
          fetch(next, start_of(chunk), false);
          update(next, start_of(chunk), false);
        }
    } else {
      for (; chunk < list.first_chunk[i + 1]; chunk += gridDim.x) {
        const long e0 = start_of(chunk);
        if (e0 >= n) continue;
        const bool vec = aligned && e0 + kStateBlock <= n;
        float g[8], w[8], m[8], v[8];
        load8(static_cast<const G*>(t.grad), e0, lane, n, vec, g);
        if (kMaster) load8(static_cast<const float*>(t.master), e0, lane, n, vec, w);
        else load8(static_cast<const P*>(t.param), e0, lane, n, vec, w);
        load8(static_cast<const float*>(t.m), e0, lane, n, vec, m);
        load8(static_cast<const float*>(t.v), e0, lane, n, vec, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          g[j] *= coef;
          m[j] = s.beta1 * m[j] + s.rest1 * g[j];
          v[j] = s.beta2 * v[j] + s.rest2 * g[j] * g[j];
          w[j] -= s.lr * (m[j] * bc1 / (sqrtf(v[j]) * root_bc2 + s.eps) + s.wd * w[j]);
        }
        if (kMaster) put8(t.master, e0, lane, n, vec, w);
        put8(static_cast<P*>(t.param), e0, lane, n, vec, w);
        put8(static_cast<float*>(t.m), e0, lane, n, vec, m);
        put8(static_cast<float*>(t.v), e0, lane, n, vec, v);
      }
    }
  }
}

}  // namespace dcpk

using namespace dcpk;

static constexpr int kAdamHead = 4;   // doubles
static int adam_norm_ctas(int chunks) { return std::min(chunks, 148 * 4); }

// doubles of `work` a call needs: what the kernels hand on, and a sum per CTA of each launch of the norm
extern "C" long dcpk_adamw_multi_work(int n_tensors) { return kAdamHead + long((n_tensors + kAdamTensors - 1) / kAdamTensors) * 148 * 4; }

// Tensors of one parameter type and one gradient type (0 fp32, 1 fp16, 2 bf16); an entry of `masters` may be null for fp32
// parameters only.  m_scales null: moments in fp32; otherwise codes with ceil(n / 256) scales.  step: one int64 on the
// device, counted up.  clip <= 0: none, and norm is not written.  factor: null, or one float on the device that the gradients
// are multiplied with.  status: up to four words that, when one is not zero, leave everything as it is.
extern "C" int dcpk_adamw_multi(int n_tensors, void* const* params, const void* const* grads, void* const* masters, void* const* ms,
                                void* const* vs, void* const* m_scales, void* const* v_scales, const long* sizes, int param_type, int grad_type,
                                int64_t* step, float lr, double beta1, double beta2, float eps, float wd, float grad_scale, float clip,
                                const float* factor, unsigned seed, float* norm, const int* const* status, int n_status, double* work,
                                void* stream) {
  if (n_status < 0 || n_status > kAdamStatus) return -3;
  AdamStatus words;
  for (int i = 0; i < kAdamStatus; ++i) words.word[i] = i < n_status ? status[i] : nullptr;
  if (n_tensors < 0 || param_type < 0 || param_type > 2 || grad_type < 0 || grad_type > 2) return -3;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  AdamShared* shared = reinterpret_cast<AdamShared*>(work);
  double* parts = work + kAdamHead;
  static_assert(sizeof(AdamShared) <= kAdamHead * 8, "work begins with it");
  const bool eight = m_scales != nullptr, has_master = masters != nullptr;
  if (!has_master && param_type != kTypeF32) return -3;
  for (int i = 0; i < n_tensors; ++i)
    if (sizes[i] < 0 || sizes[i] / kChunk >= 0x7fffffffl - kAdamTensors) return -3;
  const auto fill = [&](AdamList& list, int base) -> int {   // the next launch's tensors; returns how many it took
    list.base = base;
    list.n = 0;
    list.first_chunk[0] = 0;
    int i = base;
    for (; i < n_tensors && list.n < kAdamTensors; ++i) {
      const long chunks = (sizes[i] + kChunk - 1) / kChunk;
      if (list.first_chunk[list.n] + chunks > 0x7fffffffl) break;
      AdamTensor& t = list.t[list.n];
      t = {params[i], grads[i], has_master ? static_cast<float*>(masters[i]) : nullptr, ms[i], vs[i],
           eight ? static_cast<uint8_t*>(m_scales[i]) : nullptr, eight ? static_cast<uint8_t*>(v_scales[i]) : nullptr, sizes[i]};
      const auto at = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
      list.aligned[list.n] = at(t.param) % (param_type ? 16 : 32) == 0 && at(t.grad) % (grad_type ? 16 : 32) == 0 && at(t.master) % 32 == 0 &&
                             (at(t.m) | at(t.v)) % (eight ? 8 : 32) == 0;
      list.first_chunk[list.n + 1] = int(list.first_chunk[list.n] + chunks);
      ++list.n;
    }
    return i - base;
  };
  const auto by_type = [](int type, auto f) {
    return type == kTypeBf16 ? f(static_cast<__nv_bfloat16*>(nullptr)) : type == kTypeF16 ? f(static_cast<__half*>(nullptr)) : f(static_cast<float*>(nullptr));
  };
  AdamList list;
  int n_parts = 0;
  bool first = true;   // of the call: what ran before is not told apart from a kernel that does not wait
  if (clip > 0.f)
    for (int base = 0; base < n_tensors;) {
      base += fill(list, base);
      const int chunks = list.first_chunk[list.n];
      if (chunks == 0) continue;
      const int ctas = adam_norm_ctas(chunks);
      const cudaError_t rc = by_type(grad_type, [&](auto* g) {
        using G = std::remove_pointer_t<decltype(g)>;
        return launch_overlapped(adamw_norm_kernel<G>, dim3(ctas), kAdamThreads, 0, s, 1, !first, list, grad_scale, parts + n_parts);
      });
      if (rc != cudaSuccess || cudaGetLastError() != cudaSuccess) return -5;
      n_parts += ctas;
      first = false;
    }
  if (clip > 0.f && n_parts == 0 && cudaMemsetAsync(norm, 0, 4, s) != cudaSuccess) return -5;
  if (launch_overlapped(adamw_prepare_kernel, dim3(1), 256, 0, s, 1, !first, static_cast<const double*>(parts), n_parts, step, beta1, beta2,
                        grad_scale, clip, factor, uint32_t(seed), norm, words, shared) != cudaSuccess || cudaGetLastError() != cudaSuccess)
    return -5;
  const AdamScalars scalars = {lr, float(beta1), float(1.0 - beta1), float(beta2), float(1.0 - beta2), eps, wd};
  for (int base = 0; base < n_tensors;) {
    base += fill(list, base);
    const int chunks = list.first_chunk[list.n];
    if (chunks == 0) continue;
    const cudaError_t rc = by_type(param_type, [&](auto* p) {
      using P = std::remove_pointer_t<decltype(p)>;
      return by_type(grad_type, [&](auto* g) {
        using G = std::remove_pointer_t<decltype(g)>;
        const auto launch = [&](auto kernel) {
          return launch_overlapped(kernel, dim3(std::min(chunks, 148 * (eight ? 3 : 8))), kAdamThreads, 0, s, 1, true, list, scalars, static_cast<const AdamShared*>(shared));
        };
        if constexpr (std::is_same_v<P, float>) {
          if (!has_master) return eight ? launch(adamw_multi_kernel<P, G, false, true>) : launch(adamw_multi_kernel<P, G, false, false>);
        }
        return eight ? launch(adamw_multi_kernel<P, G, true, true>) : launch(adamw_multi_kernel<P, G, true, false>);
      });
    });
    if (rc != cudaSuccess || cudaGetLastError() != cudaSuccess) return -5;
  }
  return 0;
}
