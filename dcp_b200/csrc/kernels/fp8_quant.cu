// Makers of 8-bit codes (see fp8_common.cuh), all bound by HBM in bf16 and fp32 rows on 16 bytes: 16384 x 4096 bf16 with a
// residual 72 us (6.6 TB/s; copying runs at 6.55), its backward with an addition 81 (6.7), by rows 31 (6.4), by blocks 30
// (6.7); both ways at once 48 (5.6: 80 registers leave three CTAs to an SM, 36 % of its warps, which do not cover two barriers
// and a walk through shared memory; 61 % of the issue slots are used).  Rows that do not begin on 16 bytes run at 2.7 to 3.6 TB/s,
// in fp32 at 2.8 to 4.8.
//
//  fp8_norm        h = x + residual, rounded to x's type; y = h * rsqrt(mean(h^2) + eps) * w as codes with a scale per 128
//                  channels.  One CTA per row, the row in registers: x and the residual are read once, h and the codes written
//                  once, and y is rounded once, from fp32.
//  fp8_norm_bwd    dx = rstd * (g - xh * mean(g * xh)) + add with xh = h * rstd, g = dy * w;  dw = sum over rows of dy * xh
//  fp8_quantize    codes of a matrix with a scale per 1 x 128, 128 x 1 or 128 x 128 block, or both of the first two from one
//                  pass: a CTA holds a tile of 128 x 128 in registers
//
// A thread has eight neighbouring channels (see fp8_common.cuh for rows that do not begin on 16 bytes), sixteen threads a
// block of 128.  Packed arithmetic where there is some: with one instruction per value the norm of bf16 rows was bound by
// issuing (27 instructions per value; 16384 x 4096 with a residual 89 us, fp32 rows of twice the bytes 135).
#include <algorithm>

#include "entries.h"
#include "fp8_common.cuh"
#include "launch.cuh"
#include "ptx.cuh"
#include "smem_limit.h"

namespace dcpk {

static constexpr int kBlock = 128;

// rows of codes begin on 16 bytes and have room for whole chunks
__device__ __forceinline__ void store_codes(uint8_t* row, int chunk, int width, const uint2& codes) {
  if (chunk * 8 < width) *reinterpret_cast<uint2*>(row + chunk * 8) = codes;
}
__device__ __forceinline__ uint32_t max_of_16(uint32_t m) {
#pragma unroll
  for (int s = 8; s > 0; s >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, s));
  return m;
}
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  return v;
}
__device__ __forceinline__ float row_sum(float v, float* scratch, int warps) {
  v = lanes_sum(v);
  const int lane = threadIdx.x & 31;
  if (lane == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  return lanes_sum(lane < warps ? scratch[lane] : 0.f);
}

static constexpr int kNormThreads = 512;
static constexpr int kNormWidth = 16384;   // four chunks of eight channels per thread at most
static constexpr int kMaxStages = 8;       // rows under way in the backward pass
static constexpr int kRingBytes = 200 * 1024;   // of an SM's shared memory, for all its CTAs

// kWarps: a row per warp, eight to a CTA, where a row's chunks are few: no barrier, and a CTA per row of 512 channels is bound by
// the CTAs' coming and going (65536 rows with a residual 70 us).
template <typename T, int kVecs, bool kAligned, int kCode, bool kWarps>
__global__ void __launch_bounds__(kNormThreads)
fp8_norm_kernel(const T* x, long x_pitch, const T* residual, long residual_pitch, const T* w,
                T* h, uint8_t* codes, long code_pitch, uint8_t* scales, long scale_pitch,
                float* rstd, int n_rows, int width, float eps) {
  __shared__ float scratch[kNormThreads / 32];
  constexpr int kTop = kCode == kCodeE4m3 ? 8 : 15;
  const long row = kWarps ? long(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (kWarps && row >= n_rows) return;
  const int first = kWarps ? threadIdx.x & 31 : threadIdx.x, step = kWarps ? 32 : blockDim.x;
  Raw8<T> v[kVecs];
  grid_wait();
#pragma unroll
  for (int i = 0; i < kVecs; ++i) load_chunk<kAligned>(x + row * x_pitch, first + i * step, width, v[i]);
  if (residual) {
    // the sum goes on in x's type: what the norm sees is what the next layer adds to
    Raw8<T> r[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) load_chunk<kAligned>(residual + row * residual_pitch, first + i * step, width, r[i]);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      v[i] = add_raw(v[i], r[i]);
      store_chunk<kAligned>(h + row * width, first + i * step, width, v[i]);
    }
  }
  grid_let_next();
  uint64_t ss2[2] = {0ull, 0ull};
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    uint64_t f[4];
    widen(v[i], f);
#pragma unroll
    for (int j = 0; j < 4; ++j) ss2[j & 1] = fma_f32x2(f[j], f[j], ss2[j & 1]);
  }
  float lo, hi;
  unpack_f32x2(add_f32x2(ss2[0], ss2[1]), lo, hi);
  const float r = rsqrtf((kWarps ? lanes_sum(lo + hi) : row_sum(lo + hi, scratch, blockDim.x >> 5)) / width + eps);
  if (first == 0) rstd[row] = r;
  const uint64_t r2 = pack_f32x2(r, r);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int chunk = first + i * step;
    Raw8<T> wr;
    uint64_t f[4], g[4];
    load_chunk<kAligned>(w, chunk, width, wr);
    widen(v[i], f);
    widen(wr, g);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = mul_f32x2(mul_f32x2(f[j], r2), g[j]);
    const int byte = scale_byte<kTop>(max_of_16(amax_bits(f)));
    store_codes(codes + row * code_pitch, chunk, width, to_codes8<kCode>(f, scale_inverse(byte)));
    if ((chunk & 15) == 0 && chunk * 8 < width) scales[row * scale_pitch + (chunk >> 4)] = uint8_t(byte);
  }
}

// Persistent CTAs: each walks rows blockIdx.x, + gridDim.x, ... and keeps its part of dW in registers; the parts go to
// `part` [gridDim.x, width], which a second kernel adds up in order: the same bits in every run.
//
// kRing: the rows of h, dy and add come by bulk copies into a ring of `stages` rows in shared memory, so
// that what is under way does not depend on the registers; the barrier inside the row's sum is also what frees the stage.
// With plain loads at the beginning of a row 5003 rows of 5120 took 62 us (2.9 TB/s).
template <typename T, int kVecs, bool kAligned, bool kRing, bool kAdd>
__global__ void __launch_bounds__(kVecs == 1 ? 1024 : kVecs == 2 ? 768 : 512)   // 64, 80 and 128 registers
fp8_norm_bwd_kernel(const T* h, long h_pitch, const T* w, const float* rstd, const T* dy,
                    long dy_pitch, const T* add, long add_pitch, T* dx, float* part, int n_rows,
                    int width, int stages, int* status) {
  __shared__ float scratch[2][kNormThreads / 32];
  __shared__ uint64_t full[kMaxStages];
  __shared__ int abort_word;
  extern __shared__ __align__(128) uint8_t ring[];
  // a row in the ring: the aligned pieces of 16 bytes that hold some of it, from its offset in the first on
  const uint32_t row_bytes = uint32_t(width) * sizeof(T), slot_bytes = kAligned ? row_bytes : (row_bytes + 45) & ~15u,
                 stage_bytes = slot_bytes * (kAdd ? 3 : 2);
  const auto past = [](const T* p) { return uint32_t(reinterpret_cast<uintptr_t>(p)) & 15u; };
  uint64_t dw[kVecs][4];
  Raw8<T> wv[kVecs];
  if (kRing) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < stages; ++i) mbar_init(&full[i], 1);
      abort_word = 0;
      mbar_fence_init();
    }
    __syncthreads();
  }
  grid_wait();
  const auto fetch = [&](long row, int stage) {   // by one thread
    if (row >= n_rows) return;
    const T* from[3] = {h + row * h_pitch, dy + row * dy_pitch, add + row * add_pitch};
    uint32_t bytes[3], total = 0;
#pragma unroll
    for (int i = 0; i < (kAdd ? 3 : 2); ++i) total += bytes[i] = kAligned ? row_bytes : (past(from[i]) + row_bytes + 15) & ~15u;
    mbar_expect_tx(&full[stage], total);
#pragma unroll
    for (int i = 0; i < (kAdd ? 3 : 2); ++i)
      bulk_load(ring + size_t(stage) * stage_bytes + i * slot_bytes, reinterpret_cast<const uint8_t*>(from[i]) - past(from[i]), bytes[i], &full[stage]);
  };
  if (kRing && threadIdx.x == 0)
    for (int i = 0; i < stages; ++i) fetch(blockIdx.x + long(i) * gridDim.x, i);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    load_chunk<kAligned>(w, threadIdx.x + i * blockDim.x, width, wv[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) dw[i][j] = 0ull;
  }
  int turn = 0, stage = 0, parity = 0;
  bool ok = true;
  for (long row = blockIdx.x; row < n_rows; row += gridDim.x, turn ^= 1) {
    const float r = rstd[row];
    const uint64_t r2 = pack_f32x2(r, r);
    uint64_t xh[kVecs][4], g[kVecs][4];
    const T *hr = h + row * h_pitch, *gr = dy + row * dy_pitch, *ar = add + row * add_pitch;
    if (kRing) {
      ok = ok && mbar_wait(&full[stage], parity, &abort_word);
      const uint8_t* at = ring + size_t(stage) * stage_bytes;
      hr = reinterpret_cast<const T*>(at + past(hr));
      gr = reinterpret_cast<const T*>(at + slot_bytes + past(gr));
      ar = reinterpret_cast<const T*>(at + 2 * slot_bytes + past(ar));
    }
    uint64_t dot2[2] = {0ull, 0ull};
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int chunk = threadIdx.x + i * blockDim.x;
      Raw8<T> raw;
      uint64_t wf[4];
      load_chunk<kAligned>(hr, chunk, width, raw);
      widen(raw, xh[i]);
      load_chunk<kAligned>(gr, chunk, width, raw);
      widen(raw, g[i]);
      widen(wv[i], wf);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        xh[i][j] = mul_f32x2(xh[i][j], r2);
        dw[i][j] = fma_f32x2(g[i][j], xh[i][j], dw[i][j]);
        g[i][j] = mul_f32x2(g[i][j], wf[j]);
        dot2[j & 1] = fma_f32x2(g[i][j], xh[i][j], dot2[j & 1]);
      }
    }
    float lo, hi;
    unpack_f32x2(add_f32x2(dot2[0], dot2[1]), lo, hi);
    const float dot = row_sum(lo + hi, scratch[turn], blockDim.x >> 5) / width;   // alternating scratch: one barrier per row
    if (kRing) {
      // all are through with the row before: its stage is free
      const int before = stage == 0 ? stages - 1 : stage - 1;
      if (threadIdx.x == 0 && row != blockIdx.x) fetch(row + long(stages - 1) * gridDim.x, before);
      if (++stage == stages) { stage = 0; parity ^= 1; }
    }
    const uint64_t minus = pack_f32x2(-dot, -dot);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int chunk = threadIdx.x + i * blockDim.x;
      uint64_t a[4] = {0ull, 0ull, 0ull, 0ull};
      if (kAdd) {
        Raw8<T> raw;
        load_chunk<kAligned>(ar, chunk, width, raw);
        widen(raw, a);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t t = fma_f32x2(xh[i][j], minus, g[i][j]);
        g[i][j] = kAdd ? fma_f32x2(t, r2, a[j]) : mul_f32x2(t, r2);
      }
      store_chunk<kAligned>(dx + row * width, chunk, width, narrow<T>(g[i]));
    }
  }
  grid_let_next();
#pragma unroll
  for (int i = 0; i < kVecs; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = (threadIdx.x + i * blockDim.x) * 8 + 2 * j;
      float lo, hi;
      unpack_f32x2(dw[i][j], lo, hi);
      float* to = part + size_t(blockIdx.x) * width + c;
      if (c < width) to[0] = lo;
      if (c + 1 < width) to[1] = hi;
    }
  if (kRing && !ok) {   // copies under way get a millisecond to land
    atomicExch(status, kStatusBarrierTimeout);
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
}

// 32 columns per CTA, 32 threads of a column take every 32nd of the parts
__global__ void __launch_bounds__(1024) fp8_norm_dw_kernel(const float* part, float* dw, int n, int width) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  grid_wait();
  if (c < width)
#pragma unroll 8
    for (int i = group; i < n; i += 32) s += part[size_t(i) * width + c];
  sums[group][lane] = s;
  __syncthreads();
  s = lanes_sum(sums[lane][group]);   // a warp per column
  const int mine = blockIdx.x * 32 + group;
  if (lane == 0 && mine < width) dw[mine] = s;
}

enum : int { kRows = 1, kCols = 2, kBlocks = 4 };

struct QuantizeOut {
  uint8_t* codes;
  uint8_t* scales;
  long pitch, scale_pitch;   // of cols: scales[column * scale_pitch + tile row]
};

// Eight values as they lie in memory and their magnitudes, two to a word in 16-bit types: magnitudes order like their bits
// there too, so one instruction masks two and one compares two.
template <typename T> struct Magnitudes { uint32_t m[kWordsOf<T>]; };

template <typename T>
__device__ __forceinline__ Magnitudes<T> magnitudes(const Raw8<T>& r) {
  constexpr uint32_t kMask = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu;
  Magnitudes<T> m;
#pragma unroll
  for (int i = 0; i < kWordsOf<T>; ++i) m.m[i] = r.w[i] & kMask;
  return m;
}
template <typename T>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {   // of each half in 16-bit types
  if (sizeof(T) == 4) return max(a, b);
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <typename T> __device__ __forceinline__ uint32_t as_float_bits(uint32_t m);   // of a magnitude in the low bits
template <> __device__ __forceinline__ uint32_t as_float_bits<float>(uint32_t m) { return m; }
template <> __device__ __forceinline__ uint32_t as_float_bits<__nv_bfloat16>(uint32_t m) { return m << 16; }
template <> __device__ __forceinline__ uint32_t as_float_bits<__half>(uint32_t m) {
  return __float_as_uint(__half2float(__ushort_as_half(uint16_t(m))));
}

// Bound by HBM where rows begin on 16 bytes.  The tile stays packed, so that the registers of four CTAs (two in fp32) fit an
// SM and their loads, maxima and stores overlap.
template <typename T, int kWays, bool kAligned, int kCode>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 2 : kWays == 3 ? 3 : 4)
fp8_quantize_kernel(const T* x, long pitch, QuantizeOut by_rows, QuantizeOut by_cols, int n_rows, int width, int tiles_x) {
  constexpr int kTop = kCode == kCodeE4m3 ? 8 : 15;
  constexpr int kWords = sizeof(Magnitudes<T>) / 4, kPer = 8 / kWords;   // values to a word
  __shared__ uint32_t column_max[(kWays & kCols) ? 16 : 1][kBlock / kPer + 4];
  __shared__ float column_inv[(kWays & kCols) ? kBlock : 1];
  __shared__ uint32_t warp_max[8];
  const int tile_x = blockIdx.x % tiles_x, tile_y = blockIdx.x / tiles_x;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, chunk = tile_x * 16 + tx;
  const int row0 = tile_y * kBlock + ty, rows_left = n_rows - row0;   // thread's rows: row0 + 16 i, i < 8
  Raw8<T> v[8];
  grid_wait();
  {
    const T* p = x + row0 * pitch;
#pragma unroll
    for (int i = 0; i < 8; ++i, p += 16 * pitch) {
      if (16 * i < rows_left) load_chunk<kAligned>(p, chunk, width, v[i]);
      else v[i] = Raw8<T>{};
    }
  }
  grid_let_next();
  if (kWays & kCols) {
    Magnitudes<T> m = magnitudes(v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      const Magnitudes<T> n = magnitudes(v[i]);
#pragma unroll
      for (int k = 0; k < kWords; ++k) m.m[k] = larger<T>(m.m[k], n.m[k]);
    }
    // word tx + 16 k: of channels in the order the threads hold them
#pragma unroll
    for (int k = 0; k < kWords; ++k) column_max[ty][tx + 16 * k] = m.m[k];
    __syncthreads();
    if (threadIdx.x < kBlock) {
      const int t = threadIdx.x & 15, j = threadIdx.x >> 4;   // the j-th value of thread t
      uint32_t amax = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = larger<T>(amax, column_max[i][t + 16 * (j / kPer)]);
      if (sizeof(T) == 2) amax = j & 1 ? amax >> 16 : amax & 0xffffu;
      const int byte = scale_byte<kTop>(as_float_bits<T>(amax)), c = tile_x * kBlock + t * 8 + j;
      if (c < width) by_cols.scales[c * by_cols.scale_pitch + tile_y] = uint8_t(byte);
      column_inv[t + 16 * j] = scale_inverse(byte);
    }
  }
  if (kWays & kRows) {
    uint8_t* to = by_rows.codes + row0 * by_rows.pitch;
    uint8_t* scale = by_rows.scales + row0 * by_rows.scale_pitch + tile_x;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {   // two rows at a time: in 16-bit types their maxima share a word
      uint32_t m[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const Magnitudes<T> n = magnitudes(v[i + h]);
        m[h] = n.m[0];
#pragma unroll
        for (int k = 1; k < kWords; ++k) m[h] = larger<T>(m[h], n.m[k]);
      }
      if (sizeof(T) == 2) {
        uint32_t both = larger<T>(__byte_perm(m[0], m[1], 0x5410), __byte_perm(m[0], m[1], 0x7632));
#pragma unroll
        for (int s = 8; s > 0; s >>= 1) both = larger<T>(both, __shfl_xor_sync(0xffffffffu, both, s));
        m[0] = both & 0xffffu;
        m[1] = both >> 16;
      } else {
        m[0] = max_of_16(m[0]);
        m[1] = max_of_16(m[1]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h, to += 16 * by_rows.pitch, scale += 16 * by_rows.scale_pitch) {
        if (16 * (i + h) >= rows_left) continue;
        const int byte = scale_byte<kTop>(as_float_bits<T>(m[h]));
        uint64_t f[4];
        widen(v[i + h], f);
        store_codes(to, chunk, width, to_codes8<kCode>(f, scale_inverse(byte)));
        if (tx == 0) *scale = uint8_t(byte);
      }
    }
  }
  if (kWays & kBlocks) {
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const Magnitudes<T> n = magnitudes(v[i]);
#pragma unroll
      for (int k = 0; k < kWords; ++k) amax = larger<T>(amax, n.m[k]);
    }
    if (sizeof(T) == 2) amax = max(amax >> 16, amax & 0xffffu);
    amax = __reduce_max_sync(0xffffffffu, amax);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = amax;
    __syncthreads();
    amax = warp_max[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) amax = max(amax, warp_max[i]);
    const int byte = scale_byte<kTop>(as_float_bits<T>(amax));
    const float inv = scale_inverse(byte);
    uint8_t* to = by_rows.codes + row0 * by_rows.pitch;
#pragma unroll
    for (int i = 0; i < 8; ++i, to += 16 * by_rows.pitch) {
      if (16 * i >= rows_left) continue;
      uint64_t f[4];
      widen(v[i], f);
      store_codes(to, chunk, width, to_codes8<kCode>(f, inv));
    }
    if (threadIdx.x == 0) by_rows.scales[tile_y * by_rows.scale_pitch + tile_x] = uint8_t(byte);
  }
  if (kWays & kCols) {
    __syncthreads();
    uint64_t inv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) inv[j] = pack_f32x2(column_inv[tx + 32 * j], column_inv[tx + 32 * j + 16]);
    uint8_t* to = by_cols.codes + row0 * by_cols.pitch;
#pragma unroll
    for (int i = 0; i < 8; ++i, to += 16 * by_cols.pitch) {
      if (16 * i >= rows_left) continue;
      uint64_t f[4];
      widen(v[i], f);
      store_codes(to, chunk, width, to_codes8<kCode>(f, inv));
    }
  }
}

// Codes of other layouts into rows that begin on 16 bytes, as products read them: both operands of one in a launch.  A thread makes
// chunks of 16 from the aligned pieces that hold some of them, four rows at a time.  A product of 200 x 300 x 391 takes 12 us so and
// 9 with codes that begin on 16 bytes (43 with the layout by a call per operand), 16384 x 4096 x 14337 1092 and 881.
struct AlignJob {
  const uint8_t* from;
  uint8_t* to;
  long pitch;
  int n_rows, width;
};
struct AlignJobs { AlignJob job[2]; };

static constexpr int kAlignRows = 32;   // of a CTA: 8 warps, four rows each

__global__ void __launch_bounds__(256) fp8_align_kernel(const __grid_constant__ AlignJobs jobs) {
  const AlignJob& j = jobs.job[blockIdx.z];
  const int chunk = blockIdx.x * 32 + (threadIdx.x & 31), at = chunk * 16;
  const long to_pitch = (j.width + 15l) & ~15l;
  grid_wait();
  grid_let_next();
  if (chunk > (j.width - 1) >> 4) return;
  for (long row0 = long(blockIdx.y) * kAlignRows + (threadIdx.x >> 5); row0 < j.n_rows; row0 += long(gridDim.y) * kAlignRows) {
    uint32_t w[4][8], past[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long row = min(row0 + 8 * i, j.n_rows - 1l);
      const uint8_t *begin = j.from + row * j.pitch + at, *end = begin + (j.width - at);
      past[i] = uint32_t(reinterpret_cast<uintptr_t>(begin)) & 15u;
      const uint4* piece = reinterpret_cast<const uint4*>(begin - past[i]);
      const uint4 a = piece[0], b = reinterpret_cast<const uint8_t*>(piece + 1) < end ? piece[1] : make_uint4(0, 0, 0, 0);
      w[i][0] = a.x; w[i][1] = a.y; w[i][2] = a.z; w[i][3] = a.w;
      w[i][4] = b.x; w[i][5] = b.y; w[i][6] = b.z; w[i][7] = b.w;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      shift_words(w[i], past[i]);
      if (past[i] & 1)
#pragma unroll
        for (int k = 0; k < 4; ++k) w[i][k] = __funnelshift_r(w[i][k], w[i][k + 1], 8);
      if (row0 + 8 * i < j.n_rows)
        *reinterpret_cast<uint4*>(j.to + (row0 + 8 * i) * to_pitch + at) = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
    }
  }
}

template <typename F>
static int by_type(int type, F f) {
  return type == kTypeBf16 ? f(static_cast<const __nv_bfloat16*>(nullptr)) : type == kTypeF16 ? f(static_cast<const __half*>(nullptr))
       : type == kTypeF32 ? f(static_cast<const float*>(nullptr)) : -3;
}
static bool on_16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// chunks of 8 channels a row takes, in whole blocks of 128, and the threads for them at `vecs` chunks each
static int chunks_of(int width) { return (width + kBlock - 1) / kBlock * 16; }
static int threads_for(int width, int vecs) { return ((chunks_of(width) + vecs - 1) / vecs + 31) / 32 * 32; }

}  // namespace dcpk

using namespace dcpk;

// x, residual (or null), w, h (written where there is a residual) of one type; pitches in elements (h: width), of codes and
// scales in bytes
extern "C" int dcpk_fp8_norm(int type, int code, const void* x, long x_pitch, const void* residual, long residual_pitch, const void* w,
                             void* h, void* codes, long code_pitch, void* scales, long scale_pitch, float* rstd, long n_rows, int width,
                             float eps, void* stream) {
  if (n_rows <= 0) return 0;
  if (width <= 0 || width > kNormWidth || n_rows > 0x7fffffffl || (code != kCodeE4m3 && code != kCodeE5m2)) return -3;
  const bool aligned = width % 8 == 0 && x_pitch % 8 == 0 && on_16(x) && on_16(w) && (!residual || (residual_pitch % 8 == 0 && on_16(residual) && on_16(h))) &&
                       code_pitch % 16 == 0 && on_16(codes);
  // Rows of up to 1024 channels: a warp each (up to 256 where they do not begin on 16 bytes: 16384 x 1001 45 us against 38).  Few
  // longer rows: as many threads per row as it takes, for the shortest chain.
  const bool warps = width <= (aligned ? 1024 : 256);
  int vecs = n_rows <= 148 * 2 ? 1 : 4;
  while (vecs > 1 && threads_for(width, vecs) < 64) vecs >>= 1;
  while (threads_for(width, vecs) > kNormThreads) vecs <<= 1;
  if (warps) {
    vecs = 1;
    while (threads_for(width, vecs) > 32) vecs <<= 1;
  }
  const unsigned ctas = unsigned(warps ? (n_rows + 7) / 8 : n_rows), threads = warps ? 256 : threads_for(width, vecs);
  return by_type(type, [&](auto* t) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
    const auto launch = [&](auto kernel) {
      const cudaError_t rc = launch_overlapped(
          kernel, dim3(ctas), threads, 0, static_cast<cudaStream_t>(stream), 1, true, static_cast<const T*>(x),
          x_pitch, static_cast<const T*>(residual), residual_pitch, static_cast<const T*>(w), static_cast<T*>(h), static_cast<uint8_t*>(codes),
          code_pitch, static_cast<uint8_t*>(scales), scale_pitch, rstd, int(n_rows), width, eps);
      return rc == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -5;
    };
    const auto sized = [&](auto al, auto c) {
      constexpr bool A = decltype(al)::value;
      constexpr int C = decltype(c)::value;
      if (warps)
        return vecs == 1 ? launch(fp8_norm_kernel<T, 1, A, C, true>) : vecs == 2 ? launch(fp8_norm_kernel<T, 2, A, C, true>)
                                                                                : launch(fp8_norm_kernel<T, 4, A, C, true>);
      return vecs == 1 ? launch(fp8_norm_kernel<T, 1, A, C, false>) : vecs == 2 ? launch(fp8_norm_kernel<T, 2, A, C, false>)
                                                                               : launch(fp8_norm_kernel<T, 4, A, C, false>);
    };
    const auto coded = [&](auto al) {
      return code == kCodeE4m3 ? sized(al, std::integral_constant<int, kCodeE4m3>()) : sized(al, std::integral_constant<int, kCodeE5m2>());
    };
    return aligned ? coded(std::true_type()) : coded(std::false_type());
  });
}

// CTAs of the backward pass to an SM: as many threads as the registers allow at two chunks each, with three rows under way per
// CTA (16384 x 4096 in fp32 with three CTAs and no room for a ring 224 us, with one 152; bf16 with three CTAs of two rows 85, with
// two of four 80).  Two rows where they do not begin on 16 bytes, which takes more threads' work (fp32 one CTA 374 us, two 228).
static int norm_bwd_per_sm(int type, int width, bool add) {
  const int row = width * (type == kTypeF32 ? 4 : 2) + 45, rows = (width % 8 ? 2 : 3) * (add ? 3 : 2);
  return std::max(1, std::min({8, 768 / threads_for(width, 2), kRingBytes / (rows * row)}));
}
// CTAs in all, which is also how many rows of `width` floats `part` has
extern "C" int dcpk_fp8_norm_bwd_parts(int type, long n_rows, int width, int add) {
  return int(std::max(1l, std::min(n_rows, 148l * norm_bwd_per_sm(type, width, add))));
}

static std::atomic<uint64_t> g_ring_raised[36];

// dx [n_rows, width]; dw fp32 [width], written; add: null, or what is added to dx
extern "C" int dcpk_fp8_norm_bwd(int type, const void* h, long h_pitch, const void* w, const float* rstd, const void* dy, long dy_pitch,
                                 const void* add, long add_pitch, void* dx, float* dw, float* part, long n_rows, int width, int* status,
                                 void* stream) {
  if (width <= 0 || width > kNormWidth || n_rows > 0x7fffffffl || n_rows < 0) return -3;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n_rows == 0) return cudaMemsetAsync(dw, 0, size_t(width) * 4, s) == cudaSuccess ? 0 : -5;
  const bool aligned = width % 8 == 0 && h_pitch % 8 == 0 && dy_pitch % 8 == 0 && on_16(h) && on_16(w) && on_16(dy) && on_16(dx) &&
                       (!add || (add_pitch % 8 == 0 && on_16(add)));
  const int ctas = dcpk_fp8_norm_bwd_parts(type, n_rows, width, add != nullptr);
  int vecs = threads_for(width, 2) <= 256 && threads_for(width, 1) <= 128 ? 1 : 2;
  while (threads_for(width, vecs) > kNormThreads) vecs <<= 1;
  const int rc = by_type(type, [&](auto* t) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
    const int row_bytes = width * int(sizeof(T)), stage_bytes = (aligned ? row_bytes : (row_bytes + 45) & ~15) * (add ? 3 : 2);
    const int stages = std::min(kMaxStages, kRingBytes / norm_bwd_per_sm(type, width, add != nullptr) / stage_bytes);
    const bool ring = stages >= 2;   // not for long rows of fp32
    const auto launch = [&](auto kernel, int slot) {
      const int smem = ring ? stages * stage_bytes : 0;
      if (smem > 48 * 1024 - 512 && raise_smem_limit(kernel, kRingBytes, g_ring_raised[slot]) != cudaSuccess) return -4;
      const cudaError_t rc = launch_overlapped(kernel, dim3(ctas), threads_for(width, vecs), smem, s, 1, true, static_cast<const T*>(h), h_pitch,
                                               static_cast<const T*>(w), rstd, static_cast<const T*>(dy), dy_pitch, static_cast<const T*>(add),
                                               add_pitch, static_cast<T*>(dx), part, int(n_rows), width, stages, status);
      return rc == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -5;
    };
    const auto sized = [&](auto al, auto ri, auto ad) {
      constexpr bool A = decltype(al)::value, R = decltype(ri)::value, D = decltype(ad)::value;
      constexpr int base = (std::is_same_v<T, float> ? 0 : std::is_same_v<T, __half> ? 12 : 24) + (A * 2 + D) * 3;
      return vecs == 1 ? launch(fp8_norm_bwd_kernel<T, 1, A, R, D>, base) : vecs == 2 ? launch(fp8_norm_bwd_kernel<T, 2, A, R, D>, base + 1)
                                                                                     : launch(fp8_norm_bwd_kernel<T, 4, A, R, D>, base + 2);
    };
    const auto added = [&](auto al, auto ri) { return add ? sized(al, ri, std::true_type()) : sized(al, ri, std::false_type()); };
    return !ring ? added(std::false_type(), std::false_type()) : aligned ? added(std::true_type(), std::true_type()) : added(std::false_type(), std::true_type());
  });
  if (rc) return rc;
  const cudaError_t rc2 = launch_overlapped(fp8_norm_dw_kernel, dim3((width + 31) / 32), 1024, 0, s, 1, true, static_cast<const float*>(part), dw, ctas, width);
  return rc2 == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -5;
}

// ways: 1 a scale per 1 x 128, 2 per 128 x 1, 3 both, 4 per 128 x 128; codes_a / scales_a of ways 1 and 4, codes_b / scales_b of
// way 2 (scales_b[column * pitch + row / 128])
extern "C" int dcpk_fp8_quantize(int type, int code, int ways, const void* x, long pitch, void* codes_a, long pitch_a, void* scales_a,
                                 long scale_pitch_a, void* codes_b, long pitch_b, void* scales_b, long scale_pitch_b, long n_rows, int width,
                                 void* stream) {
  if (n_rows <= 0 || width <= 0) return 0;
  const long tiles_x = (width + kBlock - 1) / kBlock, tiles = tiles_x * ((n_rows + kBlock - 1) / kBlock);
  if (tiles > 0x7fffffffl || n_rows > 0x7fffffffl || (ways != 1 && ways != 2 && ways != 3 && ways != 4) || (code != kCodeE4m3 && code != kCodeE5m2))
    return -3;
  const QuantizeOut a = {static_cast<uint8_t*>(codes_a), static_cast<uint8_t*>(scales_a), pitch_a, scale_pitch_a};
  const QuantizeOut b = {static_cast<uint8_t*>(codes_b), static_cast<uint8_t*>(scales_b), pitch_b, scale_pitch_b};
  const bool aligned = width % 8 == 0 && pitch % 8 == 0 && on_16(x) && (ways == 2 || (pitch_a % 16 == 0 && on_16(codes_a))) &&
                       (!(ways & 2) || (pitch_b % 16 == 0 && on_16(codes_b)));
  return by_type(type, [&](auto* t) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
    const auto launch = [&](auto kernel) {
      const cudaError_t rc = launch_overlapped(kernel, dim3(unsigned(tiles)), 256, 0, static_cast<cudaStream_t>(stream), 1, true,
                                               static_cast<const T*>(x), pitch, a, b, int(n_rows), width, int(tiles_x));
      return rc == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -5;
    };
    const auto coded = [&](auto w, auto al) {
      constexpr int W = decltype(w)::value;
      constexpr bool A = decltype(al)::value;
      return code == kCodeE4m3 ? launch(fp8_quantize_kernel<T, W, A, kCodeE4m3>) : launch(fp8_quantize_kernel<T, W, A, kCodeE5m2>);
    };
    const auto way = [&](auto al) {
      return ways == 1 ? coded(std::integral_constant<int, 1>(), al) : ways == 2 ? coded(std::integral_constant<int, 2>(), al)
           : ways == 3 ? coded(std::integral_constant<int, 3>(), al) : coded(std::integral_constant<int, 4>(), al);
    };
    return aligned ? way(std::true_type()) : way(std::false_type());
  });
}

// The codes of up to two matrices into rows of whole 16 bytes (to_b null: one matrix)
extern "C" int dcpk_fp8_align(const void* from_a, long pitch_a, void* to_a, int rows_a, int width_a, const void* from_b, long pitch_b, void* to_b,
                              int rows_b, int width_b, void* stream) {
  if (rows_a <= 0 || width_a <= 0 || (to_b && (rows_b <= 0 || width_b <= 0)) || !on_16(to_a) || !on_16(to_b)) return -3;
  AlignJobs jobs = {{{static_cast<const uint8_t*>(from_a), static_cast<uint8_t*>(to_a), pitch_a, rows_a, width_a},
                     {static_cast<const uint8_t*>(from_b), static_cast<uint8_t*>(to_b), pitch_b, to_b ? rows_b : 0, to_b ? width_b : 0}}};
  const int rows = std::max(rows_a, jobs.job[1].n_rows), width = std::max(width_a, jobs.job[1].width);
  const dim3 grid((width - 1) / 512 + 1, std::min((rows - 1) / kAlignRows + 1, 65535), to_b ? 2 : 1);
  const cudaError_t rc = launch_overlapped(fp8_align_kernel, grid, 256, 0, static_cast<cudaStream_t>(stream), 1, true, jobs);
  return rc == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -5;
}
