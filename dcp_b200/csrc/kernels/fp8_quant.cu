// Makers of 8-bit codes (see fp8_common.cuh), all bound by HBM.
//
//  fp8_norm        h = x + residual, rounded to x's type; y = h * rsqrt(mean(h^2) + eps) * w as codes with a scale per 128
//                  channels.  One CTA per row, the row in registers: x and the residual are read once, h and the codes written
//                  once, and y is rounded once, from fp32.
//  fp8_norm_bwd    dx = rstd * (g - xh * mean(g * xh)) + add with xh = h * rstd, g = dy * w;  dw = sum over rows of dy * xh
//  fp8_quantize    codes of a matrix with a scale per 1 x 128, 128 x 1 or 128 x 128 block, or both of the first two from one
//                  pass: a CTA holds a tile of 128 x 128 in registers
//
// A thread has eight neighbouring channels in 16-byte accesses where rows begin on 16 bytes and hold a multiple of eight
// values; otherwise every sixteenth channel of a block of 128, so that the 16 threads of a block still read and write
// neighbours.
#include <algorithm>

#include "fp8_common.cuh"
#include "launch.cuh"

namespace dcpk {

static constexpr int kBlock = 128;

__device__ __forceinline__ int column(bool aligned, int chunk, int j) {
  return aligned ? chunk * 8 + j : (chunk >> 4) * kBlock + j * 16 + (chunk & 15);
}
template <bool kAligned, typename T>
__device__ __forceinline__ void load_chunk(const T* row, int chunk, int width, float (&f)[8]) {
  if (kAligned) {
    if (chunk * 8 < width) {
      Raw8<T> raw;
      load_raw(raw, row + chunk * 8);
      widen(raw, f);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column(false, chunk, j);
      f[j] = c < width ? to_float(row[c]) : 0.f;
    }
  }
}
template <bool kAligned, typename T>
__device__ __forceinline__ void store_chunk(T* row, int chunk, int width, const float (&f)[8]) {
  if (kAligned) {
    if (chunk * 8 < width) store8(row + chunk * 8, f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column(false, chunk, j);
      if (c < width) row[c] = from_float<T>(f[j]);
    }
  }
}
// rows of codes begin on 16 bytes in any case
template <bool kAligned>
__device__ __forceinline__ void store_codes(uint8_t* row, int chunk, int width, const uint2& codes) {
  if (kAligned) {
    if (chunk * 8 < width) *reinterpret_cast<uint2*>(row + chunk * 8) = codes;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column(false, chunk, j);
      if (c < width) row[c] = uint8_t((j < 4 ? codes.x : codes.y) >> (8 * (j & 3)));
    }
  }
}
__device__ __forceinline__ uint32_t max_of_16(uint32_t m) {
#pragma unroll
  for (int s = 8; s > 0; s >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, s));
  return m;
}
__device__ __forceinline__ float row_sum(float v, float* scratch, int warps) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  const int lane = threadIdx.x & 31;
  if (lane == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < warps ? scratch[lane] : 0.f;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  return v;
}

static constexpr int kNormThreads = 512;
static constexpr int kNormWidth = 16384;   // four chunks of eight channels per thread at most

template <typename T, int kVecs, bool kAligned, int kCode>
__global__ void __launch_bounds__(kNormThreads)
fp8_norm_kernel(const T* __restrict__ x, long x_pitch, const T* __restrict__ residual, long residual_pitch, const T* __restrict__ w,
                T* __restrict__ h, uint8_t* __restrict__ codes, long code_pitch, uint8_t* __restrict__ scales, long scale_pitch,
                float* __restrict__ rstd, int width, float eps) {
  __shared__ float scratch[kNormThreads / 32];
  constexpr int kTop = kCode == kCodeE4m3 ? 8 : 15;
  const long row = blockIdx.x;
  float v[kVecs][8];
  float ss = 0.f;
  grid_wait();
#pragma unroll
  for (int i = 0; i < kVecs; ++i) load_chunk<kAligned>(x + row * x_pitch, threadIdx.x + i * blockDim.x, width, v[i]);
  if (residual) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      float r[8];
      const int chunk = threadIdx.x + i * blockDim.x;
      load_chunk<kAligned>(residual + row * residual_pitch, chunk, width, r);
      // the sum goes on in x's type: what the norm sees is what the next layer adds to
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = to_float(from_float<T>(v[i][j] + r[j]));
      store_chunk<kAligned>(h + row * width, chunk, width, v[i]);
    }
  }
  grid_let_next();
#pragma unroll
  for (int i = 0; i < kVecs; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += v[i][j] * v[i][j];
  ss = row_sum(ss, scratch, blockDim.x >> 5);
  const float r = rsqrtf(ss / width + eps);
  if (threadIdx.x == 0) rstd[row] = r;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int chunk = threadIdx.x + i * blockDim.x;
    float g[8];
    uint32_t amax = 0;
    load_chunk<kAligned>(w, chunk, width, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[i][j] = v[i][j] * r * g[j];
      amax = amax_bits(amax, v[i][j]);
    }
    const int byte = scale_byte<kTop>(max_of_16(amax));
    store_codes<kAligned>(codes + row * code_pitch, chunk, width, to_codes8<kCode>(v[i], scale_inverse(byte)));
    if ((chunk & 15) == 0 && chunk * 8 < width) scales[row * scale_pitch + (chunk >> 4)] = uint8_t(byte);
  }
}

// Persistent CTAs: each walks rows blockIdx.x, + gridDim.x, ... and keeps its part of dW in registers; the parts go to
// `part` [gridDim.x, width], which a second kernel adds up in order: the same bits in every run.  The next row's loads are
// under way while this one is summed.
template <typename T, int kVecs, bool kAligned, bool kAdd>
__global__ void __launch_bounds__(kNormThreads)
fp8_norm_bwd_kernel(const T* __restrict__ h, long h_pitch, const T* __restrict__ w, const float* __restrict__ rstd, const T* __restrict__ dy,
                    long dy_pitch, const T* __restrict__ add, long add_pitch, T* __restrict__ dx, float* __restrict__ part, int n_rows,
                    int width) {
  __shared__ float scratch[2][kNormThreads / 32];
  float wv[kVecs][8], dw[kVecs][8];
  float xh[kVecs][8], g[kVecs][8], a[kVecs][8];
  grid_wait();
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    load_chunk<kAligned>(w, threadIdx.x + i * blockDim.x, width, wv[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = 0.f;
  }
  int turn = 0;
  for (long row = blockIdx.x; row < n_rows; row += gridDim.x, turn ^= 1) {
    const float r = rstd[row];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int chunk = threadIdx.x + i * blockDim.x;
      load_chunk<kAligned>(h + row * h_pitch, chunk, width, xh[i]);
      load_chunk<kAligned>(dy + row * dy_pitch, chunk, width, g[i]);
      if (kAdd) load_chunk<kAligned>(add + row * add_pitch, chunk, width, a[i]);
    }
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xh[i][j] *= r;
        dw[i][j] += g[i][j] * xh[i][j];
        g[i][j] *= wv[i][j];
        dot += g[i][j] * xh[i][j];
      }
    dot = row_sum(dot, scratch[turn], blockDim.x >> 5) / width;   // alternating scratch: one barrier per row
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) g[i][j] = r * (g[i][j] - xh[i][j] * dot) + (kAdd ? a[i][j] : 0.f);
      store_chunk<kAligned>(dx + row * width, threadIdx.x + i * blockDim.x, width, g[i]);
    }
  }
  grid_let_next();
#pragma unroll
  for (int i = 0; i < kVecs; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column(kAligned, threadIdx.x + i * blockDim.x, j);
      if (c < width) part[size_t(blockIdx.x) * width + c] = dw[i][j];
    }
}

// 32 columns per CTA, eight threads of a column take every eighth of the parts
__global__ void __launch_bounds__(256) fp8_norm_dw_kernel(const float* __restrict__ part, float* __restrict__ dw, int n, int width) {
  __shared__ float sums[8][32];
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  grid_wait();
  if (c < width)
#pragma unroll 8
    for (int i = group; i < n; i += 8) s += part[size_t(i) * width + c];
  sums[group][lane] = s;
  __syncthreads();
  if (group == 0 && c < width) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += sums[i][lane];
    dw[c] = s;
  }
}

enum : int { kRows = 1, kCols = 2, kBlocks = 4 };

struct QuantizeOut {
  uint8_t* codes;
  uint8_t* scales;
  long pitch, scale_pitch;   // of cols: scales[column * scale_pitch + tile row]
};

template <typename T, int kWays, bool kAligned, int kCode>
__global__ void __launch_bounds__(256)
fp8_quantize_kernel(const T* __restrict__ x, long pitch, QuantizeOut by_rows, QuantizeOut by_cols, int n_rows, int width, int tiles_x) {
  constexpr int kTop = kCode == kCodeE4m3 ? 8 : 15;
  __shared__ uint32_t column_max[(kWays & kCols) ? 16 : 1][kBlock + 8];
  __shared__ uint32_t warp_max[8];
  const int tile_x = blockIdx.x % tiles_x, tile_y = blockIdx.x / tiles_x;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, chunk = tile_x * 16 + tx;
  float v[8][8];
  grid_wait();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long row = long(tile_y) * kBlock + ty + 16 * i;
    if (row < n_rows) {
      load_chunk<kAligned>(x + row * pitch, chunk, width, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
  }
  grid_let_next();
  if (kWays & kRows) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long row = long(tile_y) * kBlock + ty + 16 * i;
      uint32_t amax = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = amax_bits(amax, v[i][j]);
      const int byte = scale_byte<kTop>(max_of_16(amax));
      if (row < n_rows) {
        store_codes<kAligned>(by_rows.codes + row * by_rows.pitch, chunk, width, to_codes8<kCode>(v[i], scale_inverse(byte)));
        if (tx == 0) by_rows.scales[row * by_rows.scale_pitch + tile_x] = uint8_t(byte);
      }
    }
  }
  if (kWays & kBlocks) {
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = amax_bits(amax, v[i][j]);
    amax = __reduce_max_sync(0xffffffffu, amax);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = amax;
    __syncthreads();
    amax = warp_max[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) amax = max(amax, warp_max[i]);
    const int byte = scale_byte<kTop>(amax);
    const float inv = scale_inverse(byte);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long row = long(tile_y) * kBlock + ty + 16 * i;
      if (row < n_rows) store_codes<kAligned>(by_rows.codes + row * by_rows.pitch, chunk, width, to_codes8<kCode>(v[i], inv));
    }
    if (threadIdx.x == 0) by_rows.scales[long(tile_y) * by_rows.scale_pitch + tile_x] = uint8_t(byte);
  }
  if (kWays & kCols) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t amax = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = amax_bits(amax, v[i][j]);
      column_max[ty][column(kAligned, tx, j)] = amax;
    }
    __syncthreads();
    if (threadIdx.x < kBlock) {
      uint32_t amax = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = max(amax, column_max[i][threadIdx.x]);
      const int byte = scale_byte<kTop>(amax), c = tile_x * kBlock + threadIdx.x;
      if (c < width) by_cols.scales[c * by_cols.scale_pitch + tile_y] = uint8_t(byte);
      column_max[0][threadIdx.x] = __float_as_uint(scale_inverse(byte));   // read by this thread alone so far
    }
    __syncthreads();
    float inv[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) inv[j] = __uint_as_float(column_max[0][column(kAligned, tx, j)]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long row = long(tile_y) * kBlock + ty + 16 * i;
      if (row >= n_rows) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= inv[j];
      store_codes<kAligned>(by_cols.codes + row * by_cols.pitch, chunk, width, to_codes8<kCode>(v[i], 1.f));
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
  // few rows: as many threads per row as it takes, for the shortest chain
  int vecs = n_rows <= 148 * 2 ? 1 : 4;
  while (vecs > 1 && threads_for(width, vecs) < 64) vecs >>= 1;
  while (threads_for(width, vecs) > kNormThreads) vecs <<= 1;
  return by_type(type, [&](auto* t) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
    const auto launch = [&](auto kernel) {
      const cudaError_t rc = launch_overlapped(
          kernel, dim3(unsigned(n_rows)), threads_for(width, vecs), 0, static_cast<cudaStream_t>(stream), 1, false, static_cast<const T*>(x),
          x_pitch, static_cast<const T*>(residual), residual_pitch, static_cast<const T*>(w), static_cast<T*>(h), static_cast<uint8_t*>(codes),
          code_pitch, static_cast<uint8_t*>(scales), scale_pitch, rstd, width, eps);
      return rc == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -5;
    };
    const auto sized = [&](auto al, auto c) {
      constexpr bool A = decltype(al)::value;
      constexpr int C = decltype(c)::value;
      return vecs == 1 ? launch(fp8_norm_kernel<T, 1, A, C>) : vecs == 2 ? launch(fp8_norm_kernel<T, 2, A, C>) : launch(fp8_norm_kernel<T, 4, A, C>);
    };
    const auto coded = [&](auto al) {
      return code == kCodeE4m3 ? sized(al, std::integral_constant<int, kCodeE4m3>()) : sized(al, std::integral_constant<int, kCodeE5m2>());
    };
    return aligned ? coded(std::true_type()) : coded(std::false_type());
  });
}

// CTAs of the backward pass, which is also how many rows of `width` floats `part` has
extern "C" int dcpk_fp8_norm_bwd_parts(long n_rows, int width) {
  const long most = threads_for(width, 2) <= 256 ? 148 * 4 : 148 * 2;
  return int(std::max(1l, std::min(n_rows, most)));
}

// dx [n_rows, width]; dw fp32 [width], written; add: null, or what is added to dx
extern "C" int dcpk_fp8_norm_bwd(int type, const void* h, long h_pitch, const void* w, const float* rstd, const void* dy, long dy_pitch,
                                 const void* add, long add_pitch, void* dx, float* dw, float* part, long n_rows, int width, void* stream) {
  if (width <= 0 || width > kNormWidth || n_rows > 0x7fffffffl || n_rows < 0) return -3;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n_rows == 0) return cudaMemsetAsync(dw, 0, size_t(width) * 4, s) == cudaSuccess ? 0 : -5;
  const bool aligned = width % 8 == 0 && h_pitch % 8 == 0 && dy_pitch % 8 == 0 && on_16(h) && on_16(w) && on_16(dy) && on_16(dx) &&
                       (!add || (add_pitch % 8 == 0 && on_16(add)));
  const int ctas = dcpk_fp8_norm_bwd_parts(n_rows, width);
  int vecs = 1;
  while (threads_for(width, vecs) > kNormThreads) vecs <<= 1;
  const int rc = by_type(type, [&](auto* t) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
    const auto launch = [&](auto kernel) {
      const cudaError_t rc = launch_overlapped(kernel, dim3(ctas), threads_for(width, vecs), 0, s, 1, false, static_cast<const T*>(h), h_pitch,
                                               static_cast<const T*>(w), rstd, static_cast<const T*>(dy), dy_pitch, static_cast<const T*>(add),
                                               add_pitch, static_cast<T*>(dx), part, int(n_rows), width);
      return rc == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -5;
    };
    const auto sized = [&](auto al, auto ad) {
      constexpr bool A = decltype(al)::value, D = decltype(ad)::value;
      return vecs == 1 ? launch(fp8_norm_bwd_kernel<T, 1, A, D>) : vecs == 2 ? launch(fp8_norm_bwd_kernel<T, 2, A, D>) : launch(fp8_norm_bwd_kernel<T, 4, A, D>);
    };
    const auto added = [&](auto al) { return add ? sized(al, std::true_type()) : sized(al, std::false_type()); };
    return aligned ? added(std::true_type()) : added(std::false_type());
  });
  if (rc) return rc;
  const cudaError_t rc2 = launch_overlapped(fp8_norm_dw_kernel, dim3((width + 31) / 32), 256, 0, s, 1, true, static_cast<const float*>(part), dw, ctas, width);
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
      const cudaError_t rc = launch_overlapped(kernel, dim3(unsigned(tiles)), 256, 0, static_cast<cudaStream_t>(stream), 1, false,
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
