// Products of 8-bit codes with a power-of-two scale per 128 values of the contraction.
//
//   out[q, p] = sum_k  a[q, k] sa[q / ga, k / 128]  b[p, k] sb[p / gb, k / 128]   (+ add[q, p])      ga, gb: 1 or 128
//
// a holds Q rows (tokens; for a weight gradient the output channels), b holds P rows.  Either operand lies with k innermost
// or with its rows innermost, so that a weight serves the forward product and the input gradient from one set of codes, and
// a weight gradient reads activations and gradients as they lie.
//
// The tensor cores apply the scales (tcgen05.mma kind::mxf8f6f4): one byte per row and 32 values of k, taken from TMEM.  Four
// instructions of 32 values go over a block of 128 with the same byte, so a 32-bit word of TMEM holds a row's scales of 512
// values, and the word is what lies in memory: four warps load words and store them to TMEM, each to its quarter of the
// lanes.
//
// The result is computed transposed: b's rows are the lanes of TMEM and a's the columns.  A thread then has one p and walks
// over q, and the 32 lanes of a warp store 32 neighbours of a row of the output, whatever its alignment and pitch.
//
//  fp8_gemm_pair   two CTAs (cta_group::2) per tile of 256 p x 256 q, persistent
//  fp8_gemm_split  one CTA per tile of 128 p x 16..128 q and part of k, for outputs too small to fill the GPU with pairs: the
//                  CTAs of a cluster hold the parts of k and add them up in the order of k through distributed shared memory.
//                  Bound by latency: 17 x 6144 x 4096 takes 9 us back to back (12 with operands from HBM, 3.9 of which are
//                  bytes): 1 us to begin, 1.5 to 2.5 to the first operands, 3 of products, 1 for the cluster to meet, 1 to join
//
// All sums are in fp32 and in a fixed order: the same bits in every run.
//
// Why a tile of 256 x 256 per pair: an instruction of 32 values of k takes 128 cycles and reads 8 KB of each CTA's shared memory,
// half of what a single CTA's 128 x 256 would need per result, and a byte from L2 serves 256 results.  TMEM holds one set of
// results (256 of 512 columns; two sets would leave no room for scales), so the epilogue takes them to registers at once and
// stores while the next tile is under way: 0.4 us of 11 between two tiles of 4096 values.  Measured: 8192 x 8192 x 4096 in 197 us
// (2790 TFLOP/s, tensor pipe 81 %), 16384 x 28672 x 4096 1380 us in a short run (2790), 1550 to 1640 under the power limit
// (2350 to 2490), which is what bounds it; a library product with one scale per tensor 2870 and 2576 in long runs where this
// has 2636 and 2391.  Adding to the product costs the reading of what is added: 8192 x 8192 x 4096 175 -> 192 us, 16384 x 4096 x
// 14336 643 -> 682 (single calls from cold, in bf16).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "entries.h"
#include "fp8_common.cuh"
#include "launch.cuh"
#include "ptx.cuh"
#include "smem_limit.h"
#include "tmap.cuh"

namespace dcpk {

static constexpr int kGemmThreads = 512;   // TMA producer, UMMA issuer, 2 idle warps; 4 scale warps; 8 epilogue warps
static constexpr int kGemmStages = 6;
static constexpr int kTileBytes = 128 * 128;  // 128 rows x 128 values, or 128 values x 128 rows
static constexpr int kScaleBufs = 4;          // of 512 values of k each
static constexpr int kGemmPairs = 148 / 2;
static constexpr int kPairParts = 8;          // of k at most, where a tile is cut
static constexpr int kPart = 32 * 128;        // sums of a warp

struct GemmOperand {
  const uint8_t* scales;
  long row_stride, k_stride;   // of the scales, in bytes
  int shift;                   // 7: 128 rows share a scale
  int rows;
  int words;                   // four scales along k can be read as a 32-bit word
};
struct GemmArgs {
  GemmOperand p, q;
  int n_kb;                    // blocks of 128 values of k
  void* out;
  const void* add;             // null, or what the product is added to, of the output's type
  long out_pitch, add_pitch;   // in elements
  int out_type;
  int tiles_p, tiles_q;
  uint32_t idesc;
  int* status;
  // pairs: tiles before `whole` are taken by one pair each, the others by `parts` pairs that have a part of k each and leave
  // sums in `part_sums`, 16 warps of kPart floats each
  int whole, parts;
  float* part_sums;
};

// Instruction descriptor of kind::mxf8f6f4: [4,6) byte of B's scale word; [7,10) / [10,13) type of A / B (0 e4m3, 1 e5m2);
// [15] / [16] A / B with rows innermost; [17,23) N >> 3; [23] scales are e8m0; [24,29) M >> 4; [29,31) byte of A's word.
__host__ __device__ constexpr uint32_t make_idesc_mx(int M, int N, int a_type, int b_type, int a_mn, int b_mn) {
  return (uint32_t(a_type) << 7) | (uint32_t(b_type) << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) |
         (uint32_t(N >> 3) << 17) | (1u << 23) | (uint32_t(M >> 4) << 24);
}
__device__ __forceinline__ uint32_t with_scale_byte(uint32_t idesc, uint32_t byte) { return idesc | (byte << 4) | (byte << 29); }

__device__ __forceinline__ void umma_mx_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_mx(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* m, uint32_t cluster_bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(cluster_bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* m, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
               : "memory");
}

// scales of a row (the last one's where it is past the end: those results are not stored) of blocks kb .. kb + 3
__device__ __forceinline__ uint32_t scale_word(const GemmOperand& o, int row, int kb, int n_kb) {
  const uint8_t* p = o.scales + long(min(row, o.rows - 1) >> o.shift) * o.row_stride + long(kb) * o.k_stride;
  if (o.words && kb + 4 <= n_kb) return *reinterpret_cast<const uint32_t*>(p);
  uint32_t v = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (kb + i < n_kb) v |= uint32_t(p[i * o.k_stride]) << (8 * i);
  return v;
}

template <int kType> struct OutType;
template <> struct OutType<kTypeF32> { using T = float; };
template <> struct OutType<kTypeF16> { using T = __half; };
template <> struct OutType<kTypeBf16> { using T = __nv_bfloat16; };

// f(type, added) with the output's type and whether there is something to add as constants: a test per store made a tile's
// stores take 50000 cycles
template <typename F>
__device__ __forceinline__ void by_output(const GemmArgs& a, F f) {
  if (a.out_type == kTypeBf16) a.add ? f(OutType<kTypeBf16>(), std::true_type()) : f(OutType<kTypeBf16>(), std::false_type());
  else if (a.out_type == kTypeF16) a.add ? f(OutType<kTypeF16>(), std::true_type()) : f(OutType<kTypeF16>(), std::false_type());
  else a.add ? f(OutType<kTypeF32>(), std::true_type()) : f(OutType<kTypeF32>(), std::false_type());
}
// `kN` results that lie a pitch apart, the first n of them, rounded once; what they are added to is read first, so that its
// loads are under way together (it may be the output itself)
template <bool kAdd, int kN, typename T>
__device__ __forceinline__ void store_results(const GemmArgs& a, T* to, const T* from, const uint32_t (&v)[kN], int n) {
  float sum[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i, from += a.add_pitch) sum[i] = __uint_as_float(v[i]) + (kAdd && i < n ? to_float(*from) : 0.f);
#pragma unroll
  for (int i = 0; i < kN; ++i, to += a.out_pitch)
    if (i < n) *to = from_float<T>(sum[i]);
}

struct __align__(1024) GemmSmem {
  uint8_t p[kGemmStages][kTileBytes];
  uint8_t q[kGemmStages][kTileBytes];
  uint32_t scales[2][128 + 256];   // words of 512 values of k: of p, of q
  // of the even CTA (bytes and arrivals of both): full, scale_full, acc_empty; the others are signalled in both
  uint64_t full[kGemmStages], empty[kGemmStages], scale_full[kScaleBufs], scale_empty[kScaleBufs], acc_full, acc_empty;
  uint32_t tmem_base;
  int abort_word;
};

// What a pair works on in its i-th turn: a tile and the blocks [kb0, kb1) of k.  Whole tiles come first; the last few, which
// would leave most pairs idle, are cut along k (in groups of four blocks, whose scales share a word).
struct Unit { int tp, tq, kb0, kb1, cut; };   // cut: index among the parts of cut tiles, -1 for a whole one
__device__ __forceinline__ void tile_at(int i, int tiles_p, int tiles_q, int& tp, int& tq);
__device__ __forceinline__ bool unit_at(const GemmArgs& a, int u, Unit& unit) {
  const int n_tiles = a.tiles_p * a.tiles_q;
  if (u >= a.whole + (n_tiles - a.whole) * a.parts) return false;
  unit.kb0 = 0;
  unit.kb1 = a.n_kb;
  unit.cut = u - a.whole;
  int tile = u;
  if (unit.cut < 0) {
    unit.cut = -1;
  } else {
    const int part = unit.cut % a.parts, groups = (a.n_kb + 3) / 4;
    tile = a.whole + unit.cut / a.parts;
    unit.kb0 = 4 * (groups * part / a.parts);
    unit.kb1 = min(4 * (groups * (part + 1) / a.parts), a.n_kb);
    if (a.parts == 1) unit.cut = -1;
  }
  tile_at(tile, a.tiles_p, a.tiles_q, unit.tp, unit.tq);
  return true;
}

// Neighbouring tiles in time share operands in L2: eight tiles of q by as many of p as are under way.
__device__ __forceinline__ void tile_at(int i, int tiles_p, int tiles_q, int& tp, int& tq) {
  constexpr int kBand = 8;
  const int band = i / (kBand * tiles_p), first = band * kBand, height = min(kBand, tiles_q - first), r = i - first * tiles_p;
  tq = first + r % height;
  tp = r / height;
}

template <bool kPMn, bool kQMn>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
fp8_gemm_pair_kernel(const __grid_constant__ CUtensorMap tm_p, const __grid_constant__ CUtensorMap tm_q,
                     const __grid_constant__ GemmArgs args) {
  extern __shared__ uint8_t smem_raw[];
  GemmSmem& sm = *reinterpret_cast<GemmSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int X = blockIdx.x & 1;   // rank in the cluster
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_p);
    tma_prefetch_desc(&tm_q);
    for (int i = 0; i < kGemmStages; ++i) { mbar_init(&sm.full[i], 1); mbar_init(&sm.empty[i], 1); }
    for (int i = 0; i < kScaleBufs; ++i) { mbar_init(&sm.scale_full[i], 8); mbar_init(&sm.scale_empty[i], 1); }
    mbar_init(&sm.acc_full, 1);
    mbar_init(&sm.acc_empty, 16);
    sm.abort_word = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc_pair(&sm.tmem_base, 512);
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  grid_let_next();
  grid_wait();
  const uint32_t tmem = sm.tmem_base;
  volatile int* abort_word = &sm.abort_word;
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1, n_kb = args.n_kb;
  Unit unit;
  constexpr int kScaleCol = 256;   // TMEM: results [0, 256), scales of the buffers behind them, 4 columns of p, 8 of q each
  // a CTA that gives up tells the other, which waits for it
  auto wait = [&](uint64_t* bar, int parity) -> bool {
    if (mbar_wait(bar, parity, abort_word)) return true;
    st_cluster_u32(smem_u32(&sm.abort_word), X ^ 1, 1u);
    return false;
  };

  if (warp >= 8) {
    // ------------------------------------------------------------ epilogue: lane = p, 128 of the tile's q
    // registers: 256 x 192 + 256 x 64 = 65536, what the block is launched with
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    const int quad = warp & 3, half = (warp - 8) >> 2;
    const uint32_t addr = tmem + (uint32_t(quad * 32) << 16) + half * 128;
    const uint32_t empty_bar = cluster_addr(smem_u32(&sm.acc_empty), 0);
    int ph = 0;
    for (int u = pair; unit_at(args, u, unit); u += n_pairs, ph ^= 1) {
      if (!__all_sync(0xffffffffu, wait(&sm.acc_full, ph))) break;
      tc_fence_after();
      uint32_t acc[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(addr + c * 32, acc + c * 32);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(empty_bar);   // the results are in registers: the next tile's products may come
      const int p = (unit.tp * 2 + X) * 128 + quad * 32 + lane, q0 = unit.tq * 256 + half * 128, n = args.q.rows - q0;
      if (unit.cut >= 0) {   // a part of k: the sums of this warp's 32 p x 128 q go to memory, four q of a lane to a piece
        float4* to = reinterpret_cast<float4*>(args.part_sums + (size_t(unit.cut) * 16 + X * 8 + warp - 8) * kPart) + lane;
#pragma unroll
        for (int c = 0; c < 32; ++c)
          to[c * 32] = make_float4(__uint_as_float(acc[4 * c]), __uint_as_float(acc[4 * c + 1]), __uint_as_float(acc[4 * c + 2]),
                                   __uint_as_float(acc[4 * c + 3]));
        continue;
      }
      if (p < args.p.rows)
        by_output(args, [&](auto type, auto added) {
          using T = typename decltype(type)::T;
          T* to = static_cast<T*>(args.out) + size_t(q0) * args.out_pitch + p;
          const T* from = static_cast<const T*>(args.add) + size_t(q0) * args.add_pitch + p;
#pragma unroll
          for (int c = 0; c < 128; c += 16, to += 16 * args.out_pitch, from += 16 * args.add_pitch)
            store_results<decltype(added)::value>(args, to, from, *reinterpret_cast<const uint32_t(*)[16]>(acc + c), n - c);
        });
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ scales: every warp to its quarter of the lanes
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    const int quad = warp & 3, t = threadIdx.x & 127;
    const uint32_t full_bar = cluster_addr(smem_u32(&sm.scale_full[0]), 0);
    int buf = 0, ph = 1, used = 0, turn = 0;
    bool ok = true;
    // Each thread brings three of the 384 words, while those before are on their way to TMEM: with scales that are not
    // neighbours along k (four bytes each) twelve words per thread, one group after the other, a weight gradient over
    // 16384 tokens took 1130 us.
    uint32_t next[3];
    const auto fetch = [&](int kb) {
      next[0] = scale_word(args.p, (unit.tp * 2 + X) * 128 + t, kb, n_kb);
      next[1] = scale_word(args.q, unit.tq * 256 + t, kb, n_kb);
      next[2] = scale_word(args.q, unit.tq * 256 + 128 + t, kb, n_kb);
    };
    int u = pair, kb = 0;
    bool more = unit_at(args, u, unit);
    if (more) fetch(kb = unit.kb0);
    while (more) {
      uint32_t* words = sm.scales[turn];
      turn ^= 1;
#pragma unroll
      for (int j = 0; j < 3; ++j) words[t + 128 * j] = next[j];
      kb += 4;
      if (kb >= unit.kb1) {
        more = unit_at(args, u += n_pairs, unit);
        kb = unit.kb0;
      }
      if (more) fetch(kb);
      asm volatile("bar.sync 1, 128;" ::: "memory");   // the words of all four warps are there, and those before the last are read
      uint32_t w[12];
#pragma unroll
      for (int j = 0; j < 12; ++j) w[j] = words[lane + 32 * j];
      ok = __all_sync(0xffffffffu, wait(&sm.scale_empty[buf], ph));
      // a warp that gave up goes on to the barriers: the others wait there
      if (ok) {
        tc_fence_after();
        const uint32_t to = tmem + (uint32_t(quad * 32) << 16) + kScaleCol + buf * 16;
        tmem_st4(to, w);
        tmem_st8(to + 4, w + 4);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(full_bar + 8 * buf);
      }
      used |= 1 << buf;
      if (++buf == kScaleBufs) { buf = 0; ph ^= 1; }
    }
    // what the even CTA's issuer signals has all come in before this CTA may retire
    for (int i = 0; i < kScaleBufs && ok; ++i) {
      if ((used >> buf) & 1) ok = wait(&sm.scale_empty[buf], ph);
      if (++buf == kScaleBufs) { buf = 0; ph ^= 1; }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------------ TMA producer
      const uint32_t full_bar = cluster_addr(smem_u32(&sm.full[0]), 0);
      int stage = 0, ph = 1, used = 0;
      bool ok = true;
      for (int u = pair; ok && unit_at(args, u, unit); u += n_pairs) {
        const int p0 = (unit.tp * 2 + X) * 128, q0 = unit.tq * 256 + X * 128;
        for (int kb = unit.kb0; kb < unit.kb1; ++kb) {
          ok = wait(&sm.empty[stage], ph);
          if (!ok) break;
          if (X == 0) mbar_expect_tx(&sm.full[stage], 4 * kTileBytes);
          tma_load_2d_pair(sm.p[stage], &tm_p, full_bar + 8 * stage, kPMn ? p0 : kb * 128, kPMn ? kb * 128 : p0);
          tma_load_2d_pair(sm.q[stage], &tm_q, full_bar + 8 * stage, kQMn ? q0 : kb * 128, kQMn ? kb * 128 : q0);
          used |= 1 << stage;
          if (++stage == kGemmStages) { stage = 0; ph ^= 1; }
        }
      }
      for (int i = 0; i < kGemmStages && ok; ++i) {
        if ((used >> stage) & 1) ok = wait(&sm.empty[stage], ph);
        if (++stage == kGemmStages) { stage = 0; ph ^= 1; }
      }
      // copies already in flight get a millisecond to land before the CTAs retire
      if (!ok)
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    } else if (warp == 1 && X == 0 && elect_one()) {
      // ------------------------------------------------------------ UMMA issuer, for both CTAs
      const uint64_t some = make_sdesc_sw128(0, 16, 1024);
      const uint32_t hi = uint32_t(some >> 32);
      const uint32_t p_lo = uint32_t(some) + sdesc_addr(sm.p[0]), q_lo = uint32_t(some) + sdesc_addr(sm.q[0]);
      auto desc = [&](uint32_t lo) { return (uint64_t(hi) << 32) | lo; };
      constexpr uint32_t kStep = kTileBytes >> 4;             // in a descriptor's 16-byte units
      constexpr uint32_t kPK = kPMn ? 256 : 2, kQK = kQMn ? 256 : 2;   // 32 values of k
      int stage = 0, ph = 0, buf = 0, sph = 0, aph = 1, done = 0;
      bool ok = true;
      for (int u = pair; ok && unit_at(args, u, unit); u += n_pairs) {
        ok = wait(&sm.acc_empty, aph);   // the last tile's results are in registers
        aph ^= 1;
        for (int kb = unit.kb0; kb < unit.kb1 && ok; ++kb) {
          if ((kb & 3) == 0) ok = wait(&sm.scale_full[buf], sph);
          ok = ok && wait(&sm.full[stage], ph);
          if (!ok) break;
          tc_fence_after();
          const uint32_t idesc = with_scale_byte(args.idesc, kb & 3), scales = tmem + kScaleCol + buf * 16;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_mx_pair(tmem, desc(p_lo + stage * kStep + k * kPK), desc(q_lo + stage * kStep + k * kQK), idesc, scales, scales + 4,
                         (kb > unit.kb0 || k > 0) ? 1u : 0u);
          umma_commit_pair(&sm.empty[stage]);
          if ((kb & 3) == 3 || kb + 1 == unit.kb1) {
            umma_commit_pair(&sm.scale_empty[buf]);
            if (++buf == kScaleBufs) { buf = 0; sph ^= 1; }
          }
          if (++stage == kGemmStages) { stage = 0; ph ^= 1; }
        }
        umma_commit_pair(&sm.acc_full);
        ++done;
      }
      // TMEM and operands stay until all has retired
      for (int spin = 0; spin < 200000 && done > 0 && !mbar_try_wait(&sm.acc_full, (done - 1) & 1); ++spin) {}
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
  if (threadIdx.x == 0 && sm.abort_word) atomicExch(args.status, kStatusBarrierTimeout);
}

// Adds up the parts of cut tiles in the order of k: a thread has four q of one p.  A kernel of its own over the whole GPU takes
// 3 us; the last of a tile's pairs to be through, which has the parts in reach of one SM, took 2.4 us for each of them.
__global__ void __launch_bounds__(256) fp8_gemm_join_kernel(const __grid_constant__ GemmArgs args) {
  const int lane = threadIdx.x & 31, piece = (blockIdx.x * 256 + threadIdx.x) >> 5, c = piece & 31, mine = (piece >> 5) & 15, tile = piece >> 9;
  int tp, tq;
  tile_at(args.whole + tile, args.tiles_p, args.tiles_q, tp, tq);
  const int half = (mine >> 2) & 1, p = (tp * 2 + (mine >> 3)) * 128 + (mine & 3) * 32 + lane, q = tq * 256 + half * 128 + c * 4;
  grid_wait();
  const float4* from = reinterpret_cast<const float4*>(args.part_sums + (size_t(tile) * args.parts * 16 + mine) * kPart) + c * 32 + lane;
  float4 v[kPairParts];
#pragma unroll
  for (int r = 0; r < kPairParts; ++r)
    if (r < args.parts) v[r] = from[size_t(r) * 16 * (kPart / 4)];
  grid_let_next();
#pragma unroll
  for (int r = 1; r < kPairParts; ++r)
    if (r < args.parts) { v[0].x += v[r].x; v[0].y += v[r].y; v[0].z += v[r].z; v[0].w += v[r].w; }
  if (p >= args.p.rows) return;
  const uint32_t sum[4] = {__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[0].z), __float_as_uint(v[0].w)};
  by_output(args, [&](auto type, auto added) {
    using T = typename decltype(type)::T;
    store_results<decltype(added)::value>(args, static_cast<T*>(args.out) + size_t(q) * args.out_pitch + p,
                                          static_cast<const T*>(args.add) + size_t(q) * args.add_pitch + p, sum, args.q.rows - q);
  });
}

// ------------------------------------------------------------------ small outputs
static constexpr int kSplitThreads = 256;   // TMA producer, UMMA issuer, 2 idle warps; 4 warps for scales, then results
static constexpr int kSplitMax = 8;

template <int kN> constexpr int split_stages() { return kN <= 16 ? 11 : kN <= 32 ? 10 : kN <= 64 ? 8 : 6; }

template <int kN>
struct __align__(1024) SplitSmem {
  union {
    struct {
      uint8_t p[split_stages<kN>()][kTileBytes];
      uint8_t q[split_stages<kN>()][kN * 128];
    };
    float part[kN][128];   // this CTA's sums, when all products are through
  };
  uint32_t scales[2][256];
  uint64_t full[split_stages<kN>()], empty[split_stages<kN>()], scale_full[kScaleBufs], scale_empty[kScaleBufs], acc_full;
  uint32_t tmem_base;
  int abort_word;
};

template <int kN, bool kPMn, bool kQMn>
__global__ void __launch_bounds__(kSplitThreads, 1)
fp8_gemm_split_kernel(const __grid_constant__ CUtensorMap tm_p, const __grid_constant__ CUtensorMap tm_q,
                      const __grid_constant__ GemmArgs args, int splits) {
  static_assert(!kQMn || kN == 128, "rows innermost: a tile is 128 of them wide");
  constexpr int kStages = split_stages<kN>();
  extern __shared__ uint8_t smem_raw[];
  SplitSmem<kN>& sm = *reinterpret_cast<SplitSmem<kN>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_p);
    tma_prefetch_desc(&tm_q);
    for (int i = 0; i < kStages; ++i) { mbar_init(&sm.full[i], 1); mbar_init(&sm.empty[i], 1); }
    for (int i = 0; i < kScaleBufs; ++i) { mbar_init(&sm.scale_full[i], 4); mbar_init(&sm.scale_empty[i], 1); }
    mbar_init(&sm.acc_full, 1);
    sm.abort_word = 0;
    mbar_fence_init();
  }
  constexpr int kColumns = 256;   // results up to 128, scales behind them
  if (warp == 1) {
    tmem_alloc(&sm.tmem_base, kColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_let_next();
  grid_wait();
  const uint32_t tmem = sm.tmem_base;
  volatile int* abort_word = &sm.abort_word;
  constexpr int kScaleCol = 128;
  const int rank = blockIdx.x % splits, tile = blockIdx.x / splits;
  const int tp = tile % args.tiles_p, tq = tile / args.tiles_p;
  const int kb0 = args.n_kb * rank / splits, kb1 = args.n_kb * (rank + 1) / splits;   // a scale word may belong to two parts
  const int p0 = tp * 128, q0 = tq * kN;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, ph = 1;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = mbar_wait(&sm.empty[stage], ph, abort_word);
        if (!ok) break;
        mbar_expect_tx(&sm.full[stage], kTileBytes + kN * 128);
        tma_load_2d(sm.p[stage], &tm_p, &sm.full[stage], kPMn ? p0 : kb * 128, kPMn ? kb * 128 : p0);
        tma_load_2d(sm.q[stage], &tm_q, &sm.full[stage], kQMn ? q0 : kb * 128, kQMn ? kb * 128 : q0);
        if (++stage == kStages) { stage = 0; ph ^= 1; }
      }
      if (!ok)
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint64_t some = make_sdesc_sw128(0, 16, 1024);
      const uint32_t hi = uint32_t(some >> 32);
      const uint32_t p_lo = uint32_t(some) + sdesc_addr(sm.p[0]), q_lo = uint32_t(some) + sdesc_addr(sm.q[0]);
      auto desc = [&](uint32_t lo) { return (uint64_t(hi) << 32) | lo; };
      constexpr uint32_t kPK = kPMn ? 256 : 2, kQK = kQMn ? 256 : 2;
      int stage = 0, ph = 0, buf = 0, sph = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if ((kb & 3) == 0 || kb == kb0) ok = mbar_wait(&sm.scale_full[buf], sph, abort_word);
        ok = ok && mbar_wait(&sm.full[stage], ph, abort_word);
        if (!ok) break;
        tc_fence_after();
        const uint32_t idesc = with_scale_byte(args.idesc, kb & 3), scales = tmem + kScaleCol + buf * 8;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_mx(tmem, desc(p_lo + stage * (kTileBytes >> 4) + k * kPK), desc(q_lo + stage * (kN * 128 >> 4) + k * kQK), idesc, scales,
                  scales + 4, (kb > kb0 || k > 0) ? 1u : 0u);
        umma_commit(&sm.empty[stage]);
        if ((kb & 3) == 3 || kb + 1 == kb1) {
          umma_commit(&sm.scale_empty[buf]);
          if (++buf == kScaleBufs) { buf = 0; sph ^= 1; }
        }
        if (++stage == kStages) { stage = 0; ph ^= 1; }
      }
      umma_commit(&sm.acc_full);
      // TMEM and operands stay until all has retired
      for (int spin = 0; spin < 200000 && !mbar_try_wait(&sm.acc_full, 0); ++spin) {}
    }
  } else if (warp >= 4) {
    const int quad = warp & 3, t = threadIdx.x & 127;
    int buf = 0, ph = 1, turn = 0;
    bool ok = true;
    uint32_t next[2];
    const auto fetch = [&](int kb) {
      next[0] = scale_word(args.p, p0 + t, kb, args.n_kb);
      next[1] = t < kN ? scale_word(args.q, q0 + t, kb, args.n_kb) : 0u;
    };
    fetch(kb0 & ~3);
    for (int kb = kb0 & ~3; kb < kb1; kb += 4) {
      uint32_t* words = sm.scales[turn];
      turn ^= 1;
      words[t] = next[0];
      words[128 + t] = next[1];
      if (kb + 4 < kb1) fetch(kb + 4);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = words[lane + 32 * j];
      ok = __all_sync(0xffffffffu, mbar_wait(&sm.scale_empty[buf], ph, abort_word));
      if (ok) {   // a warp that gave up goes on to the barriers: the others wait there
        tc_fence_after();
        const uint32_t to = tmem + (uint32_t(quad * 32) << 16) + kScaleCol + buf * 8;
        tmem_st4(to, w);
        tmem_st4(to + 4, w + 4);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.scale_full[buf]);
      }
      if (++buf == kScaleBufs) { buf = 0; ph ^= 1; }
    }
    ok = __all_sync(0xffffffffu, ok && mbar_wait(&sm.acc_full, 0, abort_word));
    const int row = quad * 32 + lane, p = p0 + row;
    if (ok) {
      tc_fence_after();
#pragma unroll 1
      for (int c0 = 0; c0 < kN; c0 += 16) {
        uint32_t acc[16];
        tmem_ld16(tmem + (uint32_t(quad * 32) << 16) + c0, acc);
        tmem_wait_ld();
        if (splits > 1) {
#pragma unroll
          for (int c = 0; c < 16; ++c) sm.part[c0 + c][row] = __uint_as_float(acc[c]);
        } else if (p < args.p.rows) {
          by_output(args, [&](auto type, auto added) {
            using T = typename decltype(type)::T;
            T* to = static_cast<T*>(args.out) + size_t(q0 + c0) * args.out_pitch + p;
            const T* from = static_cast<const T*>(args.add) + size_t(q0 + c0) * args.add_pitch + p;
            store_results<decltype(added)::value>(args, to, from, acc, args.q.rows - q0 - c0);
          });
        }
      }
      tc_fence_before();
    }
  }
  if (splits > 1) {
    __syncwarp();
    cluster_sync();
    // every CTA adds up its share of the columns, in the order of k: a warp has a column, a lane four neighbours of it
    if (!sm.abort_word) {
      const int n = min(kN, args.q.rows - q0), stop = n * (rank + 1) / splits, p = p0 + 4 * lane;
      const uint32_t at = smem_u32(&sm.part[0][4 * lane]);
      by_output(args, [&](auto type, auto added) {
        using T = typename decltype(type)::T;
#pragma unroll 2
        for (int c = n * rank / splits + warp; c < stop; c += kSplitThreads / 32) {
          float4 v[kSplitMax];
#pragma unroll
          for (int r = 0; r < kSplitMax; ++r)
            if (r < splits) v[r] = ld_cluster_f4(at + c * 512, r);
#pragma unroll
          for (int r = 1; r < kSplitMax; ++r)
            if (r < splits) { v[0].x += v[r].x; v[0].y += v[r].y; v[0].z += v[r].z; v[0].w += v[r].w; }
          T* to = static_cast<T*>(args.out) + size_t(q0 + c) * args.out_pitch + p;
          const T* from = static_cast<const T*>(args.add) + size_t(q0 + c) * args.add_pitch + p;
          float f[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (decltype(added)::value && p + j < args.p.rows) f[j] += to_float(from[j]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (p + j < args.p.rows) to[j] = from_float<T>(f[j]);
        }
      });
    }
    cluster_sync();
  } else {
    __syncthreads();
  }
  if (warp == 1) tmem_dealloc(tmem, kColumns);
  if (threadIdx.x == 0 && sm.abort_word) atomicExch(args.status, kStatusBarrierTimeout);
}

// codes [rows, cols] of `pitch` bytes per row; tiles of 128 bytes x box_rows, 128-byte swizzle, zeros outside
static int encode_codes_map(CUtensorMap* out, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch, uint32_t box_rows) {
  EncodeTiledFn fn = get_encode_fn();
  if (!fn) return -1;
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {pitch};
  cuuint32_t box[2] = {128, box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -2;
}

static std::atomic<uint64_t> g_gemm_smem_raised[16];

template <bool kPMn, bool kQMn>
static int launch_pair(const CUtensorMap& tm_p, const CUtensorMap& tm_q, const GemmArgs& args, cudaStream_t stream) {
  const int smem = int(sizeof(GemmSmem)) + 1024;
  auto kernel = fp8_gemm_pair_kernel<kPMn, kQMn>;
  if (raise_smem_limit(kernel, smem, g_gemm_smem_raised[kPMn * 2 + kQMn]) != cudaSuccess) return -4;
  const int units = args.whole + (args.tiles_p * args.tiles_q - args.whole) * args.parts;
  const cudaError_t rc = launch_overlapped(kernel, dim3(2 * std::min(units, kGemmPairs)), kGemmThreads, smem, stream, 1, true, tm_p, tm_q, args);
  if (rc == cudaSuccess && args.parts > 1) {
    const cudaError_t join = launch_overlapped(fp8_gemm_join_kernel, dim3((args.tiles_p * args.tiles_q - args.whole) * 64), 256, 0, stream, 1, true, args);
    if (join != cudaSuccess) return -5;
  }
  return rc == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -5;
}

template <int kN, bool kPMn, bool kQMn>
static int launch_split(const CUtensorMap& tm_p, const CUtensorMap& tm_q, const GemmArgs& args, int splits, int slot, cudaStream_t stream) {
  const int smem = int(sizeof(SplitSmem<kN>)) + 1024;
  auto kernel = fp8_gemm_split_kernel<kN, kPMn, kQMn>;
  if (raise_smem_limit(kernel, smem, g_gemm_smem_raised[slot]) != cudaSuccess) return -4;
  const cudaError_t rc = launch_overlapped(kernel, dim3(args.tiles_p * args.tiles_q * splits), kSplitThreads, smem, stream, splits, true,
                                           tm_p, tm_q, args, splits);
  return rc == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : -5;
}

}  // namespace dcpk

using namespace dcpk;

// Which kernel, and how its work is cut.
struct GemmPlan {
  bool pairs;
  int n;                    // q of a tile
  long tiles_p, tiles_q;
  int whole, parts;         // pairs: see GemmArgs; split: parts
  long work() const { return pairs && parts > 1 ? (tiles_p * tiles_q - whole) * parts * 16l * kPart * 4 : 0; }
};
static GemmPlan plan_gemm(long p_rows, long q_rows, bool q_rows_inner, int k, int form) {
  GemmPlan g;
  const int groups = ((k + 127) / 128 + 3) / 4;
  g.tiles_p = (p_rows + 255) / 256;
  g.tiles_q = (q_rows + 255) / 256;
  const long pair_tiles = g.tiles_p * g.tiles_q;
  // Pairs where their tiles give two thirds of them work, or fewer tiles long sums, which are cut, or where the other kernel,
  // which is not persistent, has more CTAs than processors and so a second round; us with pairs / split:
  // 2048 x 1536 x 1024 (48 tiles) 9.5 / 12.4, 200 x 28672 x 4096 (112) 32 / 49, 1024 x 2048 x 4096 (32) 18.4 / 13.5, 512 x 4096 x
  // 14336 (32) 32.5 / 34.8, 1536 x 1024 x 16384 (24) 28 / 37, 512 x 1024 x 4096 (8) 14.3 / 10.5; a second round, from cold: 256 x
  // 9728 x 4096 (38 tiles, 152 CTAs) 23.6 / 31.7, 512 x 5120 x 5120 (40, 160) 25.6 / 33.8, 768 x 3328 x 512 (39, 156) 13.3 / 15.4, 256 x
  // 12032 x 2048 (47, 188) 19.5 / 23.6; none: 1536 x 1536 x 2048 (36, 144) 21.5 / 13.3, 300 x 5120 x 4096 (40, 120) 22.8 / 18.5.
  const long split_ctas = ((p_rows + 127) / 128) * ((q_rows + 127) / 128);
  g.pairs = form == 1 || (form == 0 && q_rows > 128 && (pair_tiles >= 48 || pair_tiles * ((k + 127) / 128) >= 2304 || split_ctas > 2 * kGemmPairs));
  if (g.pairs) {
    g.n = 256;
    const int rest = int(pair_tiles % kGemmPairs);
    g.parts = rest > 0 ? std::max(1, std::min({kGemmPairs / rest, groups, kPairParts})) : 1;
    g.whole = int(std::min(g.parts > 1 ? pair_tiles - rest : pair_tiles, 0x7fffffffl));
    return g;
  }
  g.n = q_rows_inner || q_rows > 64 ? 128 : q_rows > 32 ? 64 : q_rows > 16 ? 32 : 16;
  g.tiles_p = (p_rows + 127) / 128;
  g.tiles_q = (q_rows + g.n - 1) / g.n;
  g.whole = 0;
  // as many parts as still are all under way at once: clusters of so many CTAs that fit the GPU's processors (one CTA per SM; by
  // cudaOccupancyMaxActiveClusters).  A second round costs more than the shorter sums give: 17 x 6144 x 4096 in 48 clusters of
  // six 16 us, of two 12 (operands from HBM, as all of these).
  constexpr int kFit[kSplitMax + 1] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
  g.parts = 1;
  for (int parts = 2; parts <= std::min(kSplitMax, (k + 127) / 128); ++parts)
    if (g.tiles_p * g.tiles_q <= kFit[parts]) g.parts = parts;
  return g;
}

// bytes of scratch a call needs; 0: none
extern "C" long dcpk_fp8_gemm_work(long q_rows, long p_rows, int q_rows_inner, int k, int form) {
  return q_rows <= 0 || p_rows <= 0 || k <= 0 ? 0 : plan_gemm(p_rows, q_rows, q_rows_inner, k, form).work();
}

// out [q.rows, p.rows] = q p^T + add.  form: 0 by rule, 1 pairs, 2 split (tests and measurements).  work: scratch of
// dcpk_fp8_gemm_work() bytes.
extern "C" int dcpk_fp8_gemm(const DcpkFp8Operand* q, const DcpkFp8Operand* p, int k, void* out, long out_pitch, const void* add,
                             long add_pitch, int out_type, int form, void* work, int* status, void* stream) {
  if (q->rows <= 0 || p->rows <= 0) return 0;
  if (k <= 0 || out_type < 0 || out_type > 2) return -3;
  GemmArgs args;
  const DcpkFp8Operand* from[2] = {p, q};
  GemmOperand* to[2] = {&args.p, &args.q};
  for (int i = 0; i < 2; ++i) {
    const DcpkFp8Operand& o = *from[i];
    if (o.pitch % 16 || reinterpret_cast<uintptr_t>(o.codes) % 16 || (o.shift != 0 && o.shift != 7) || o.code_type < 0 || o.code_type > 1)
      return -3;
    *to[i] = {static_cast<const uint8_t*>(o.scales), o.scale_row_stride, o.scale_k_stride, o.shift, o.rows,
              o.scale_k_stride == 1 && o.scale_row_stride % 4 == 0 && reinterpret_cast<uintptr_t>(o.scales) % 4 == 0};
  }
  args.n_kb = (k + 127) / 128;
  args.out = out;
  args.add = add;
  args.out_pitch = out_pitch;
  args.add_pitch = add_pitch;
  args.out_type = out_type;
  args.status = status;
  const GemmPlan plan = plan_gemm(p->rows, q->rows, q->rows_inner, k, form);
  const bool pairs = plan.pairs;
  const int n = plan.n;
  if (plan.tiles_p * plan.tiles_q * kSplitMax > 0x7fffffffl) return -3;
  args.tiles_p = int(plan.tiles_p);
  args.tiles_q = int(plan.tiles_q);
  args.whole = plan.whole;
  args.parts = plan.parts;
  args.part_sums = nullptr;
  const auto map = [&](CUtensorMap* m, const DcpkFp8Operand& o, int box) {
    return o.rows_inner ? encode_codes_map(m, o.codes, k, o.rows, o.pitch, 128) : encode_codes_map(m, o.codes, o.rows, k, o.pitch, box);
  };
  CUtensorMap tm_p, tm_q;
  if (map(&tm_p, *p, 128) || map(&tm_q, *q, n < 128 ? n : 128)) return -1;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int mode = p->rows_inner * 2 + q->rows_inner;
  if (pairs) {
    if (plan.work() > 0 && !work) return -3;
    args.part_sums = static_cast<float*>(work);
    args.idesc = make_idesc_mx(256, 256, p->code_type, q->code_type, p->rows_inner, q->rows_inner);
    return mode == 0 ? launch_pair<false, false>(tm_p, tm_q, args, s) : mode == 1 ? launch_pair<false, true>(tm_p, tm_q, args, s)
         : mode == 2 ? launch_pair<true, false>(tm_p, tm_q, args, s) : launch_pair<true, true>(tm_p, tm_q, args, s);
  }
  args.idesc = make_idesc_mx(128, n, p->code_type, q->code_type, p->rows_inner, q->rows_inner);
  const int splits = plan.parts;
#define DCPK_SPLIT(N, PM, QM, SLOT) launch_split<N, PM, QM>(tm_p, tm_q, args, splits, SLOT, s)
  if (q->rows_inner) return p->rows_inner ? DCPK_SPLIT(128, true, true, 4) : DCPK_SPLIT(128, false, true, 5);
  if (p->rows_inner)
    return n == 16 ? DCPK_SPLIT(16, true, false, 6) : n == 32 ? DCPK_SPLIT(32, true, false, 7) : n == 64 ? DCPK_SPLIT(64, true, false, 8)
                                                                                               : DCPK_SPLIT(128, true, false, 9);
  return n == 16 ? DCPK_SPLIT(16, false, false, 10) : n == 32 ? DCPK_SPLIT(32, false, false, 11) : n == 64 ? DCPK_SPLIT(64, false, false, 12)
                                                                                              : DCPK_SPLIT(128, false, false, 13);
#undef DCPK_SPLIT
}
