// Linear layer with bias, activation and residual, forward and backward.
//
//   forward    z = x w^T + bias,  y = act(z) + residual       (x [m][k], w [n][k])
//   backward   dz = dy act'(z),  dx = dz w,  dw = dz^T x,  dbias = sum of dz's rows
//
// The three products run on the fifth-generation tensor cores (tcgen05.mma, fp32
// accumulators in TMEM) fed by TMA, in one kernel: its operand tiles are K-major
// or MN-major per product (the matrix descriptor says which), so dx reads w and dw
// reads dz and x as they lie in memory, without a transposed copy. Everything after
// the product -- bias, activation, residual, the rounding to the rows' type -- is
// done on the accumulator before it leaves the SM.
//
// Bound: 2 m n k operations at the tensor cores' rate for batches of hundreds of
// rows and more; the weights' bytes below that, where linear_small_kernel (up to
// kLinearSmallRows rows) streams them once with CUDA cores.
//
// The pre-activation z is kept for the backward pass as fp16, also for bf16 rows:
// the activations' derivatives are constant where fp16 ends (|z| > 65504), and
// fp16's 11 bits keep the derivative's error an order below bf16's own rounding.
// dz is rounded once to the rows' type, because both products that read it take
// half-precision operands.
#include "cvs_device.cuh"
#include "cvs_elem.cuh"
#include "cvs_kernels.h"

#include <algorithm>

namespace cvs {

namespace {

// ---------------------------------------------------------------------------
// Activations
// ---------------------------------------------------------------------------
__device__ __forceinline__ float act_value(float z, int act) {
  if (act == kActRelu) return z > 0.f ? z : (z != z ? z : 0.f);
  if (act == kActGelu) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  if (act == kActSilu) return z / (1.f + expf(-z));
  return z;
}

__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == kActRelu) return z > 0.f ? 1.f : (z != z ? z : 0.f);
  // Beyond +-100 both slopes are 0 or 1 to the last bit; the clamp keeps an
  // infinite z (an overflowed fp16 pre-activation) from giving inf x 0. NaN stays.
  const float c = z != z ? z : fminf(fmaxf(z, -100.f), 100.f);
  if (act == kActGelu) {
    const float cdf = 0.5f * (1.f + erff(c * 0.70710678118654752f));
    return fmaf(c * 0.39894228040143268f, expf(-0.5f * c * c), cdf);
  }
  if (act == kActSilu) {
    const float s = 1.f / (1.f + expf(-c));
    return s * fmaf(c, 1.f - s, 1.f);
  }
  return 1.f;
}

// Two fp32 values as a pair of halves of the given type.
__device__ __forceinline__ uint32_t pack2(float lo, float hi, bool bf16) {
  if (bf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float2 unpack2(uint32_t u, bool bf16) {
  if (bf16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}

__device__ __forceinline__ float half_at(const void* p, size_t i, bool bf16) {
  return bf16 ? to_f32(static_cast<const __nv_bfloat16*>(p)[i]) : to_f32(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ uint16_t half_bits(float v, bool bf16) {
  return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// ---------------------------------------------------------------------------
// tcgen05 product
// ---------------------------------------------------------------------------
constexpr int kGemmM = 128;   // rows of the output tile per CTA (TMEM lanes)
constexpr int kGemmK = 64;    // halves per K slice: one 128-byte swizzled row
constexpr int kGemmEpiWarps = 8;
constexpr int kGemmThreads = 64 + 32 * kGemmEpiWarps;
constexpr int kGemmMaxStages = 8;

// Shared memory: ring of operand stages, then per epilogue warp a staging buffer
// of 32 rows x one column chunk and 32 columns' bias, then the barriers.
template <int CG, int BN>
struct GemmShape {
  static constexpr int kBRows = BN / CG;                    // columns of the tile whose operand rows this CTA loads
  static constexpr int kABytes = kGemmM * kGemmK * 2;
  static constexpr int kBBytes = kBRows * kGemmK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kChunk = BN >= 128 ? 64 : 32;        // columns staged at a time
  static constexpr int kUnits = kChunk / 8;                 // 16-byte units per staged row
  static constexpr int kWarpStage = 32 * kChunk * 2;
  static constexpr int kBiasBytes = kGemmEpiWarps * 32 * 4;
  static constexpr int kBarBytes = 8 * (2 * kGemmMaxStages + 5) + 16;
  static constexpr int kTail = kGemmEpiWarps * kWarpStage + kBiasBytes + kBarBytes;
  static constexpr int kFit = (kSmemBudget - kTail) / kStageBytes;
  static constexpr int kStages = kFit < kGemmMaxStages ? kFit : kGemmMaxStages;
  static constexpr int kTotal = kStages * kStageBytes + kTail;
  static constexpr uint32_t kTmemCols = 2 * BN < 32 ? 32 : 2 * BN;
};

__device__ __forceinline__ void tma_load_tile(void* dst, const void* desc, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(desc)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}

__device__ __forceinline__ void tma_load_tile_pair(void* dst, const void* desc, uint32_t bar_cluster, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(desc)), "r"(bar_cluster), "r"(x), "r"(y)
      : "memory");
}

// Matrix descriptor of a 128-byte-swizzled operand tile. K-major: rows of 64
// halves along K, 8-row groups 1024 bytes apart. MN-major: blocks of 64 rows or
// columns x 64 K steps (8 KB, one TMA box), each K step a 128-byte row: groups of
// 8 K steps are 1024 bytes apart (stride offset), blocks 8192 (leading offset).
__device__ __forceinline__ uint64_t gemm_desc(uint32_t saddr, bool mn) {
  uint64_t d = static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(mn ? 8192u >> 4 : 1u) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

// Instruction descriptor, kind::f16: half-precision operands of one type, fp32 accumulator.
__device__ __forceinline__ uint32_t gemm_idesc(int m, int n, bool bf16, bool a_mn, bool b_mn) {
  const uint32_t fmt = bf16 ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

struct TileAt {
  int prob, mt, nt, split, tile;
};

// Tile t of the call: which product, which output tile, which part of K. Within a
// product the tiles go down groups of 8 row tiles before the next column tile, so
// that the CTAs at work share operand tiles in L2.
__device__ __forceinline__ TileAt tile_at(const GemmArgs& a, int t) {
  TileAt r;
  r.prob = t < a.p[0].work ? 0 : 1;
  const GemmProblem& p = a.p[r.prob];
  int i = r.prob ? t - a.p[0].work : t;
  const int tiles = p.tiles_m * p.tiles_n;
  r.split = i / tiles;
  i -= r.split * tiles;
  r.tile = i;
  const int group = i / (8 * p.tiles_n);
  const int rows = min(8, p.tiles_m - group * 8);
  i -= group * 8 * p.tiles_n;
  r.mt = group * 8 + i % rows;
  r.nt = i / rows;
  return r;
}

// One 32-row x chunk block between global memory and registers, rows in
// coalesced order: lane l handles 16-byte unit l % units of row l / units, then
// every (32 / units)-th row below it.
template <int UNITS>
struct BlockIo {
  static constexpr int kRowsPerStep = 32 / UNITS;
  static __device__ __forceinline__ int swizzle(int row, int unit) {
    const int s = UNITS == 8 ? row & 7 : (row >> 1) & 3;
    return (row * UNITS + (unit ^ s)) * 16;
  }
  static __device__ __forceinline__ void load(const void* src, long long ld, bool vec, int row0, int rows, int col0,
                                              int cols, int lane, uint4 (&v)[UNITS]) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const int r = lane / UNITS + i * kRowsPerStep, c = col0 + (lane % UNITS) * 8;
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (row0 + r >= rows || c >= cols) continue;
      const uint16_t* p = static_cast<const uint16_t*>(src) + static_cast<long long>(row0 + r) * ld + c;
      if (vec && c + 8 <= cols) {
        v[i] = *reinterpret_cast<const uint4*>(p);
      } else {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int t = 0; t < 8; ++t)
          if (c + t < cols) w[t / 2] |= static_cast<uint32_t>(p[t]) << (16 * (t & 1));
        v[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  static __device__ __forceinline__ void stage(uint8_t* buf, int lane, const uint4 (&v)[UNITS]) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i)
      *reinterpret_cast<uint4*>(buf + swizzle(lane / UNITS + i * kRowsPerStep, lane % UNITS)) = v[i];
  }
  static __device__ __forceinline__ void store(void* dst, long long ld, bool vec, int row0, int rows, int col0, int cols,
                                               int lane, const uint8_t* buf) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const int r = lane / UNITS + i * kRowsPerStep, c = col0 + (lane % UNITS) * 8;
      if (row0 + r >= rows || c >= cols) continue;
      const uint4 v = *reinterpret_cast<const uint4*>(buf + swizzle(r, lane % UNITS));
      uint16_t* p = static_cast<uint16_t*>(dst) + static_cast<long long>(row0 + r) * ld + c;
      if (vec && c + 8 <= cols) {
        *reinterpret_cast<uint4*>(p) = v;
      } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int t = 0; t < 8; ++t)
          if (c + t < cols) p[t] = static_cast<uint16_t>(w[t / 2] >> (16 * (t & 1)));
      }
    }
  }
};

template <int CG, int BN>
struct GemmShared {
  using S = GemmShape<CG, BN>;
  uint8_t* base;
  __device__ uint8_t* a(int s) const { return base + s * S::kStageBytes; }
  __device__ uint8_t* b(int s) const { return base + s * S::kStageBytes + S::kABytes; }
  __device__ uint8_t* stage(int w) const { return base + S::kStages * S::kStageBytes + w * S::kWarpStage; }
  __device__ float* bias(int w) const {
    return reinterpret_cast<float*>(base + S::kStages * S::kStageBytes + kGemmEpiWarps * S::kWarpStage) + w * 32;
  }
  __device__ uint64_t* bar(int i) const {
    return reinterpret_cast<uint64_t*>(base + S::kStages * S::kStageBytes + kGemmEpiWarps * S::kWarpStage +
                                       S::kBiasBytes) + i;
  }
  __device__ uint64_t* full(int s) const { return bar(s); }
  __device__ uint64_t* empty(int s) const { return bar(kGemmMaxStages + s); }
  __device__ uint64_t* tfull(int i) const { return bar(2 * kGemmMaxStages + i); }
  __device__ uint64_t* tempty(int i) const { return bar(2 * kGemmMaxStages + 2 + i); }
  __device__ uint64_t* done() const { return bar(2 * kGemmMaxStages + 4); }
  __device__ uint32_t* tmem_holder() const { return reinterpret_cast<uint32_t*>(bar(2 * kGemmMaxStages + 5)); }
  __device__ volatile int* abort_flag() const {
    return reinterpret_cast<volatile int*>(bar(2 * kGemmMaxStages + 5)) + 1;
  }
};

// One CTA (CG = 1, 128 x BN tiles) or a pair of CTAs (CG = 2, 256 x BN tiles; each
// CTA holds its 128 rows of A and half of B's rows) per work item, persistent over
// the call's tiles: warp 0 loads, warp 1 issues the MMAs, 8 warps drain one of two
// accumulators while the other is computed. Waits are bounded (cvs_device.cuh); a
// wait that runs out stops every role of the CTA, and the pair still meets at the
// last barrier.
template <int CG, int BN>
__global__ void __launch_bounds__(kGemmThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap a0, const __grid_constant__ CUtensorMap b0,
                const __grid_constant__ CUtensorMap a1, const __grid_constant__ CUtensorMap b1,
                const __grid_constant__ GemmArgs args) {
  using S = GemmShape<CG, BN>;
  constexpr int kS = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  GemmShared<CG, BN> sh;
  sh.base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int first = static_cast<int>(blockIdx.x) / CG;
  const int step = static_cast<int>(gridDim.x) / CG;
  const int total = args.p[0].work + args.p[1].work;
  volatile int* abort = sh.abort_flag();

  if (threadIdx.x == 0) {
    for (int s = 0; s < kS; ++s) {
      mbar_init(sh.full(s), 1);
      mbar_init(sh.empty(s), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(sh.tfull(t), 1);
      mbar_init(sh.tempty(t), leader ? CG * kGemmEpiWarps : 1);
    }
    mbar_init(sh.done(), 1);
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&a0);
    tma_prefetch_desc(&b0);
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(sh.tmem_holder(), S::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(sh.tmem_holder(), S::kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *sh.tmem_holder();
  grid_dependency_wait();

  if (warp == 0) {
    // ------------------------------ TMA producer ---------------------------
    if (elect_one_lane()) {
      int it = 0;
      bool ok = true;
      for (int t = first; ok && t < total; t += step) {
        const TileAt w = tile_at(args, t);
        const GemmProblem& p = args.p[w.prob];
        const CUtensorMap* am = w.prob ? &a1 : &a0;
        const CUtensorMap* bm = w.prob ? &b1 : &b0;
        const int arow = (w.mt * CG + static_cast<int>(rank)) * kGemmM;
        const int brow = w.nt * BN + static_cast<int>(rank) * S::kBRows;
        const int k0 = w.split * p.kper, k1 = min(p.kblocks, k0 + p.kper);
        for (int kb = k0; kb < k1; ++kb, ++it) {
          const int s = it % kS;
          if (!mbar_wait(sh.empty(s), ((it / kS) & 1) ^ 1, abort, args.err, 33)) {
            ok = false;
            break;
          }
          if (leader) mbar_arrive_expect_tx(sh.full(s), CG * S::kStageBytes);
          auto load = [&](uint8_t* dst, const CUtensorMap* map, int x, int y) {
            if (leader) tma_load_tile(dst, map, sh.full(s), x, y);
            else tma_load_tile_pair(dst, map, map_to_rank(smem_u32(sh.full(s)), 0), x, y);
          };
          if (p.a_mn) {
            for (int j = 0; j < kGemmM / 64; ++j) load(sh.a(s) + j * 8192, am, arow + j * 64, kb * kGemmK);
          } else {
            load(sh.a(s), am, kb * kGemmK, arow);
          }
          if (p.b_mn) {
            for (int j = 0; j < S::kBRows / 64; ++j) load(sh.b(s) + j * 8192, bm, brow + j * 64, kb * kGemmK);
          } else {
            load(sh.b(s), bm, kb * kGemmK, brow);
          }
        }
      }
      if (!ok && leader) {
        // The leader's barriers count both CTAs' copies: wait (bounded) for what was armed.
        for (int j = max(0, it - kS); j < it; ++j) mbar_wait_drain(sh.full(j % kS), (j / kS) & 1);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------ MMA issuer -----------------------------
    if (elect_one_lane()) {
      if (leader) {
        int it = 0, n = 0;
        bool ok = true;
        for (int t = first; ok && t < total; t += step, ++n) {
          const TileAt w = tile_at(args, t);
          const GemmProblem& p = args.p[w.prob];
          const int acc = n & 1;
          if (!mbar_wait(sh.tempty(acc), ((n >> 1) & 1) ^ 1, abort, args.err, 34)) break;
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
          const bool a_mn = p.a_mn != 0, b_mn = p.b_mn != 0;
          const uint32_t idesc = gemm_idesc(CG * kGemmM, BN, args.bf16 != 0, a_mn, b_mn);
          const uint32_t a_step = a_mn ? 2048u : 32u, b_step = b_mn ? 2048u : 32u;
          const int k0 = w.split * p.kper, k1 = min(p.kblocks, k0 + p.kper);
          for (int kb = k0; kb < k1; ++kb, ++it) {
            const int s = it % kS;
            if (!mbar_wait(sh.full(s), (it / kS) & 1, abort, args.err, 35)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sa = smem_u32(sh.a(s)), sb = smem_u32(sh.b(s));
#pragma unroll
            for (int kk = 0; kk < kGemmK / 16; ++kk) {
              const uint64_t da = gemm_desc(sa + kk * a_step, a_mn), db = gemm_desc(sb + kk * b_step, b_mn);
              const uint32_t accumulate = (kb != k0 || kk != 0) ? 1u : 0u;
              if constexpr (CG == 2) tc_mma_f16_pair(d_tmem, da, db, idesc, accumulate);
              else tc_mma_f16(d_tmem, da, db, idesc, accumulate);
            }
            if constexpr (CG == 2) tc_commit_pair(sh.empty(s), 0x3);
            else tc_commit(sh.empty(s));
          }
          if (!ok) break;
          if constexpr (CG == 2) tc_commit_pair(sh.tfull(acc), 0x3);
          else tc_commit(sh.tfull(acc));
        }
        if constexpr (CG == 2) tc_commit_pair(sh.done(), 0x3);
        else tc_commit(sh.done());
      }
      // Both CTAs stay until every MMA, which reads both CTAs' shared memory, has retired.
      mbar_wait_drain(sh.done(), 0);
    }
    __syncwarp();
  } else {
    // ------------------------------ epilogue -------------------------------
    constexpr int kHalf = BN / 2;                  // columns per warp
    constexpr int kChunks = kHalf / S::kChunk;
    using Io = BlockIo<S::kUnits>;
    const int ew = warp - 2;
    const int sub = ew >> 2;
    const int quad = warp & 3;
    uint8_t* buf = sh.stage(ew);
    float* bias_s = sh.bias(ew);
    const bool bf16 = args.bf16 != 0;
    int n = 0;
    for (int t = first; t < total; t += step, ++n) {
      const TileAt w = tile_at(args, t);
      const GemmProblem& p = args.p[w.prob];
      const int acc = n & 1;
      const int row0 = (w.mt * CG + static_cast<int>(rank)) * kGemmM + quad * 32;
      const int col0 = w.nt * BN + sub * kHalf;
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) +
                             static_cast<uint32_t>(acc * BN + sub * kHalf);
      const int act = p.act;
      uint4 res[S::kUnits];
      if (p.residual)
        Io::load(p.residual, p.ld_res, p.vec_res != 0, row0, p.m, col0, p.n, lane, res);
      float bias_r[kHalf / 32];  // lane's column of every 32
#pragma unroll
      for (int i = 0; i < kHalf / 32; ++i)
        bias_r[i] = p.bias && col0 + 32 * i + lane < p.n ? half_at(p.bias, col0 + 32 * i + lane, bf16) : 0.f;
      if (!mbar_wait(sh.tfull(acc), (n >> 1) & 1, abort, args.err, 36)) break;
      tc_fence_after();
      if (p.partial) {
        // A part of K: fp32 sums in an order of our own (16 bytes per lane side by
        // side), added up by linear_finish_kernel.
        float* out = p.partial + ((static_cast<size_t>(w.split) * p.tiles_m * p.tiles_n + w.tile) * CG + rank) *
                                     (kGemmM * BN) + static_cast<size_t>(sub * 4 + quad) * (kHalf / 32) * 1024;
        for (int c = 0; c < kHalf / 32; ++c) {
          uint32_t r[32];
          tmem_ld32(taddr + c * 32, r);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(out + c * 1024 + j * 128 + lane * 4) =
                make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
        }
      } else {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int cc = col0 + c * S::kChunk;
          if (cc >= p.n) break;
          if (p.z) {
#pragma unroll
            for (int h = 0; h < S::kChunk / 32; ++h) {
              uint32_t r[32];
              tmem_ld32(taddr + c * S::kChunk + h * 32, r);
              __syncwarp();
              bias_s[lane] = bias_r[c * (S::kChunk / 32) + h];
              __syncwarp();
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int i = 8 * j + 2 * e;
                  float v0 = __uint_as_float(r[i]) + bias_s[i], v1 = __uint_as_float(r[i + 1]) + bias_s[i + 1];
                  if (act == kActRelu) {
                    // A positive z must stay positive in fp16: the backward pass reads its sign.
                    v0 = v0 > 0.f ? fmaxf(v0, 6e-8f) : v0;
                    v1 = v1 > 0.f ? fmaxf(v1, 6e-8f) : v1;
                  }
                  o[e] = pack2(v0, v1, false);
                }
                *reinterpret_cast<uint4*>(buf + Io::swizzle(lane, h * 4 + j)) = make_uint4(o[0], o[1], o[2], o[3]);
              }
            }
            __syncwarp();
            Io::store(p.z, p.ld_z, true, row0, p.m, cc, p.n, lane, buf);
            __syncwarp();
          }
          if (p.residual) {
            Io::stage(buf, lane, res);
            __syncwarp();
            if (c + 1 < kChunks)
              Io::load(p.residual, p.ld_res, p.vec_res != 0, row0, p.m, cc + S::kChunk, p.n, lane, res);
          }
#pragma unroll
          for (int h = 0; h < S::kChunk / 32; ++h) {
            uint32_t r[32];
            tmem_ld32(taddr + c * S::kChunk + h * 32, r);
            __syncwarp();
            bias_s[lane] = bias_r[c * (S::kChunk / 32) + h];
            __syncwarp();
            tmem_wait_ld();
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]) + bias_s[i];
            if (act == kActRelu) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = act_value(v[i], kActRelu);
            } else if (act == kActGelu) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = act_value(v[i], kActGelu);
            } else if (act == kActSilu) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = act_value(v[i], kActSilu);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint4* at = reinterpret_cast<uint4*>(buf + Io::swizzle(lane, h * 4 + j));
              if (p.residual) {
                const uint4 q = *at;
                const uint32_t qs[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float2 f = unpack2(qs[e], bf16);
                  v[8 * j + 2 * e] += f.x;
                  v[8 * j + 2 * e + 1] += f.y;
                }
              }
              uint32_t o[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) o[e] = pack2(v[8 * j + 2 * e], v[8 * j + 2 * e + 1], bf16);
              *at = make_uint4(o[0], o[1], o[2], o[3]);
            }
          }
          __syncwarp();
          Io::store(p.out, p.ld_out, p.vec_out != 0, row0, p.m, cc, p.n, lane, buf);
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (leader) mbar_arrive(sh.tempty(acc));
        else mbar_arrive_cluster(map_to_rank(smem_u32(sh.tempty(acc)), 0));
      }
    }
  }

  // The next kernel may be scheduled from here on. Not earlier: the kernels of this
  // file trigger only behind their last read of global memory, so that no later
  // kernel of a chain is resident (its L1 cache in use) while an input is still
  // being read whose memory the chain reuses for another kernel's result.
  grid_launch_dependents();
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2) tmem_dealloc_pair(tmem_base, S::kTmemCols);
    else tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// Few rows: the weights streamed once by CUDA cores
// ---------------------------------------------------------------------------
// One warp per output column: lanes split K in 16-byte steps, every weight is used
// for all ROWS rows, whose elements come from L1.
template <int ROWS>
__global__ void __launch_bounds__(256) linear_small_kernel(const LinearSmallArgs a) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int col = static_cast<int>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (col >= a.n) return;
  const bool bf16 = a.bf16 != 0;
  const uint16_t* w = static_cast<const uint16_t*>(a.w) + static_cast<long long>(col) * a.ld_w;
  const uint16_t* x = static_cast<const uint16_t*>(a.x);
  float acc[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) acc[r] = 0.f;
  if (a.vec) {
    for (int c = lane * 8; c < a.k; c += 256) {
      const uint4 wv = *reinterpret_cast<const uint4*>(w + c);
      const uint32_t ws[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (r < a.m) {
          const uint4 xv = *reinterpret_cast<const uint4*>(x + r * a.ld_x + c);
          const uint32_t xs[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 fw = unpack2(ws[e], bf16), fx = unpack2(xs[e], bf16);
            acc[r] = fmaf(fw.x, fx.x, acc[r]);
            acc[r] = fmaf(fw.y, fx.y, acc[r]);
          }
        }
      }
    }
  } else {
    for (int c = lane; c < a.k; c += 32) {
      const float fw = half_at(w, c, bf16);
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        if (r < a.m) acc[r] = fmaf(fw, half_at(x, r * a.ld_x + c, bf16), acc[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) acc[r] = warp_sum(acc[r]);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (lane != r || r >= a.m) continue;
    float v = acc[r];
    if (a.bias) v += half_at(a.bias, col, bf16);
    if (a.z) {
      const float kept = a.act == kActRelu && v > 0.f ? fmaxf(v, 6e-8f) : v;
      static_cast<__half*>(a.z)[r * a.ld_z + col] = __float2half_rn(kept);
    }
    v = act_value(v, a.act);
    if (a.residual) v += half_at(a.residual, r * a.ld_res + col, bf16);
    static_cast<uint16_t*>(a.out)[r * a.ld_out + col] = half_bits(v, bf16);
  }
}

// ---------------------------------------------------------------------------
// Backward: dz and the columns' sums
// ---------------------------------------------------------------------------
constexpr int kDzCols = 256;  // columns per block: one warp reads 32 x 16 bytes of a row
constexpr int kDzWarps = 8;

// dz = dy act'(z) in the rows' type (skipped where dz is null: no activation), and
// the block's share of every column's sum, in fp32 from the unrounded dz.
__global__ void __launch_bounds__(32 * kDzWarps) linear_dz_kernel(const LinearDzArgs a) {
  grid_dependency_wait();
  __shared__ float sums[kDzWarps][kDzCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = static_cast<int>(blockIdx.x) * kDzCols + lane * 8;
  const bool bf16 = a.bf16 != 0;
  float s[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) s[t] = 0.f;
  if (c < a.n) {
    const bool whole = c + 8 <= a.n;
    for (long long row = static_cast<long long>(blockIdx.y) * kDzWarps + warp; row < a.m;
         row += static_cast<long long>(gridDim.y) * kDzWarps) {
      uint32_t g[4] = {0u, 0u, 0u, 0u};
      const uint16_t* dy = static_cast<const uint16_t*>(a.dy) + row * a.ld_dy + c;
      if (a.vec_dy && whole) {
        const uint4 v = *reinterpret_cast<const uint4*>(dy);
        g[0] = v.x, g[1] = v.y, g[2] = v.z, g[3] = v.w;
      } else {
#pragma unroll
        for (int t = 0; t < 8; ++t)
          if (c + t < a.n) g[t / 2] |= static_cast<uint32_t>(dy[t]) << (16 * (t & 1));
      }
      float f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 v = unpack2(g[e], bf16);
        f[2 * e] = v.x;
        f[2 * e + 1] = v.y;
      }
      if (a.z) {  // z's rows are padded to whole 16-byte units
        const uint4 zv = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.z) + row * a.ld_z + c);
        const uint32_t zs[4] = {zv.x, zv.y, zv.z, zv.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 v = unpack2(zs[e], false);
          if (c + 2 * e < a.n) f[2 * e] *= act_slope(v.x, a.act);
          if (c + 2 * e + 1 < a.n) f[2 * e + 1] *= act_slope(v.y, a.act);
        }
      }
      if (a.dz) {
        uint4 o;
        o.x = pack2(f[0], f[1], bf16);
        o.y = pack2(f[2], f[3], bf16);
        o.z = pack2(f[4], f[5], bf16);
        o.w = pack2(f[6], f[7], bf16);
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.dz) + row * a.ld_dz + c) = o;
      }
#pragma unroll
      for (int t = 0; t < 8; ++t) s[t] += f[t];
    }
  }
  if (a.partial == nullptr) return;
#pragma unroll
  for (int t = 0; t < 8; ++t) sums[warp][lane * 8 + t] = s[t];
  __syncthreads();
  const int col = static_cast<int>(blockIdx.x) * kDzCols + threadIdx.x;
  if (col >= a.n) return;
  float v = 0.f;
#pragma unroll
  for (int w = 0; w < kDzWarps; ++w) v += sums[w][threadIdx.x];
  a.partial[static_cast<size_t>(blockIdx.y) * a.n + col] = v;
}

// Adds the parts in a fixed order: blocks below db_blocks sum dbias (32 columns
// each), the others one 32 x 32 piece of dw per warp.
__global__ void __launch_bounds__(256) linear_finish_kernel(const LinearFinishArgs a) {
  grid_dependency_wait();
  const bool bf16 = a.bf16 != 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __shared__ float sums[8][33];
  __shared__ uint16_t piece[8][32][34];
  if (static_cast<int>(blockIdx.x) < a.db_blocks) {
    const int c = static_cast<int>(blockIdx.x) * 32 + lane;
    float s = 0.f;
    if (c < a.n)
      for (int b = warp; b < a.db_parts; b += 8) s += a.db_partial[static_cast<size_t>(b) * a.n + c];
    sums[warp][lane] = s;
    __syncthreads();
    if (warp != 0 || c >= a.n) return;
    for (int w = 1; w < 8; ++w) s += sums[w][lane];
    static_cast<uint16_t*>(a.dbias)[c] = half_bits(s, bf16);
    return;
  }
  // Piece: [tile][rank][sub][quad][chunk of 32 columns], as gemm_kernel wrote it.
  const int per_tile = a.cg * 8 * (a.bn / 64);
  const int piece_id = (static_cast<int>(blockIdx.x) - a.db_blocks) * 8 + warp;
  if (piece_id >= a.tiles_m * a.tiles_n * per_tile) return;
  const int tile = piece_id / per_tile;
  int i = piece_id - tile * per_tile;
  const int rank = i / (8 * (a.bn / 64));
  i -= rank * 8 * (a.bn / 64);
  const int sub = i / (4 * (a.bn / 64));
  i -= sub * 4 * (a.bn / 64);
  const int quad = i / (a.bn / 64), chunk = i % (a.bn / 64);
  const size_t tile_floats = static_cast<size_t>(kGemmM) * a.bn;
  const float* src = a.dw_partial + (static_cast<size_t>(tile) * a.cg + rank) * tile_floats +
                     (static_cast<size_t>(sub * 4 + quad) * (a.bn / 64) + chunk) * 1024 + lane * 4;
  const size_t split_stride = static_cast<size_t>(a.tiles_m) * a.tiles_n * a.cg * tile_floats;
  float v[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = 0.f;
  for (int s = 0; s < a.splits; ++s) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 f = *reinterpret_cast<const float4*>(src + s * split_stride + j * 128);
      v[4 * j] += f.x;
      v[4 * j + 1] += f.y;
      v[4 * j + 2] += f.z;
      v[4 * j + 3] += f.w;
    }
  }
  const int group = tile / (8 * a.tiles_n);
  const int rows = min(8, a.tiles_m - group * 8);
  const int in_group = tile - group * 8 * a.tiles_n;
  const int row0 = ((group * 8 + in_group % rows) * a.cg + rank) * kGemmM + quad * 32;
  const int col0 = (in_group / rows) * a.bn + sub * (a.bn / 2) + chunk * 32;
#pragma unroll
  for (int j = 0; j < 32; ++j) piece[warp][lane][j] = half_bits(v[j], bf16);
  __syncwarp();
  if (col0 + lane < a.k) {
    for (int r = 0; r < 32 && row0 + r < a.n; ++r)
      static_cast<uint16_t*>(a.dw)[static_cast<long long>(row0 + r) * a.ld_dw + col0 + lane] = piece[warp][r][lane];
  }
}

template <int CG, int BN>
cudaError_t gemm_launch_one(const CUtensorMap (&maps)[4], const GemmArgs& a, int ctas, cudaStream_t stream) {
  using S = GemmShape<CG, BN>;
  constexpr int smem = S::kTotal + 1024;
  auto kern = gemm_kernel<CG, BN>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, maps[0], maps[1], maps[2], maps[3], a);
}

}  // namespace

cudaError_t gemm_launch(int cg, int bn, const CUtensorMap (&maps)[4], const GemmArgs& a, int ctas, cudaStream_t stream) {
  if (cg == 2 && bn == 256) return gemm_launch_one<2, 256>(maps, a, ctas, stream);
  if (cg == 1 && bn == 128) return gemm_launch_one<1, 128>(maps, a, ctas, stream);
  if (cg == 1 && bn == 64) return gemm_launch_one<1, 64>(maps, a, ctas, stream);
  return cudaErrorInvalidValue;
}

cudaError_t linear_small_launch(const LinearSmallArgs& a, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((a.n + 7) / 8));
  if (a.m <= 1) return launch_programmatic(linear_small_kernel<1>, grid, dim3(256), 0, stream, a);
  if (a.m <= 2) return launch_programmatic(linear_small_kernel<2>, grid, dim3(256), 0, stream, a);
  if (a.m <= 4) return launch_programmatic(linear_small_kernel<4>, grid, dim3(256), 0, stream, a);
  if (a.m <= kLinearSmallRows) return launch_programmatic(linear_small_kernel<8>, grid, dim3(256), 0, stream, a);
  return cudaErrorInvalidValue;
}

int linear_dz_parts(long long m, int n, int num_sms) {
  const int cols = (n + kDzCols - 1) / kDzCols;
  const long long want = std::max(1, 8 * num_sms / cols);
  return static_cast<int>(std::max<long long>(1, std::min<long long>(want, (m + kDzWarps - 1) / kDzWarps)));
}

cudaError_t linear_dz_launch(const LinearDzArgs& a, int parts, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((a.n + kDzCols - 1) / kDzCols), static_cast<unsigned>(parts));
  return launch_programmatic(linear_dz_kernel, grid, dim3(32 * kDzWarps), 0, stream, a);
}

cudaError_t linear_finish_launch(const LinearFinishArgs& a, cudaStream_t stream) {
  const int pieces = a.dw_partial ? a.tiles_m * a.tiles_n * a.cg * 8 * (a.bn / 64) : 0;
  const int grid = a.db_blocks + (pieces + 7) / 8;
  if (grid == 0) return cudaSuccess;
  return launch_programmatic(linear_finish_kernel, dim3(static_cast<unsigned>(grid)), dim3(256), 0, stream, a);
}

}  // namespace cvs
