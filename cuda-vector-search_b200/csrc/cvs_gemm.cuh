// The linear layer's tcgen05 product with its epilogue (gemm_kernel), and the element
// arithmetic that the layer's other kernels share with it (activations, their slopes,
// half-precision packing). Included by one translation unit per activation, which
// instantiates the kernel for it, and by cvs_linear.cu.
#pragma once

#include "cvs_device.cuh"
#include "cvs_elem.cuh"
#include "cvs_kernels.h"

#include <algorithm>
#include <atomic>

namespace cvs {

namespace {

// ---------------------------------------------------------------------------
// Activations
// ---------------------------------------------------------------------------
// GELU z Phi(z) = max(z, 0) - |z| Q(|z|) with the tail probability Q(a) = Phi(-a) as
// 2^P(-a): log2 Q is smooth and nearly quadratic, so a degree-8 polynomial does. It is a
// least-squares fit on 0 .. 13.3 reweighted towards the smallest largest share of what is
// allowed: an error of Q that stays a fixed number of roundings of |z| (12 e are reached, e =
// 2^-24), and 2e-5 of Q itself up to 6, growing to 1e-2 at the end. Reached: 5e-5 of Q up to
// 6, 5e-4 up to 9, 1.2e-3 up to 11 and 1.4e-2 up to 12.95, where Q passes fp32's smallest
// normal number and becomes zero; bf16, which has fp32's range, sees all of it. It costs eight
// multiply-adds, on pairs (fma.rn.f32x2: two elements an instruction), and one ex2. With erff
// the epilogue, not the tensor cores, set the pace: 16384 x 768 -> 1536 took 112 us, against
// 47 us without an activation.
constexpr float kTailEnd = 13.3f;
constexpr int kTailDegree = 8;
__device__ constexpr float kTail[kTailDegree + 1] = {-0.9999980330467224f, 1.1511892080307007f, -0.4586566388607025f,
                                                    0.0537852942943573f, 0.00846633780747652f, 0.0009411636856384575f,
                                                    6.787561142118648e-05f, 2.80283438769402e-06f, 4.9737455043441514e-08f};
constexpr float kLog2E = 1.4426950408889634f;

// The larger (smaller) of the two; NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Q(-b) of two elements, b = max(-|z|, -kTailEnd).
__device__ __forceinline__ void tail_pair(Pair b, float& q0, float& q1) {
  Pair p = both(kTail[kTailDegree]);
#pragma unroll
  for (int i = kTailDegree - 1; i >= 0; --i) p = pair_fma(p, b, both(kTail[i]));
  float p0, p1;
  split(p, p0, p1);
  q0 = exp2_approx(p0);
  q1 = exp2_approx(p1);
}

template <int ACT>
__device__ __forceinline__ void act_pair(float& z0, float& z1) {
  if constexpr (ACT == kActRelu) {
    z0 = max_nan(z0, 0.f);
    z1 = max_nan(z1, 0.f);
  } else if constexpr (ACT == kActGelu) {
    const Pair b = pair_of(fmaxf(-fabsf(z0), -kTailEnd), fmaxf(-fabsf(z1), -kTailEnd));
    float q0, q1;
    tail_pair(b, q0, q1);
    split(pair_fma(b, pair_of(q0, q1), pair_of(max_nan(z0, 0.f), max_nan(z1, 0.f))), z0, z1);
  } else if constexpr (ACT == kActSilu) {
    float e0, e1;
    split(pair_mul(pair_of(z0, z1), pair_of(-kLog2E, -kLog2E)), e0, e1);
    z0 *= rcp_approx(1.f + exp2_approx(e0));
    z1 *= rcp_approx(1.f + exp2_approx(e1));
  }
}

template <int ACT, int N>
__device__ __forceinline__ void act_values(float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) act_pair<ACT>(v[i], v[i + 1]);
}

template <int N>
__device__ __forceinline__ void act_values(float (&v)[N], int act) {
  if (act == kActRelu) act_values<kActRelu>(v);
  else if (act == kActGelu) act_values<kActGelu>(v);
  else if (act == kActSilu) act_values<kActSilu>(v);
}

// g act'(z) for two elements. Beyond +-30 the slopes are 0 and 1 to the last bit; the
// clamp keeps an infinite z (an overflowed fp16 pre-activation) from giving inf x 0 and
// passes NaN on.
template <int ACT>
__device__ __forceinline__ void slope_pair(float z0, float z1, float& g0, float& g1) {
  if constexpr (ACT == kActRelu) {
    g0 = z0 > 0.f ? g0 : (z0 != z0 ? z0 : 0.f);
    g1 = z1 > 0.f ? g1 : (z1 != z1 ? z1 : 0.f);
    return;
  }
  const float c0 = min_nan(max_nan(z0, -30.f), 30.f), c1 = min_nan(max_nan(z1, -30.f), 30.f);
  if constexpr (ACT == kActGelu) {
    // Phi(z) + z phi(z), phi(z) = 2^(-z^2 log2(e) / 2) / sqrt(2 pi).
    float q0, q1, e0, e1;
    tail_pair(pair_of(fmaxf(-fabsf(c0), -kTailEnd), fmaxf(-fabsf(c1), -kTailEnd)), q0, q1);
    const Pair c = pair_of(c0, c1);
    split(pair_mul(pair_mul(c, both(-0.5f * kLog2E)), c), e0, e1);
    const Pair phi = pair_of(exp2_approx(e0), exp2_approx(e1));
    const Pair cdf = pair_of(c0 > 0.f ? 1.f - q0 : q0, c1 > 0.f ? 1.f - q1 : q1);
    const Pair s = pair_fma(pair_mul(c, both(0.39894228040143268f)), phi, cdf);
    split(pair_mul(s, pair_of(g0, g1)), g0, g1);
  } else {
    float e0, e1;
    split(pair_mul(pair_of(c0, c1), both(-kLog2E)), e0, e1);
    const Pair s = pair_of(rcp_approx(1.f + exp2_approx(e0)), rcp_approx(1.f + exp2_approx(e1)));
    // s (1 + z (1 - s))
    const Pair t = pair_fma(pair_of(c0, c1), pair_fma(s, both(-1.f), both(1.f)), both(1.f));
    split(pair_mul(pair_mul(s, t), pair_of(g0, g1)), g0, g1);
  }
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

// Eight halves of a row from column c on (columns outside read as zero).
__device__ __forceinline__ uint4 load_unit8(const uint16_t* p, int c, int n, bool vec) {
  if (vec && c + 8 <= n) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int t = 0; t < 8; ++t)
    if (c + t < n) w[t / 2] |= static_cast<uint32_t>(p[t]) << (16 * (t & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// ---------------------------------------------------------------------------
// tcgen05 product
// ---------------------------------------------------------------------------
constexpr int kGemmM = 128;   // rows of the output tile per CTA (TMEM lanes)
constexpr int kGemmK = 64;    // halves per K slice: one 128-byte swizzled row
constexpr int kGemmMaxStages = 8;
constexpr int kBufBytes = 32 * 64 * 2;  // one staging buffer: 32 rows x 64 columns of halves, 128-byte swizzled

// Epilogue warps: four quadrants of 32 TMEM lanes x column halves (tiles of 64
// columns are not halved).
__host__ __device__ constexpr int gemm_subs(int bn) { return bn >= 128 ? 2 : 1; }

// Shared memory: ring of operand stages, then per epilogue warp two staging buffers
// and 32 columns' bias, then the barriers.
template <int CG, int BN>
struct GemmShape {
  static constexpr int kSubs = gemm_subs(BN);
  static constexpr int kEpiWarps = 4 * kSubs;
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kBRows = BN / CG;                    // columns of the tile whose operand rows this CTA loads
  static constexpr int kABytes = kGemmM * kGemmK * 2;
  static constexpr int kBBytes = kBRows * kGemmK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kBiasBytes = kEpiWarps * 32 * 4;
  static constexpr int kBars = 2 * kGemmMaxStages + 5 + 2 * kEpiWarps;
  static constexpr int kTail = kEpiWarps * 2 * kBufBytes + kBiasBytes + 8 * kBars + 16;
  static constexpr int kFit = (kSmemBudget - kTail) / kStageBytes;
  static constexpr int kStages = kFit < kGemmMaxStages ? kFit : kGemmMaxStages;
  static constexpr int kBufs = kStages * kStageBytes;       // offset of the staging buffers
  static constexpr int kBias = kBufs + kEpiWarps * 2 * kBufBytes;
  static constexpr int kTotal = kBufs + kTail;
  static constexpr uint32_t kTmemCols = 2 * BN;
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

// A staging buffer holds 32 rows x 64 columns of halves as the tensor-memory
// accelerator lays them out (128-byte rows whose 16-byte units are swapped by the
// row's low three bits), so that it can move the block to and from global memory;
// one row per lane meets no bank twice.
__device__ __forceinline__ int buf_at(int row, int unit) { return row * 128 + ((unit ^ (row & 7)) << 4); }

// One row per lane, columns 32 h .. 32 h + 31 of the buffer.
__device__ __forceinline__ void buf_put(uint8_t* buf, int lane, int h, const float (&v)[32], bool bf16) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(buf + buf_at(lane, 4 * h + j)) =
        make_uint4(pack2(v[8 * j], v[8 * j + 1], bf16), pack2(v[8 * j + 2], v[8 * j + 3], bf16),
                   pack2(v[8 * j + 4], v[8 * j + 5], bf16), pack2(v[8 * j + 6], v[8 * j + 7], bf16));
}

__device__ __forceinline__ void buf_add(const uint8_t* buf, int lane, int h, float (&v)[32], bool bf16) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 q = *reinterpret_cast<const uint4*>(buf + buf_at(lane, 4 * h + j));
    const uint32_t qs[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack2(qs[e], bf16);
      v[8 * j + 2 * e] += f.x;
      v[8 * j + 2 * e + 1] += f.y;
    }
  }
}

// The block between its buffer and rows of any alignment: lane = column, so that a
// warp's two-byte accesses are consecutive. Functions of their own, called where the
// accelerator cannot address the rows: inlined, their code stretched the epilogue that
// never calls them (16384 x 768 -> 1536, GELU and residual: 71 us against 46).
__device__ __noinline__ void buf_to_rows(const uint8_t* buf, void* dst, long long ld, int row0, int rows, int col0,
                                            int cols, int lane) {
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += 16) {
    uint16_t v[16][2];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = lane + 32 * h;
        v[r][h] = *reinterpret_cast<const uint16_t*>(buf + buf_at(r0 + r, c >> 3) + 2 * (c & 7));
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      uint16_t* p = static_cast<uint16_t*>(dst) + (row0 + r0 + r) * ld + col0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = lane + 32 * h;
        if (row0 + r0 + r < rows && col0 + c < cols) p[c] = v[r][h];
      }
    }
  }
}
__device__ __noinline__ void rows_to_buf(uint8_t* buf, const void* src, long long ld, int row0, int rows, int col0,
                                            int cols, int lane) {
  // Sixteen rows' loads are under way before the first of them is staged.
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += 16) {
    uint16_t v[16][2];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const uint16_t* p = static_cast<const uint16_t*>(src) + (row0 + r0 + r) * ld + col0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = lane + 32 * h;
        v[r][h] = row0 + r0 + r < rows && col0 + c < cols ? p[c] : static_cast<uint16_t>(0);
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = lane + 32 * h;
        *reinterpret_cast<uint16_t*>(buf + buf_at(r0 + r, c >> 3) + 2 * (c & 7)) = v[r][h];
      }
    }
  }
}

// Bulk stores of a staging buffer: issued and waited for by one lane per warp.
__device__ __forceinline__ void tma_store_tile(const void* desc, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(desc)),
               "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// All but the last N groups have read their buffers.
template <int N>
__device__ __forceinline__ void tma_store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
// This thread's writes to shared memory are visible to the copies issued after it.
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Waits for this thread's tensor-memory loads; the values are not used before.
__device__ __forceinline__ void tmem_wait_ld32(uint32_t (&r)[32]) {
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i])::"memory");
}

template <int CG, int BN>
struct GemmShared {
  using S = GemmShape<CG, BN>;
  uint8_t* base;
  __device__ uint8_t* a(int s) const { return base + s * S::kStageBytes; }
  __device__ uint8_t* b(int s) const { return base + s * S::kStageBytes + S::kABytes; }
  __device__ uint8_t* buf(int w) const { return base + S::kBufs + w * 2 * kBufBytes; }
  __device__ float* bias(int w) const { return reinterpret_cast<float*>(base + S::kBias) + w * 32; }
  __device__ uint64_t* bar(int i) const { return reinterpret_cast<uint64_t*>(base + S::kBias + S::kBiasBytes) + i; }
  __device__ uint64_t* full(int s) const { return bar(s); }
  __device__ uint64_t* empty(int s) const { return bar(kGemmMaxStages + s); }
  __device__ uint64_t* tfull(int i) const { return bar(2 * kGemmMaxStages + i); }
  __device__ uint64_t* tempty(int i) const { return bar(2 * kGemmMaxStages + 2 + i); }
  __device__ uint64_t* done() const { return bar(2 * kGemmMaxStages + 4); }
  __device__ uint64_t* rfull(int w, int b) const { return bar(2 * kGemmMaxStages + 5 + 2 * w + b); }
  __device__ uint32_t* tmem_holder() const { return reinterpret_cast<uint32_t*>(bar(S::kBars)); }
  __device__ volatile int* abort_flag() const { return reinterpret_cast<volatile int*>(bar(S::kBars)) + 1; }
};

// One CTA (CG = 1, 128 x BN tiles) or a pair of CTAs (CG = 2, 256 x BN tiles; each
// CTA holds its 128 rows of A and half of B's rows) per work item, persistent over
// the call's tiles: warp 0 loads, warp 1 issues the MMAs, 4 or 8 warps drain one of two
// accumulators while the other is computed. Results leave, and residuals arrive, as
// 32 x 64 blocks moved by the tensor-memory accelerator through each warp's two staging
// buffers (rows it cannot address, by ordinary accesses): a residual is requested one
// block ahead, into the buffer whose block has just left. Waits are bounded (cvs_device.cuh); a
// wait that runs out stops every role of the CTA, and the pair still meets at the
// last barrier.
//
// The activation, the residual (RES) and the kept pre-activation (Z) are template
// arguments: with all of them in one kernel the epilogue's code, one copy per 32
// columns, spread over more than the instruction caches hold, and fetching it took
// longer than running it. Cycles a tile's epilogue takes at 16384 x 768 -> 1536, one
// kernel for all / one for each: bias alone 7168 / 3766, GELU 10154 / 7936, GELU and
// residual 16229 / 9753, GELU and z 11257 / 8939; the tile's products take at least 6144.
template <int CG, int BN, int ACT, bool RES, bool Z>
__global__ void __launch_bounds__(GemmShape<CG, BN>::kThreads, 1)
    gemm_kernel(const __grid_constant__ GemmMaps maps, const __grid_constant__ GemmArgs args) {
  using S = GemmShape<CG, BN>;
  constexpr int kS = S::kStages;
  constexpr bool kParts = ACT == kActNone && !RES && !Z;  // products of the backward pass, whose K may be cut
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
      mbar_init(sh.tempty(t), leader ? CG * S::kEpiWarps : 1);
    }
    for (int w = 0; w < S::kEpiWarps; ++w) {
      mbar_init(sh.rfull(w, 0), 1);
      mbar_init(sh.rfull(w, 1), 1);
    }
    mbar_init(sh.done(), 1);
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&maps.a[0]);
    tma_prefetch_desc(&maps.b[0]);
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
        const CUtensorMap* am = &maps.a[w.prob];
        const CUtensorMap* bm = &maps.b[w.prob];
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
    constexpr int kHalf = BN / S::kSubs;  // columns per warp
    constexpr int kSteps = kHalf / 32, kChunks = kHalf / 64;
    const int ew = warp - 2;
    const int sub = ew >> 2;
    const int quad = warp & 3;
    uint8_t* bufs = sh.buf(ew);
    float* bias_s = sh.bias(ew);
    const bool bf16 = args.bf16 != 0;
    // Where this warp's part of a work item lies.
    const auto row_of = [&](const TileAt& w) { return (w.mt * CG + static_cast<int>(rank)) * kGemmM + quad * 32; };
    const auto col_of = [&](const TileAt& w) { return w.nt * BN + sub * kHalf; };
    // Requests the residual of one block into buffer b (one lane).
    const auto request = [&](int t, int chunk, int b) {
      if (t >= total) return;
      const TileAt w = tile_at(args, t);
      const GemmProblem& p = args.p[w.prob];
      const int row = row_of(w), col = col_of(w) + 64 * chunk;
      if (!p.vec_res || row >= p.m || col >= p.n) return;
      mbar_arrive_expect_tx(sh.rfull(ew, b), kBufBytes);
      tma_load_tile(bufs + b * kBufBytes, &maps.residual, sh.rfull(ew, b), col, row);
    };
    // Only a call's first product has a residual or keeps z. With z the second buffer
    // is z's, and a residual is requested when its own block begins.
    const bool ahead = RES && args.p[0].vec_res && !Z;
    if (ahead && lane == 0) request(first, 0, 0);
    uint32_t rphase = 0;  // bit b: parity of buffer b's next residual
    bool ok = true;
    int n = 0;
    for (int t = first; t < total; t += step, ++n) {
      const TileAt w = tile_at(args, t);
      const GemmProblem& p = args.p[w.prob];
      const int acc = n & 1;
      const int row0 = row_of(w), col0 = col_of(w);
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) +
                             static_cast<uint32_t>(acc * BN + sub * kHalf);
      float bias_r[kSteps];  // lane's column of every 32
#pragma unroll
      for (int c = 0; c < kSteps; ++c)
        bias_r[c] = p.bias && col0 + 32 * c + lane < p.n ? half_at(p.bias, col0 + 32 * c + lane, bf16) : 0.f;
      // One answer for the warp: what follows is done by all its lanes or by none.
      if (!__all_sync(0xffffffffu, mbar_wait(sh.tfull(acc), (n >> 1) & 1, abort, args.err, 36))) break;
      tc_fence_after();
      // The accumulator is free once its last 32 columns are in registers.
      const auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (leader) mbar_arrive(sh.tempty(acc));
          else mbar_arrive_cluster(map_to_rank(smem_u32(sh.tempty(acc)), 0));
        }
      };
      uint32_t r[2][32];
      tmem_ld32(taddr, r[0]);
      // A part of K: fp32 sums in an order of our own (16 bytes per lane side by
      // side), added up by linear_finish_kernel.
      float* part = kParts && p.partial ? p.partial + ((static_cast<size_t>(w.split) * p.tiles_m * p.tiles_n + w.tile) * CG + rank) *
                                                (kGemmM * BN) + static_cast<size_t>(sub * 4 + quad) * kSteps * 1024
                              : nullptr;
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        uint32_t (&now)[32] = r[c & 1];
        tmem_wait_ld32(now);
        if (c + 1 < kSteps) tmem_ld32(taddr + (c + 1) * 32, r[(c + 1) & 1]);
        else release();
        const int cc = col0 + 32 * (c & ~1);  // first column of the 64-column block
        if (part) {
          if (col0 + 32 * c < p.n) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<uint4*>(part + c * 1024 + j * 128 + lane * 4) =
                  make_uint4(now[4 * j], now[4 * j + 1], now[4 * j + 2], now[4 * j + 3]);
          }
          continue;
        }
        const int b = Z ? 0 : (n * kChunks + (c >> 1)) & 1;
        uint8_t* buf = bufs + b * kBufBytes;
        const bool live = row0 < p.m && cc < p.n;
        if (RES && (c & 1) == 0) {
          // The residual's block comes into the buffer that its result will leave from,
          // one block ahead into the other buffer where that is free.
          if (lane == 0) {
            tma_store_wait_read<0>();
            if (!ahead) request(t, c >> 1, b);
            else if (c + 2 < kSteps) request(t, (c >> 1) + 1, b ^ 1);
            else request(t + step, 0, b ^ 1);
          }
          __syncwarp();
          if (live && !p.vec_res) {
            rows_to_buf(buf, p.residual, p.ld_res, row0, p.m, cc, p.n, lane);
            __syncwarp();
          }
        }
        if (!live) {
          // An empty group, so that "all but the last group" still means the other buffer's.
          if ((c & 1) != 0 && lane == 0) tma_store_commit();
          continue;
        }
        float v[32];
        if (p.bias) {
          bias_s[lane] = bias_r[c];
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 b4 = *reinterpret_cast<const float4*>(bias_s + i);
            split(pair_add(pair_of(__uint_as_float(now[i]), __uint_as_float(now[i + 1])), pair_of(b4.x, b4.y)), v[i], v[i + 1]);
            split(pair_add(pair_of(__uint_as_float(now[i + 2]), __uint_as_float(now[i + 3])), pair_of(b4.z, b4.w)), v[i + 2],
                  v[i + 3]);
          }
          __syncwarp();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(now[i]);
        }
        if (!RES && (c & 1) == 0) {
          // A new block's first values: its buffers' last blocks have left.
          if (lane == 0) {
            if constexpr (Z) tma_store_wait_read<0>();
            else tma_store_wait_read<1>();
          }
          __syncwarp();
        }
        if constexpr (Z) {
          if constexpr (ACT == kActRelu) {
            // A positive z must stay positive in fp16: the backward pass reads its sign.
            float kept[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) kept[i] = v[i] > 0.f ? fmaxf(v[i], 6e-8f) : v[i];
            buf_put(bufs + kBufBytes, lane, c & 1, kept, false);
          } else {
            buf_put(bufs + kBufBytes, lane, c & 1, v, false);
          }
        }
        act_values<ACT>(v);
        if constexpr (RES) {
          if (p.vec_res && (c & 1) == 0) {
            ok = __all_sync(0xffffffffu, mbar_wait(sh.rfull(ew, b), (rphase >> b) & 1, abort, args.err, 37)) && ok;
            rphase ^= 1u << b;
          }
          buf_add(buf, lane, c & 1, v, bf16);
        }
        buf_put(buf, lane, c & 1, v, bf16);
        if ((c & 1) == 0) continue;
        fence_async_proxy();
        __syncwarp();
        if (lane == 0) {
          if constexpr (Z) tma_store_tile(&maps.z, bufs + kBufBytes, cc, row0);
          if (p.vec_out) tma_store_tile(&maps.out[w.prob], buf, cc, row0);
          tma_store_commit();
        }
        if (!p.vec_out) {
          buf_to_rows(buf, p.out, p.ld_out, row0, p.m, cc, p.n, lane);
          fence_async_proxy();  // the buffer's next content may be a residual's copy
          __syncwarp();
        }
      }
      if (!ok) break;
    }
    // Nothing of this warp's is in flight when the block ends. After a wait that ran
    // out that may be residuals' copies (at most one per buffer), else only stores.
    if (RES && *abort && lane == 0) {
      mbar_wait_drain(sh.rfull(ew, 0), rphase & 1);
      mbar_wait_drain(sh.rfull(ew, 1), rphase >> 1);
    }
    if (lane == 0) tma_store_wait_read<0>();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  // The next kernel may be scheduled from here on. Not earlier: no kernel of a forward
  // pass triggers before all its warps' last read of global memory, so that no later
  // kernel of a chain is resident (its L1 cache in use) while an input is still being
  // read whose memory the chain reuses for another kernel's result.
  grid_launch_dependents();
  if constexpr (CG == 2) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2) tmem_dealloc_pair(tmem_base, S::kTmemCols);
    else tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

template <int CG, int BN, int ACT, bool RES, bool Z>
cudaError_t gemm_launch_one(const GemmMaps& maps, const GemmArgs& a, int ctas, cudaStream_t stream) {
  using S = GemmShape<CG, BN>;
  constexpr int smem = S::kTotal + 1024;
  auto kern = gemm_kernel<CG, BN, ACT, RES, Z>;
  static std::atomic<unsigned long long> allowed{0};
  const cudaError_t e = allow_smem(kern, smem, allowed);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(S::kThreads);
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
  return cudaLaunchKernelEx(&cfg, kern, maps, a);
}

template <int ACT, bool RES, bool Z>
cudaError_t gemm_launch_tile(int cg, int bn, const GemmMaps& maps, const GemmArgs& a, int ctas, cudaStream_t stream) {
  if (cg == 2 && bn == 256) return gemm_launch_one<2, 256, ACT, RES, Z>(maps, a, ctas, stream);
  if (cg == 1 && bn == 128) return gemm_launch_one<1, 128, ACT, RES, Z>(maps, a, ctas, stream);
  if (cg == 1 && bn == 64) return gemm_launch_one<1, 64, ACT, RES, Z>(maps, a, ctas, stream);
  return cudaErrorInvalidValue;
}

// Without an activation nothing needs z.
template <int ACT>
cudaError_t gemm_launch_act(int cg, int bn, const GemmMaps& maps, const GemmArgs& a, int ctas, cudaStream_t stream) {
  const bool res = a.p[0].residual != nullptr;
  if constexpr (ACT != kActNone) {
    if (a.p[0].z != nullptr)
      return res ? gemm_launch_tile<ACT, true, true>(cg, bn, maps, a, ctas, stream)
                 : gemm_launch_tile<ACT, false, true>(cg, bn, maps, a, ctas, stream);
  }
  return res ? gemm_launch_tile<ACT, true, false>(cg, bn, maps, a, ctas, stream)
             : gemm_launch_tile<ACT, false, false>(cg, bn, maps, a, ctas, stream);
}

}  // namespace
}  // namespace cvs
