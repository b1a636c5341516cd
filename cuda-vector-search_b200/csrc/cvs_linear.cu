// Linear layer with bias, activation and residual, forward and backward.
//
//   forward    z = x w^T + bias,  y = act(z) + residual       (x [m][k], w [n][k])
//   backward   dz = dy act'(z),  dx = dz w,  dw = dz^T x,  dbias = sum of dz's rows
//
// The three products run on the fifth-generation tensor cores (tcgen05.mma, fp32
// accumulators in TMEM) fed by TMA, in one kernel (cvs_gemm.cuh): its operand tiles are K-major
// or MN-major per product (the matrix descriptor says which), so dx reads w and dw
// reads dz and x as they lie in memory, without a transposed copy. Everything after
// the product -- bias, activation, residual, the rounding to the rows' type -- is
// done on the accumulator before it leaves the SM.
//
// Bound: 2 m n k operations at the tensor cores' rate for batches of thousands of rows;
// below that latency and the weights' bytes, where split_kernel shares K among a cluster
// and linear_small_kernel (one row, two narrow ones) streams the weights once with CUDA cores.
// Measured: 131072 x 1536 -> 768 bf16 with bias 234-240 us at an SM clock of 1965 MHz (1.3
// PF/s), with residual 253-260 us; in runs of about a second, which the power cap holds near
// 1050 MHz, 274 and 299 us. 16384 x 768 -> 1536 with bias 33 us, forward for training with
// GELU 44 us, backward 96 us; 256 x 768 -> 1536 GELU 7.1 us; one row 2.5 us.
//
// The pre-activation z is kept for the backward pass as fp16, also for bf16 rows:
// the activations' derivatives are constant where fp16 ends (|z| > 65504), and
// fp16's 11 bits keep the derivative's error an order below bf16's own rounding.
// dz is rounded once to the rows' type, because both products that read it take
// half-precision operands. That puts dx and dw 2.3e-3 (bf16; fp16 3.0e-4) of their norm from
// float64, where one rounding of the exact gradient is 1.7e-3 (2.1e-4) away; carrying dz's
// remainder as a second operand would double the products. dbias sums the unrounded dz.
#include "cvs_gemm.cuh"

namespace cvs {

namespace {

// ---------------------------------------------------------------------------
// Few tiles: K split over a cluster
// ---------------------------------------------------------------------------
// Where 128 x 64 tiles do not fill the GPU, the S CTAs of a cluster share one tile's K
// dimension. Each sends its fp32 sums of column slice c to CTA c through distributed
// shared memory; after one cluster barrier CTA c adds the S parts in order and finishes
// its 64 / S columns (bias, activation, residual). No workspace, one launch, the same
// result every run. Another CTA's shared memory exists only once that CTA has started:
// every thread arrives on a cluster barrier in the prologue and waits for it after the
// products, ahead of the first store to a peer.
constexpr int kSplitN = 64;
constexpr int kSplitStages = 3;
constexpr int kSplitThreads = 192;

struct SplitLayout {
  static constexpr int kABytes = kGemmM * kGemmK * 2, kBBytes = kSplitN * kGemmK * 2;
  static constexpr int kStage = kABytes + kBBytes;
  static constexpr int kParts = kSplitStages * kStage;              // offset of the received parts
  static constexpr int kBars = kParts + kGemmM * kSplitN * 4;
  static constexpr int kTotal = kBars + 8 * (2 * kSplitStages + 1) + 16;
};

template <int S>
__global__ void __launch_bounds__(kSplitThreads)
    split_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                 const __grid_constant__ SplitArgs a) {
  using L = SplitLayout;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(base + L::kBars);
  uint64_t* empty = full + kSplitStages;
  uint64_t* done = empty + kSplitStages;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(done + 1) + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int tile = static_cast<int>(blockIdx.x) / S;
  const int mt = tile % a.tiles_m, nt = tile / a.tiles_m;
  const int k0 = static_cast<int>(rank) * a.kper, k1 = min(a.kblocks, k0 + a.kper);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSplitStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    mbar_init(done, 1);
    *abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&amap);
    tma_prefetch_desc(&bmap);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, kSplitN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  cluster_arrive();
  const uint32_t tmem = *tmem_holder;
  grid_dependency_wait();
  if (warp == 0) {
    if (elect_one_lane()) {
      int it = 0;
      for (int kb = k0; kb < k1; ++kb, ++it) {
        const int s = it % kSplitStages;
        if (!mbar_wait(empty + s, ((it / kSplitStages) & 1) ^ 1, abort, a.err, 44)) {
          for (int j = max(0, it - kSplitStages); j < it; ++j)
            mbar_wait_drain(full + j % kSplitStages, (j / kSplitStages) & 1);
          break;
        }
        // A's box ends with the last row (rows below it in the tile keep what they had:
        // they only reach accumulator rows that nobody stores).
        mbar_arrive_expect_tx(full + s, static_cast<uint32_t>(a.a_rows) * (kGemmK * 2) + L::kBBytes);
        tma_load_tile(base + s * L::kStage, &amap, full + s, kb * kGemmK, mt * kGemmM);
        tma_load_tile(base + s * L::kStage + L::kABytes, &bmap, full + s, kb * kGemmK, nt * kSplitN);
      }
    }
    __syncwarp();
    cluster_wait();
  } else if (warp == 1) {
    if (elect_one_lane()) {
      const uint32_t idesc = gemm_idesc(kGemmM, kSplitN, a.bf16 != 0, false, false);
      int it = 0;
      for (int kb = k0; kb < k1; ++kb, ++it) {
        const int s = it % kSplitStages;
        if (!mbar_wait(full + s, (it / kSplitStages) & 1, abort, a.err, 45)) break;
        tc_fence_after();
        const uint32_t sa = smem_u32(base + s * L::kStage), sb = sa + L::kABytes;
#pragma unroll
        for (int kk = 0; kk < kGemmK / 16; ++kk)
          tc_mma_f16(tmem, gemm_desc(sa + kk * 32, false), gemm_desc(sb + kk * 32, false), idesc, (it | kk) != 0 ? 1u : 0u);
        tc_commit(empty + s);
      }
      tc_commit(done);
      mbar_wait_drain(done, 0);
    }
    __syncwarp();
    cluster_wait();
  } else {
    const int quad = warp & 3;
    const int row = quad * 32 + lane;
    const bool ok = __all_sync(0xffffffffu, mbar_wait(done, 0, abort, a.err, 46));
    tc_fence_after();
    __syncwarp();
    cluster_wait();  // every CTA of the cluster has started
    const uint32_t parts = smem_u32(base + L::kParts);
    constexpr int kQ = kSplitN / S / 4;  // float4 groups per slice
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t r[32];
      if (ok && k0 < k1) {
        tmem_ld32(tmem + (static_cast<uint32_t>(quad * 32) << 16) + 32 * h, r);
        tmem_wait_ld32(r);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) r[i] = 0u;
      }
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const int group = 8 * h + g;  // columns 4 group .. 4 group + 3
        const uint32_t to = map_to_rank(parts + ((rank * kQ + group % kQ) * kGemmM + row) * 16, group / kQ);
        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(r[4 * g]), "r"(r[4 * g + 1]),
                     "r"(r[4 * g + 2]), "r"(r[4 * g + 3])
                     : "memory");
      }
    }
  }
  tc_fence_before();
  cluster_sync_all();  // every part has arrived; nobody writes to another CTA after this
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kSplitN);
  }
  if (warp < 2) return;
  const int row = (warp & 3) * 32 + lane;
  const long long out_row = static_cast<long long>(mt) * kGemmM + row;
  if (out_row >= a.m) return;
  const bool bf16 = a.bf16 != 0;
  constexpr int kQ = kSplitN / S / 4;
  const float4* parts = reinterpret_cast<const float4*>(base + L::kParts);
#pragma unroll
  for (int e = 0; e < kQ / 2; ++e) {
    const int col = nt * kSplitN + static_cast<int>(rank) * (kSplitN / S) + 8 * e;
    if (col >= a.n) break;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const float4 lo = parts[(s * kQ + 2 * e) * kGemmM + row], hi = parts[(s * kQ + 2 * e + 1) * kGemmM + row];
      v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w;
      v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
    }
    if (a.bias) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < a.n) v[i] += half_at(a.bias, col + i, bf16);
    }
    if (a.z) {
      float kept[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) kept[i] = a.act == kActRelu && v[i] > 0.f ? fmaxf(v[i], 6e-8f) : v[i];
      // z's rows are whole 16-byte units.
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.z) + out_row * a.ld_z + col) =
          make_uint4(pack2(kept[0], kept[1], false), pack2(kept[2], kept[3], false), pack2(kept[4], kept[5], false),
                     pack2(kept[6], kept[7], false));
    }
    act_values(v, a.act);
    if (a.residual) {
      const uint4 q = load_unit8(static_cast<const uint16_t*>(a.residual) + out_row * a.ld_res + col, col, a.n, a.vec_res != 0);
      const uint32_t qs[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2(qs[i], bf16);
        v[2 * i] += f.x;
        v[2 * i + 1] += f.y;
      }
    }
    uint16_t* out = static_cast<uint16_t*>(a.out) + out_row * a.ld_out + col;
    if (a.vec_out && col + 8 <= a.n) {
      *reinterpret_cast<uint4*>(out) = make_uint4(pack2(v[0], v[1], bf16), pack2(v[2], v[3], bf16), pack2(v[4], v[5], bf16),
                                                  pack2(v[6], v[7], bf16));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < a.n) out[i] = half_bits(v[i], bf16);
    }
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
    float va[2] = {v, 0.f};
    act_values(va, a.act);
    v = va[0];
    if (a.residual) v += half_at(a.residual, r * a.ld_res + col, bf16);
    static_cast<uint16_t*>(a.out)[r * a.ld_out + col] = half_bits(v, bf16);
  }
}

// ---------------------------------------------------------------------------
// Backward: dz and the columns' sums
// ---------------------------------------------------------------------------
constexpr int kDzCols = 256;  // columns per block: one warp reads 32 x 16 bytes of a row
constexpr int kDzWarps = 8;
constexpr int kDzRows = 4;    // rows a thread has in flight

// dz = dy act'(z) in the rows' type (dz null: nothing to write, no activation), and
// the block's share of every column's sum, in fp32 from the unrounded dz. Bound by
// HBM: each thread has kDzRows rows' loads in flight before it computes. 16384 x 1536:
// ReLU 24 us, GELU 29 us (150 MB: 23 us at HBM rate).
// VEC: dy's rows are 16-byte aligned. Others come in two-byte loads that are consecutive
// over the warp and are regrouped in shared memory (97742 x 339: 111 us with each lane
// loading its own eight columns).
template <int ACT, bool VEC>
__global__ void __launch_bounds__(32 * kDzWarps) linear_dz_kernel(const LinearDzArgs a) {
  grid_dependency_wait();
  __shared__ float sums[kDzWarps][kDzCols];
  __shared__ __align__(16) uint16_t rows_s[VEC ? 1 : kDzWarps][VEC ? 1 : kDzRows][VEC ? 8 : kDzCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = static_cast<int>(blockIdx.x) * kDzCols, c = c0 + lane * 8;
  const bool bf16 = a.bf16 != 0;
  float s[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) s[t] = 0.f;
  const long long stride = static_cast<long long>(gridDim.y) * kDzWarps;
  for (long long row0 = static_cast<long long>(blockIdx.y) * kDzWarps + warp; row0 < a.m; row0 += stride * kDzRows) {
    uint4 g[kDzRows], z[kDzRows];
#pragma unroll
    for (int i = 0; i < kDzRows; ++i) {
      const long long row = row0 + i * stride;
      g[i] = z[i] = make_uint4(0u, 0u, 0u, 0u);
      if (row >= a.m || c >= a.n) continue;
      if constexpr (VEC) g[i] = load_unit8(static_cast<const uint16_t*>(a.dy) + row * a.ld_dy + c, c, a.n, true);
      // z's rows are padded to whole units; what lies in the padding meets a dy of zero below.
      if constexpr (ACT != kActNone)
        z[i] = load_unit8(static_cast<const uint16_t*>(a.z) + row * a.ld_z + c, c, a.n, true);
    }
    if constexpr (!VEC) {
      uint16_t v[kDzRows][8];
#pragma unroll
      for (int i = 0; i < kDzRows; ++i) {
        const long long row = row0 + i * stride;
        const uint16_t* p = static_cast<const uint16_t*>(a.dy) + row * a.ld_dy + c0 + lane;
#pragma unroll
        for (int t = 0; t < 8; ++t)
          v[i][t] = row < a.m && c0 + 32 * t + lane < a.n ? p[32 * t] : static_cast<uint16_t>(0);
      }
#pragma unroll
      for (int i = 0; i < kDzRows; ++i) {
#pragma unroll
        for (int t = 0; t < 8; ++t) rows_s[warp][i][32 * t + lane] = v[i][t];
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kDzRows; ++i) g[i] = *reinterpret_cast<const uint4*>(&rows_s[warp][i][lane * 8]);
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < kDzRows; ++i) {
      const long long row = row0 + i * stride;
      if (row >= a.m || c >= a.n) continue;
      const uint32_t gs[4] = {g[i].x, g[i].y, g[i].z, g[i].w}, zs[4] = {z[i].x, z[i].y, z[i].z, z[i].w};
      uint32_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float2 f = unpack2(gs[e], bf16);
        if constexpr (ACT != kActNone) {
          const float2 zf = unpack2(zs[e], false);
          slope_pair<ACT>(zf.x, zf.y, f.x, f.y);
        }
        s[2 * e] += f.x;
        s[2 * e + 1] += f.y;
        o[e] = pack2(f.x, f.y, bf16);
      }
      if (a.dz)
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.dz) + row * a.ld_dz + c) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
  grid_launch_dependents();
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
// each), the others two 32 x 32 pieces of dw each, one warp for 8 columns.
__global__ void __launch_bounds__(256) linear_finish_kernel(const LinearFinishArgs a) {
  grid_dependency_wait();
  const bool bf16 = a.bf16 != 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __shared__ float sums[8][33];
  __shared__ __align__(16) uint8_t pieces[2][kBufBytes];
  if (static_cast<int>(blockIdx.x) < a.db_blocks) {
    const int c = static_cast<int>(blockIdx.x) * 32 + lane;
    float s = 0.f;
    if (c < a.n) {
#pragma unroll 8
      for (int b = warp; b < a.db_parts; b += 8) s += a.db_partial[static_cast<size_t>(b) * a.n + c];
    }
    sums[warp][lane] = s;
    __syncthreads();
    if (warp != 0 || c >= a.n) return;
    for (int w = 1; w < 8; ++w) s += sums[w][lane];
    static_cast<uint16_t*>(a.dbias)[c] = half_bits(s, bf16);
    return;
  }
  // Piece: [tile][rank][sub][quad][32 columns], as gemm_kernel wrote it.
  const int subs = gemm_subs(a.bn), steps = a.bn / subs / 32;
  const int per_rank = subs * 4 * steps, per_tile = a.cg * per_rank;
  const int piece = (static_cast<int>(blockIdx.x) - a.db_blocks) * 2 + (warp >> 2);
  const bool live = piece < a.tiles_m * a.tiles_n * per_tile;
  const int tile = piece / per_tile;
  int i = piece - tile * per_tile;
  const int rank = i / per_rank;
  i -= rank * per_rank;
  const int sub = i / (4 * steps);
  i -= sub * 4 * steps;
  const int quad = i / steps, chunk = i % steps;
  const int group = tile / (8 * a.tiles_n);
  const int rows = min(8, a.tiles_m - group * 8);
  const int in_group = tile - group * 8 * a.tiles_n;
  const int row0 = ((group * 8 + in_group % rows) * a.cg + rank) * kGemmM + quad * 32;
  const int col0 = (in_group / rows) * a.bn + sub * (a.bn / subs) + chunk * 32;
  const int unit = warp & 3;
  uint8_t* buf = pieces[warp >> 2];
  if (live && col0 < a.k) {
    const size_t tile_floats = static_cast<size_t>(kGemmM) * a.bn;
    const float* src = a.dw_partial + (static_cast<size_t>(tile) * a.cg + rank) * tile_floats +
                       (static_cast<size_t>(sub * 4 + quad) * steps + chunk) * 1024 + unit * 256 + lane * 4;
    const size_t split_stride = static_cast<size_t>(a.tiles_m) * a.tiles_n * a.cg * tile_floats;
    float v[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) v[t] = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
      const float4 lo = *reinterpret_cast<const float4*>(src + s * split_stride);
      const float4 hi = *reinterpret_cast<const float4*>(src + s * split_stride + 128);
      v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w;
      v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
    }
    *reinterpret_cast<uint4*>(buf + buf_at(lane, unit)) =
        make_uint4(pack2(v[0], v[1], bf16), pack2(v[2], v[3], bf16), pack2(v[4], v[5], bf16), pack2(v[6], v[7], bf16));
  }
  __syncthreads();
  if (!live) return;
  // Each of the piece's four warps writes 8 of its rows, 64 bytes a row.
  const int rr = unit * 8 + (lane >> 2), r = row0 + rr, c = col0 + (lane & 3) * 8;
  if (r >= a.n || c >= a.k) return;
  const uint4 o = *reinterpret_cast<const uint4*>(buf + buf_at(rr, lane & 3));
  uint16_t* p = static_cast<uint16_t*>(a.dw) + r * a.ld_dw + c;
  if (a.vec_dw && c + 8 <= a.k) {
    *reinterpret_cast<uint4*>(p) = o;
  } else {
    const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
    for (int t = 0; t < 8; ++t)
      if (c + t < a.k) p[t] = static_cast<uint16_t>(w[t / 2] >> (16 * (t & 1)));
  }
}

// ---------------------------------------------------------------------------
// Operands the tensor-memory accelerator cannot address
// ---------------------------------------------------------------------------
// Copies rows of any alignment into rows of whole 16-byte units: one warp per row and 256
// columns at a time, eight two-byte loads under way per lane, consecutive over the warp,
// regrouped through shared memory into 16-byte stores.
__global__ void __launch_bounds__(256) pad_rows_kernel(const uint16_t* src, long long rows, int cols, long long ld_src,
                                                       uint16_t* dst, long long ld_dst) {
  __shared__ __align__(16) uint16_t buf[8][256];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunks = (cols + 255) / 256;
  const long long items = rows * chunks;
  for (long long i = static_cast<long long>(blockIdx.x) * 8 + warp; i < items; i += static_cast<long long>(gridDim.x) * 8) {
    const long long row = i / chunks;
    const int c0 = static_cast<int>(i - row * chunks) * 256;
    const uint16_t* p = src + row * ld_src + c0;
    uint16_t v[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) v[t] = c0 + 32 * t + lane < cols ? p[32 * t + lane] : static_cast<uint16_t>(0);
#pragma unroll
    for (int t = 0; t < 8; ++t) buf[warp][32 * t + lane] = v[t];
    __syncwarp();
    const int c = c0 + lane * 8;
    if (c < ld_dst)
      *reinterpret_cast<uint4*>(dst + row * ld_dst + c) = *reinterpret_cast<const uint4*>(&buf[warp][lane * 8]);
    __syncwarp();
  }
}

}  // namespace

cudaError_t gemm_launch(int cg, int bn, const GemmMaps& maps, const GemmArgs& a, int ctas, cudaStream_t stream) {
  switch (a.act) {
    case kActNone: return gemm_launch_none(cg, bn, maps, a, ctas, stream);
    case kActRelu: return gemm_launch_relu(cg, bn, maps, a, ctas, stream);
    case kActGelu: return gemm_launch_gelu(cg, bn, maps, a, ctas, stream);
    case kActSilu: return gemm_launch_silu(cg, bn, maps, a, ctas, stream);
    default: return cudaErrorInvalidValue;
  }
}

namespace {
template <int S>
cudaError_t split_launch_one(const CUtensorMap& amap, const CUtensorMap& bmap, const SplitArgs& a, int ctas, cudaStream_t stream) {
  constexpr int smem = SplitLayout::kTotal + 1024;
  auto kern = split_kernel<S>;
  static std::atomic<unsigned long long> allowed{0};
  const cudaError_t e = allow_smem(kern, smem, allowed);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = S;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, amap, bmap, a);
}
}  // namespace

cudaError_t split_launch(int splits, const CUtensorMap& amap, const CUtensorMap& bmap, const SplitArgs& a, int tiles,
                         cudaStream_t stream) {
  switch (splits) {
    case 2: return split_launch_one<2>(amap, bmap, a, 2 * tiles, stream);
    case 4: return split_launch_one<4>(amap, bmap, a, 4 * tiles, stream);
    case 8: return split_launch_one<8>(amap, bmap, a, 8 * tiles, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t linear_small_launch(const LinearSmallArgs& a, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((a.n + 7) / 8));
  if (a.m <= 1) return launch_programmatic(linear_small_kernel<1>, grid, dim3(256), 0, stream, a);
  if (a.m <= 2) return launch_programmatic(linear_small_kernel<2>, grid, dim3(256), 0, stream, a);
  if (a.m <= 4) return launch_programmatic(linear_small_kernel<4>, grid, dim3(256), 0, stream, a);
  if (a.m <= kLinearSmallRows) return launch_programmatic(linear_small_kernel<8>, grid, dim3(256), 0, stream, a);
  return cudaErrorInvalidValue;
}

cudaError_t pad_rows_launch(const void* src, long long rows, int cols, long long ld_src, void* dst, long long ld_dst,
                            int num_sms, cudaStream_t stream) {
  const long long items = rows * ((cols + 255) / 256);
  const dim3 grid(static_cast<unsigned>(std::max<long long>(1, std::min<long long>((items + 7) / 8, 8LL * num_sms))));
  return launch_programmatic(pad_rows_kernel, grid, dim3(256), 0, stream, static_cast<const uint16_t*>(src), rows, cols,
                             ld_src, static_cast<uint16_t*>(dst), ld_dst);
}

int linear_dz_parts(long long m, int n, int num_sms) {
  const int cols = (n + kDzCols - 1) / kDzCols;
  const long long want = std::max(1, 2 * num_sms / cols);  // one round of blocks, few sums to add
  return static_cast<int>(std::max<long long>(1, std::min<long long>(want, (m + kDzWarps - 1) / kDzWarps)));
}

namespace {
template <int ACT>
cudaError_t dz_launch_act(const LinearDzArgs& a, dim3 grid, cudaStream_t stream) {
  const dim3 block(32 * kDzWarps);
  return a.vec_dy ? launch_programmatic(linear_dz_kernel<ACT, true>, grid, block, 0, stream, a)
                  : launch_programmatic(linear_dz_kernel<ACT, false>, grid, block, 0, stream, a);
}
}  // namespace

cudaError_t linear_dz_launch(const LinearDzArgs& a, int parts, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((a.n + kDzCols - 1) / kDzCols), static_cast<unsigned>(parts));
  switch (a.z ? a.act : kActNone) {
    case kActNone: return dz_launch_act<kActNone>(a, grid, stream);
    case kActRelu: return dz_launch_act<kActRelu>(a, grid, stream);
    case kActGelu: return dz_launch_act<kActGelu>(a, grid, stream);
    case kActSilu: return dz_launch_act<kActSilu>(a, grid, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t linear_finish_launch(const LinearFinishArgs& a, cudaStream_t stream) {
  const int pieces = a.dw_partial ? a.tiles_m * a.tiles_n * a.cg * 4 * (a.bn / 32) : 0;
  const int grid = a.db_blocks + (pieces + 1) / 2;
  if (grid == 0) return cudaSuccess;
  return launch_programmatic(linear_finish_kernel, dim3(static_cast<unsigned>(grid)), dim3(256), 0, stream, a);
}

}  // namespace cvs
