// Layer norm over the rows of a matrix, forward and backward.
//
//   forward   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r,
//             y = h w + b; mu and r are kept for the backward pass (8 bytes a row).
//   backward  g = dy w;  dx = r (g - mean(g) - h mean(g h));
//             dw = sum over rows of dy h;  db = sum over rows of dy.
//
// Both are bound by HBM traffic (forward: read x, write y; backward: read x and
// dy, write dx), so every row is read once and kept in registers, in its stored
// type, between the statistics and the result. The variance is the mean of
// squared differences from the mean, a second pass over the registers, so that
// rows far from zero lose nothing. All sums are fp32.
//
// A row belongs to one warp (width up to 1024: no barrier) or to one block of 8 warps
// (up to 8192). Aligned rows of one warp come as bulk copies into a ring per warp in
// shared memory (forward: in large matrices, norm_staged), so that the bytes in flight cost no
// registers and each SM's warps never wait for one another's rows. In the backward pass
// every thread keeps the sums of dw and db for the columns it owns while its warp walks
// the rows, so the weights' gradients cost no traffic per row; the blocks' sums go to the
// workspace and a second small kernel adds them in a fixed order, which makes the result
// the same on every run. Measured: 262144 x 768 fp16 forward 140-150 us (5.4-5.8 TB/s),
// backward 192 us (6.3 TB/s); with rows loaded into registers 157 and 372 us. 16384 x 768
// bf16: 12 and 20 us, of which about half is the kernels' start and end.
#include "cvs_device.cuh"
#include "cvs_elem.cuh"
#include "cvs_kernels.h"

#include <algorithm>
#include <climits>

namespace cvs {

namespace {

constexpr int kNormThreads = 256;
constexpr int kNormWarps = kNormThreads / 32;
constexpr int kNormSlots = 4;    // most row pairs in a warp's ring of the backward pass
constexpr int kForwardSlots = 8; // most rows in a warp's ring of the forward pass
constexpr int kForwardRows = 2;  // rows a warp has at work in the forward pass
constexpr int kForwardShared = 72 * 1024;  // most shared memory of a staged forward block: weight and bias, the ring

// Sum over the threads of a row: one warp, or all 8 warps of the block (scratch
// holds two buffers used in turn, so one barrier per sum is enough).
template <int WARPS>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2* scratch) {
  a = warp_sum(a);
  b = warp_sum(b);
  if constexpr (WARPS > 1) {
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float2 s = scratch[w];
      a += s.x;
      b += s.y;
    }
  }
  return make_float2(a, b);
}

// Weights of a row's threads as fp32 pairs: group j, pair i of thread tid at [(j * 4 + i)
// * THREADS + tid], one conflict-free 8-byte read. Staged by the whole block.
template <class T, bool VEC, int THREADS, int CPL>
__device__ __forceinline__ void stage_weights(const void* w, bool w32, int d, float2* out) {
#pragma unroll
  for (int k = threadIdx.x; k < CPL * 4 * THREADS; k += kNormThreads) {
    const int tid = k % THREADS, i = k / THREADS % 4, j = k / THREADS / 4;
    float v[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int c = Cols<VEC>::at(tid, THREADS, j, 2 * i + t);
      v[t] = 0.f;
      if (c < d) v[t] = w32 ? static_cast<const float*>(w)[c] : to_f32(static_cast<const T*>(w)[c]);
    }
    out[k] = make_float2(v[0], v[1]);
  }
}
// Group j of the thread's weights straight from global memory (L1).
template <class T, bool VEC>
__device__ __forceinline__ void weight_group(const void* w, bool w32, int d, int tid, int threads, int j, float missing,
                                             Pair (&out)[4]) {
  if (w == nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = both(missing);
  } else if (w32) {
    const Raw8<float> r = Cols<VEC>::load(static_cast<const float*>(w), d, tid, threads, j);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = pair_at(r, i);
  } else {
    const Raw8<T> r = Cols<VEC>::load(static_cast<const T*>(w), d, tid, threads, j);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = pair_at(r, i);
  }
}
template <int THREADS>
__device__ __forceinline__ Pair weight_at(const float2* w, int tid, int j, int i) {
  const float2 f = w[(j * 4 + i) * THREADS + tid];
  return pair_of(f.x, f.y);
}

// Pair i of group j with columns outside the row replaced by zeros.
template <bool VEC>
__device__ __forceinline__ Pair inside(Pair p, int d, int tid, int threads, int j, int i) {
  float lo, hi;
  split(p, lo, hi);
  if (Cols<VEC>::at(tid, threads, j, 2 * i) >= d) lo = 0.f;
  if (Cols<VEC>::at(tid, threads, j, 2 * i + 1) >= d) hi = 0.f;
  return pair_of(lo, hi);
}

template <bool VEC, int WARPS>
__host__ __device__ constexpr bool norm_ring() { return VEC && WARPS == 1; }

// STAGED: weights in shared memory, for blocks that walk many rows; otherwise straight
// from global memory, where the staging and its barrier would be a large part of the
// work (256 rows of 768: 5.2 us staged, 4.3 us straight; 262144 rows: 140 and 185 us).
template <class T, bool VEC, int WARPS, int CPL, bool STAGED>
__global__ void __launch_bounds__(kNormThreads) norm_forward_kernel(const __grid_constant__ NormArgs a) {
  constexpr int kRowThreads = 32 * WARPS;
  constexpr int kRowsPerBlock = kNormThreads / kRowThreads;
  constexpr bool kRing = STAGED && norm_ring<VEC, WARPS>();
  constexpr int kRows = WARPS == 1 && !kRing ? kForwardRows : 1;  // rows a warp (block) has at work
  // The first group of columns that a row may end in (launch_width: every width of one warp
  // has its own CPL; a block's has 1, 2 or 4, and the row fills more than half of them).
  constexpr int kFirstPartial = WARPS == 1 ? CPL - 1 : CPL / 2;
  __shared__ float2 scratch[2][WARPS > 1 ? WARPS : 1];
  __shared__ __align__(8) uint64_t bars[kRing ? kNormWarps : 1][kRing ? kForwardSlots : 1];
  __shared__ int abort_s;
  extern __shared__ __align__(128) uint8_t shared_f[];  // STAGED: weight and bias, [2][CPL * 4][kRowThreads]; the ring
  const float2* weight_s = reinterpret_cast<const float2*>(shared_f);
  const float2* bias_s = weight_s + CPL * 4 * kRowThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tid = threadIdx.x % kRowThreads;
  const int d = a.d;
  const float inv_d = 1.f / static_cast<float>(d);
  if constexpr (kRing) {
    if (lane == 0) {
      for (int k = 0; k < a.slots; ++k) mbar_init(&bars[warp][k], 1);
      if (warp == 0) abort_s = 0;
      fence_barrier_init();
    }
  }
  grid_dependency_wait();
  if constexpr (STAGED) {
    float2* out = reinterpret_cast<float2*>(shared_f);
    if (a.weight) stage_weights<T, VEC, kRowThreads, CPL>(a.weight, a.w32, d, out);
    if (a.bias) stage_weights<T, VEC, kRowThreads, CPL>(a.bias, a.w32, d, out + CPL * 4 * kRowThreads);
    __syncthreads();
  }
  const long long slots = static_cast<long long>(gridDim.x) * kRowsPerBlock;
  long long row0 = static_cast<long long>(blockIdx.x) * kRowsPerBlock + threadIdx.x / kRowThreads;
  const uint32_t row_bytes = static_cast<uint32_t>(d) * sizeof(T);
  uint8_t* ring = shared_f + 2 * CPL * 4 * kRowThreads * sizeof(float2) + static_cast<size_t>(warp) * a.slots * row_bytes;
  const auto request = [&](long long r, int k) {  // one lane
    if (r >= a.rows || a.stall) return;
    mbar_arrive_expect_tx(&bars[warp][k], row_bytes);
    bulk_load(ring + k * row_bytes, static_cast<const T*>(a.x) + r * a.x_stride, row_bytes, &bars[warp][k]);
  };
  if constexpr (kRing) {
    if (lane == 0) {
      for (int k = 0; k < a.slots; ++k) request(row0 + k * slots, k);
    }
  }
  int slot = 0;
  uint32_t parity = 0;
  bool ok = true;
  const long long limit = a.wait_cycles > 0 ? a.wait_cycles : kWaitCycles;
  for (; row0 < a.rows; row0 += slots * kRows) {
    Raw8<T> raw[kRows][CPL];
    float mean[kRows], rstd[kRows];
    if constexpr (kRing) {
      ok = __all_sync(0xffffffffu, mbar_wait(&bars[warp][slot], parity, &abort_s, a.err, 42, limit));
      if (!ok) break;
    }
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      const long long row = row0 + q * slots;
      const T* x = kRing ? reinterpret_cast<const T*>(ring + slot * row_bytes)
                         : static_cast<const T*>(a.x) + (row < a.rows ? row : row0) * a.x_stride;
#pragma unroll
      for (int j = 0; j < CPL; ++j) raw[q][j] = Cols<VEC>::load(x, d, tid, kRowThreads, j);
    }
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      Pair sum = both(0.f);
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = pair_add(sum, pair_at(raw[q][j], i));
      }
      mean[q] = row_sum2<WARPS>(pair_total(sum), 0.f, scratch[0]).x * inv_d;
    }
    if constexpr (kRing) {
      // Every lane has its part of the row in registers (the sum needed all of them).
      if (lane == 0) request(row0 + a.slots * slots, slot);
      if (++slot == a.slots) {
        slot = 0;
        parity ^= 1;
      }
    }
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      Pair sq = both(0.f);
      const Pair shift = both(-mean[q]);
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          Pair c = pair_add(pair_at(raw[q][j], i), shift);
          if (!VEC || j >= kFirstPartial) c = inside<VEC>(c, d, tid, kRowThreads, j, i);
          sq = pair_fma(c, c, sq);
        }
      }
      rstd[q] = 1.f / sqrtf(row_sum2<WARPS>(pair_total(sq), 0.f, scratch[1]).x * inv_d + a.eps);
    }
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      const long long row = row0 + q * slots;
      if (tid == 0 && row < a.rows) {
        if (a.mean) a.mean[row] = mean[q];
        if (a.rstd) a.rstd[row] = rstd[q];
      }
    }
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      Raw8<T> out[kRows];
      Pair w[4], b[4];
      if constexpr (STAGED) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = a.weight ? weight_at<kRowThreads>(weight_s, tid, j, i) : both(1.f);
          b[i] = a.bias ? weight_at<kRowThreads>(bias_s, tid, j, i) : both(0.f);
        }
      } else {
        weight_group<T, VEC>(a.weight, a.w32, d, tid, kRowThreads, j, 1.f, w);
        weight_group<T, VEC>(a.bias, a.w32, d, tid, kRowThreads, j, 0.f, b);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int q = 0; q < kRows; ++q) {
          const Pair h = pair_mul(pair_add(pair_at(raw[q][j], i), both(-mean[q])), both(rstd[q]));
          set_pair(out[q], i, pair_fma(h, w[i], b[i]));
        }
      }
#pragma unroll
      for (int q = 0; q < kRows; ++q) {
        const long long row = row0 + q * slots;
        if (row < a.rows) Cols<VEC>::store(static_cast<T*>(a.y) + row * a.y_stride, d, tid, kRowThreads, j, out[q]);
      }
    }
  }
  if constexpr (kRing) {
    if (!ok && !a.stall && lane == 0) {  // after a wait that ran out: copies under way land
      for (int k = 0; k < a.slots; ++k, row0 += slots) {
        if (row0 < a.rows) mbar_wait_drain(&bars[warp][(slot + k) % a.slots], slot + k < a.slots ? parity : parity ^ 1);
      }
    }
  }
}

// Backward. Aligned rows of one warp (kRing) come as bulk copies into a ring of `slots`
// row pairs (x, dy) per warp in shared memory, so that the bytes in flight cost no
// registers, which the sums of dw and db need (16 a group of columns); other rows are
// loaded into registers, the next row's loads under way where that fits. Two blocks an
// SM, except for wide fp32 rows.
template <class T, int CPL>
constexpr int backward_blocks() { return sizeof(T) == 4 && CPL > 3 ? 1 : 2; }

template <class T, bool VEC, int WARPS, int CPL>
__global__ void __launch_bounds__(kNormThreads, (backward_blocks<T, CPL>()))
    norm_backward_kernel(const __grid_constant__ NormArgs a) {
  constexpr int kRowThreads = 32 * WARPS;
  constexpr int kRowsPerBlock = kNormThreads / kRowThreads;
  constexpr bool kRing = norm_ring<VEC, WARPS>();
  __shared__ float2 scratch[2][WARPS > 1 ? WARPS : 1];
  __shared__ __align__(8) uint64_t bars[kRing ? kNormWarps : 1][kRing ? kNormSlots : 1];
  __shared__ int abort_s;
  // The weights, then the ring; after the last row (single-warp rows) the warps' sums [8][2][d].
  extern __shared__ __align__(128) uint8_t shared_b[];
  float2* shared = reinterpret_cast<float2*>(shared_b);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tid = threadIdx.x % kRowThreads;
  const int d = a.d;
  const float inv_d = 1.f / static_cast<float>(d);
  Pair dw[CPL][4], db[CPL][4];
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[j][i] = db[j][i] = both(0.f);
  }
  if constexpr (kRing) {
    if (lane == 0) {
      for (int k = 0; k < a.slots; ++k) mbar_init(&bars[warp][k], 1);
      if (warp == 0) abort_s = 0;
      fence_barrier_init();
    }
  }
  grid_dependency_wait();
  if (a.weight) stage_weights<T, VEC, kRowThreads, CPL>(a.weight, a.w32, d, shared);
  __syncthreads();
  const long long slots = static_cast<long long>(gridDim.x) * kRowsPerBlock;
  long long row = static_cast<long long>(blockIdx.x) * kRowsPerBlock + threadIdx.x / kRowThreads;
  const uint32_t row_bytes = static_cast<uint32_t>(d) * sizeof(T);
  uint8_t* ring = shared_b + CPL * 4 * kRowThreads * sizeof(float2) + static_cast<size_t>(warp) * a.slots * 2 * row_bytes;
  const auto request = [&](long long r, int k) {  // one lane
    if (r >= a.rows || a.stall) return;
    mbar_arrive_expect_tx(&bars[warp][k], 2 * row_bytes);
    bulk_load(ring + k * 2 * row_bytes, static_cast<const T*>(a.x) + r * a.x_stride, row_bytes, &bars[warp][k]);
    bulk_load(ring + k * 2 * row_bytes + row_bytes, static_cast<const T*>(a.dy) + r * a.dy_stride, row_bytes, &bars[warp][k]);
  };
  Raw8<T> xr[CPL], gr[CPL];
  float mean_n = 0.f, rstd_n = 0.f;
  if (row < a.rows) {
    mean_n = a.mean[row];
    rstd_n = a.rstd[row];
  }
  if constexpr (kRing) {
    if (lane == 0) {
      for (int k = 0; k < a.slots; ++k) request(row + k * slots, k);
    }
  }
  int turn = 0, slot = 0;
  uint32_t parity = 0;
  bool ok = true;
  const long long limit = a.wait_cycles > 0 ? a.wait_cycles : kWaitCycles;
  for (; row < a.rows; row += slots, turn ^= 1) {
    const float mean = mean_n, rstd = rstd_n;
    if (row + slots < a.rows) {
      mean_n = a.mean[row + slots];
      rstd_n = a.rstd[row + slots];
    }
    const T *xs, *gs;  // this row
    if constexpr (kRing) {
      ok = __all_sync(0xffffffffu, mbar_wait(&bars[warp][slot], parity, &abort_s, a.err, 41, limit));
      if (!ok) break;
      xs = reinterpret_cast<const T*>(ring + slot * 2 * row_bytes);
      gs = reinterpret_cast<const T*>(ring + slot * 2 * row_bytes + row_bytes);
    } else {
      xs = static_cast<const T*>(a.x) + row * a.x_stride;
      gs = static_cast<const T*>(a.dy) + row * a.dy_stride;
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        xr[j] = Cols<VEC>::load(xs, d, tid, kRowThreads, j);
        gr[j] = Cols<VEC>::load(gs, d, tid, kRowThreads, j);
      }
    }
    // h = (x - mu) r, the difference first: x r - mu r would round mu r, which for rows far
    // from zero is larger than h. Columns outside the row: dy reads as zero there, so g is
    // zero and they add nothing to any sum.
    const Pair r2 = both(rstd), shift = both(-mean);
    Pair s1 = both(0.f), s2 = both(0.f);
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      if constexpr (kRing) {
        xr[j] = Cols<VEC>::load(xs, d, tid, kRowThreads, j);
        gr[j] = Cols<VEC>::load(gs, d, tid, kRowThreads, j);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Pair g = pair_at(gr[j], i);
        const Pair h = pair_mul(pair_add(pair_at(xr[j], i), shift), r2);
        const Pair gw = a.weight ? pair_mul(g, weight_at<kRowThreads>(shared, tid, j, i)) : g;
        s1 = pair_add(s1, gw);
        s2 = pair_fma(gw, h, s2);
        dw[j][i] = pair_fma(g, h, dw[j][i]);
        db[j][i] = pair_add(db[j][i], g);
      }
    }
    const float2 s = row_sum2<WARPS>(pair_total(s1), pair_total(s2), scratch[turn]);
    if (a.dx) {
      const Pair c1 = both(-s.x * inv_d), c2 = both(-s.y * inv_d);
      T* dx = static_cast<T*>(a.dx) + row * a.dx_stride;
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        if constexpr (sizeof(T) == 2) {
          forget(xr[j]);
          forget(gr[j]);
        }
        Raw8<T> out;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const Pair g = pair_at(gr[j], i);
          const Pair h = pair_mul(pair_add(pair_at(xr[j], i), shift), r2);
          const Pair gw = a.weight ? pair_mul(g, weight_at<kRowThreads>(shared, tid, j, i)) : g;
          set_pair(out, i, pair_mul(r2, pair_add(gw, pair_fma(h, c2, c1))));
        }
        Cols<VEC>::store(dx, d, tid, kRowThreads, j, out);
      }
    }
    if constexpr (kRing) {
      __syncwarp();  // the row has been read
      if (lane == 0) request(row + a.slots * slots, slot);
      if (++slot == a.slots) {
        slot = 0;
        parity ^= 1;
      }
    }
  }
  if constexpr (kRing) {
    if (!ok && !a.stall && lane == 0) {  // after a wait that ran out: copies under way land
      for (int k = 0; k < a.slots; ++k, row += slots) {
        if (row < a.rows) mbar_wait_drain(&bars[warp][(slot + k) % a.slots], slot + k < a.slots ? parity : parity ^ 1);
      }
    }
    __syncwarp();
  }
  grid_launch_dependents();
  if (a.partial == nullptr) return;
  float* block_out = a.partial + static_cast<size_t>(blockIdx.x) * 2 * d;
  float* sums = WARPS > 1 ? block_out : reinterpret_cast<float*>(shared) + static_cast<size_t>(warp) * 2 * d;
  if constexpr (WARPS == 1) __syncthreads();  // weights and rows are no longer read
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float w[2], b[2];
      split(dw[j][i], w[0], w[1]);
      split(db[j][i], b[0], b[1]);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int c = Cols<VEC>::at(tid, kRowThreads, j, 2 * i + t);
        if (c < d) {
          sums[c] = w[t];
          sums[d + c] = b[t];
        }
      }
    }
  }
  if constexpr (WARPS == 1) {
    __syncthreads();
    const float* all = reinterpret_cast<const float*>(shared);
    for (int i = threadIdx.x; i < 2 * d; i += kNormThreads) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kNormWarps; ++w) v += all[static_cast<size_t>(w) * 2 * d + i];
      block_out[i] = v;
    }
  }
}

// out[c] = sum over blocks of partial[block][c], in a fixed order: 32 columns a
// block, 32 threads a column.
__global__ void __launch_bounds__(1024) norm_finish_kernel(const float* partial, int blocks, int d, void* dweight,
                                                           void* dbias, int out_dtype) {
  __shared__ float sums[32][33];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;  // column of [2][d]
  float s = 0.f;
  if (c < 2 * d) {
#pragma unroll 4
    for (int b = part; b < blocks; b += 32) s += partial[static_cast<size_t>(b) * 2 * d + c];
  }
  sums[part][lane] = s;
  __syncthreads();
  s = warp_sum(sums[lane][part]);  // column `part` of this block's 32
  const int col = blockIdx.x * 32 + part;
  if (lane != 0 || col >= 2 * d) return;
  void* out = col < d ? dweight : dbias;
  const int i = col < d ? col : col - d;
  if (out == nullptr) return;
  if (out_dtype == kSrcF32) static_cast<float*>(out)[i] = s;
  else if (out_dtype == kSrcF16) static_cast<__half*>(out)[i] = __float2half_rn(s);
  else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(s);
}

int row_warps(int d) { return d <= 1024 ? 1 : kNormWarps; }

unsigned norm_grid(long long rows, int rows_per_block, int blocks) {
  return static_cast<unsigned>(std::max<long long>(1, std::min<long long>((rows + rows_per_block - 1) / rows_per_block, blocks)));
}


// Whether forward blocks walk several rounds of rows with the weights (and, aligned rows of
// one warp, the rows) staged in shared memory: where the matrix is large against one round
// of blocks. Straight / staged, us:
//   fp16, one warp a row: 64 columns, 65536 rows 20.1 / 21.0; 256 columns, 16384 rows 6.9 /
//     7.2, 131072 39.2 / 38.6; 400 columns, 16384 rows 10.8 / 9.2, 131072 61 / 51; 768
//     columns, 4096 rows 5.3 / 5.8, 16384 16.3 / 12.8, 131072 99 / 78; unaligned: 391 columns,
//     16384 rows 13.7 / 12.9, 131072 87 / 69; 767 columns, 131072 rows 120 / 127.
//   fp16, a block a row: 2048 columns, 2048 rows 8.0 / 8.6, 4096 14.2 / 12.9, 16384 50 / 40;
//     8192 columns, 4096 rows 34.5 / 35.4, 16384 115 / 113.
//   fp32, one warp a row (whose ring is half as deep): 512 columns, 16384 rows 14.3 / 15.0,
//     131072 83 / 102; 768 columns, 16384 rows 20.6 / 20.3, 131072 127 / 149; 1000 columns,
//     4096 rows 9.4 / 9.4, 16384 30 / 26, 32768 53 / 52, 131072 186 / 199; unaligned: 511
//     columns, 131072 rows 86 / 93; 1001 columns, 131072 rows 182 / 175.
//   fp32, a block a row: 1031 columns, 8192 rows 26 / 22, 65536 194 / 153; 2048 columns, 4096
//     rows 16.4 / 18.1, 8192 30.1 / 30.5, 32768 110 / 101; 8192 columns, 16384 rows 179 / 185.
template <class T, bool VEC, int WARPS, int CPL>
constexpr bool may_stage() { return sizeof(T) == 2 || WARPS > 1 || CPL > 3; }
template <class T, bool VEC, int WARPS, int CPL>
bool norm_staged(long long rows, int d) {
  constexpr bool kHalf = sizeof(T) == 2;
  if (WARPS > 1) return rows >= (kHalf ? 4096 : 8192);
  const long long cells = rows * d;
  return may_stage<T, VEC, WARPS, CPL>() && cells > (1 << 22) && (kHalf || !VEC || cells <= (1 << 25));
}

// Blocks of `kern` an SM holds at once.
template <class K>
int blocks_per_sm(K kern, size_t smem) {
  int n = 0;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, kNormThreads, smem) == cudaSuccess && n > 0 ? n : 1;
}

template <class T, bool VEC, int WARPS, int CPL>
cudaError_t launch_one(NormArgs a, bool backward, int num_sms, cudaStream_t stream) {
  constexpr int kPerBlock = kNormWarps / WARPS;
  const size_t weights = static_cast<size_t>(CPL) * 4 * 32 * WARPS * sizeof(float2);
  const bool stage = norm_staged<T, VEC, WARPS, CPL>(a.rows, a.d);
  if (a.stall && !(norm_ring<VEC, WARPS>() && (backward || stage))) return cudaErrorNotSupported;
  if (!backward) {
    if constexpr (may_stage<T, VEC, WARPS, CPL>()) {
      if (stage) {
        // One round of blocks: each SM's share of the rows is the same.
        auto kern = norm_forward_kernel<T, VEC, WARPS, CPL, true>;
        size_t smem = 2 * weights;
        int per_warp = 1;  // rows a warp has at work
        if (norm_ring<VEC, WARPS>()) {
          const size_t per = static_cast<size_t>(kNormWarps) * a.d * sizeof(T);
          a.slots = static_cast<int>(std::max<size_t>(1, std::min<size_t>(kForwardSlots, (kForwardShared - smem) / per)));
          smem += a.slots * per;
        } else if (WARPS == 1) {
          per_warp = kForwardRows;
        }
        static std::atomic<unsigned long long> allowed{0};
        const cudaError_t e = allow_smem(kern, kForwardShared, allowed);
        if (e != cudaSuccess) return e;
        const unsigned grid = norm_grid(a.rows, kPerBlock * per_warp, blocks_per_sm(kern, smem) * num_sms);
        return launch_programmatic(kern, dim3(grid), dim3(kNormThreads), smem, stream, a);
      }
    }
    const unsigned grid = norm_grid(a.rows, WARPS == 1 ? kPerBlock * kForwardRows : 1, INT_MAX);
    return launch_programmatic(norm_forward_kernel<T, VEC, WARPS, CPL, false>, dim3(grid), dim3(kNormThreads), 0, stream, a);
  }
  constexpr int kShared = backward_blocks<T, CPL>() == 1 ? 216 * 1024 : 108 * 1024;  // most of any call
  const size_t sums = WARPS == 1 && a.partial ? static_cast<size_t>(kNormWarps) * 2 * a.d * 4 : 0;
  size_t ring = 0;
  a.slots = 1;
  if (norm_ring<VEC, WARPS>()) {
    const size_t per = static_cast<size_t>(kNormWarps) * 2 * a.d * sizeof(T);
    const size_t room = kShared - weights;
    a.slots = static_cast<int>(std::max<size_t>(1, std::min<size_t>(kNormSlots, room / per)));
    ring = a.slots * per;
  }
  const size_t smem = std::max(weights + ring, sums);
  auto kern = norm_backward_kernel<T, VEC, WARPS, CPL>;
  static std::atomic<unsigned long long> allowed{0};
  const cudaError_t e = allow_smem(kern, kShared, allowed);
  if (e != cudaSuccess) return e;
  const unsigned grid = static_cast<unsigned>(norm_backward_blocks(a.rows, a.d, num_sms));
  return launch_programmatic(kern, dim3(grid), dim3(kNormThreads), smem, stream, a);
}

template <class T, bool VEC>
cudaError_t launch_width(const NormArgs& a, bool backward, int num_sms, cudaStream_t stream) {
  const int groups = (a.d + 255) / 256;  // groups of eight columns per lane of one warp
  if (groups <= 1) return launch_one<T, VEC, 1, 1>(a, backward, num_sms, stream);
  if (groups <= 2) return launch_one<T, VEC, 1, 2>(a, backward, num_sms, stream);
  if (groups <= 3) return launch_one<T, VEC, 1, 3>(a, backward, num_sms, stream);
  if (groups <= 4) return launch_one<T, VEC, 1, 4>(a, backward, num_sms, stream);
  if (groups <= 8) return launch_one<T, VEC, 8, 1>(a, backward, num_sms, stream);
  if (groups <= 16) return launch_one<T, VEC, 8, 2>(a, backward, num_sms, stream);
  return launch_one<T, VEC, 8, 4>(a, backward, num_sms, stream);
}

template <class T>
cudaError_t launch_type(const NormArgs& a, bool backward, int num_sms, cudaStream_t stream) {
  const auto ok = [&](const void* p, long long stride, size_t es) {
    return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (stride * es) % 16 == 0);
  };
  const size_t es = sizeof(T), ws = a.w32 ? 4 : es;
  const bool vec = a.d % 8 == 0 && ok(a.x, a.x_stride, es) && ok(a.y, a.y_stride, es) && ok(a.dy, a.dy_stride, es) &&
                   ok(a.dx, a.dx_stride, es) && ok(a.weight, 0, ws) && ok(a.bias, 0, ws);
  return vec ? launch_width<T, true>(a, backward, num_sms, stream) : launch_width<T, false>(a, backward, num_sms, stream);
}

}  // namespace

int norm_backward_blocks(long long rows, int d, int num_sms) {
  return static_cast<int>(norm_grid(rows, kNormWarps / row_warps(d), 2 * num_sms));
}

cudaError_t norm_launch(const NormArgs& a, int dtype, bool backward, int num_sms, cudaStream_t stream) {
  if (a.d < 1 || a.d > kNormMaxWidth || a.rows < 1) return cudaErrorInvalidValue;
  cudaError_t e;
  switch (dtype) {
    case kSrcF32: e = launch_type<float>(a, backward, num_sms, stream); break;
    case kSrcF16: e = launch_type<__half>(a, backward, num_sms, stream); break;
    case kSrcBF16: e = launch_type<__nv_bfloat16>(a, backward, num_sms, stream); break;
    default: return cudaErrorInvalidValue;
  }
  if (e != cudaSuccess || !backward || a.partial == nullptr) return e;
  return launch_programmatic(norm_finish_kernel, dim3(static_cast<unsigned>((2 * a.d + 31) / 32)), dim3(1024), 0, stream,
                             static_cast<const float*>(a.partial), norm_backward_blocks(a.rows, a.d, num_sms), a.d, a.dweight, a.dbias,
                             a.w32 ? static_cast<int>(kSrcF32) : dtype);
}

}  // namespace cvs
