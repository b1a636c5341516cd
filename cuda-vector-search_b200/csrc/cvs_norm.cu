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
// (up to 8192). Weights are held as fp32 pairs in shared memory, in the order the lanes
// read them. Forward, a warp takes two rows at a time, which doubles the loads in flight
// and halves the reads of the weights. In the backward pass a block walks rows with a
// stride of the grid, the next row's loads under way, and every thread keeps the sums of
// dw and db for the columns it owns, so the weights' gradients cost no traffic per row;
// the blocks' sums go to the workspace and a second small kernel adds them in a fixed
// order, which makes the result the same on every run.
#include "cvs_device.cuh"
#include "cvs_elem.cuh"
#include "cvs_kernels.h"

#include <algorithm>

namespace cvs {

namespace {

constexpr int kNormThreads = 256;
constexpr int kNormWarps = kNormThreads / 32;
constexpr int kForwardRows = 2;  // rows a warp has at work in the forward pass

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

// Weights of the thread's columns as fp32 pairs: group j, pair i at [(j * 4 + i) * threads
// + tid], one conflict-free 8-byte read.
template <class T, bool VEC, int THREADS, int CPL>
__device__ __forceinline__ void stage_weights(const void* w, bool w32, int d, int tid, float missing, float2* out) {
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int c = Cols<VEC>::at(tid, THREADS, j, 2 * i + t);
        v[t] = missing;
        if (w != nullptr && c < d) v[t] = w32 ? static_cast<const float*>(w)[c] : to_f32(static_cast<const T*>(w)[c]);
      }
      out[(j * 4 + i) * THREADS + tid] = make_float2(v[0], v[1]);
    }
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

template <class T, bool VEC, int WARPS, int CPL>
__global__ void __launch_bounds__(kNormThreads) norm_forward_kernel(const NormArgs a) {
  constexpr int kRowThreads = 32 * WARPS;
  constexpr int kRowsPerBlock = kNormThreads / kRowThreads;
  constexpr int kRows = WARPS == 1 ? kForwardRows : 1;  // rows a warp (block) has at work
  __shared__ float2 scratch[2][WARPS > 1 ? WARPS : 1];
  extern __shared__ float2 weights[];  // [2][CPL * 4][kRowThreads]
  const int tid = threadIdx.x % kRowThreads;
  const int d = a.d;
  const float inv_d = 1.f / static_cast<float>(d);
  float2* w_s = weights;
  float2* b_s = weights + CPL * 4 * kRowThreads;
  grid_dependency_wait();
  if (threadIdx.x < kRowThreads) {
    if (a.weight) stage_weights<T, VEC, kRowThreads, CPL>(a.weight, a.w32, d, tid, 1.f, w_s);
    if (a.bias) stage_weights<T, VEC, kRowThreads, CPL>(a.bias, a.w32, d, tid, 0.f, b_s);
  }
  __syncthreads();
  const long long slots = static_cast<long long>(gridDim.x) * kRowsPerBlock;
  for (long long row0 = static_cast<long long>(blockIdx.x) * kRowsPerBlock + threadIdx.x / kRowThreads; row0 < a.rows;
       row0 += slots * kRows) {
    Raw8<T> raw[kRows][CPL];
    float mean[kRows], rstd[kRows];
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      const long long row = row0 + q * slots;
      const T* x = static_cast<const T*>(a.x) + (row < a.rows ? row : row0) * a.x_stride;
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
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      Pair sq = both(0.f);
      const Pair shift = both(-mean[q]);
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          Pair c = pair_add(pair_at(raw[q][j], i), shift);
          if (!VEC || j == CPL - 1) c = inside<VEC>(c, d, tid, kRowThreads, j, i);
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
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Pair w = a.weight ? weight_at<kRowThreads>(w_s, tid, j, i) : both(1.f);
        const Pair b = a.bias ? weight_at<kRowThreads>(b_s, tid, j, i) : both(0.f);
#pragma unroll
        for (int q = 0; q < kRows; ++q) {
          const Pair h = pair_mul(pair_add(pair_at(raw[q][j], i), both(-mean[q])), both(rstd[q]));
          set_pair(out[q], i, pair_fma(h, w, b));
        }
      }
#pragma unroll
      for (int q = 0; q < kRows; ++q) {
        const long long row = row0 + q * slots;
        if (row < a.rows) Cols<VEC>::store(static_cast<T*>(a.y) + row * a.y_stride, d, tid, kRowThreads, j, out[q]);
      }
    }
  }
}

template <class T, bool VEC, int WARPS, int CPL>
__global__ void __launch_bounds__(kNormThreads) norm_backward_kernel(const NormArgs a) {
  constexpr int kRowThreads = 32 * WARPS;
  constexpr int kRowsPerBlock = kNormThreads / kRowThreads;
  // The next row is fetched while this one is computed where registers allow it.
  constexpr bool kAhead = sizeof(T) * CPL <= 8;
  __shared__ float2 scratch[2][WARPS > 1 ? WARPS : 1];
  // The weights, and after the last row (single-warp rows) the warps' sums [8][2][d].
  extern __shared__ float2 shared[];
  const int tid = threadIdx.x % kRowThreads;
  const int d = a.d;
  const float inv_d = 1.f / static_cast<float>(d);
  Pair dw[CPL][4], db[CPL][4];
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[j][i] = db[j][i] = both(0.f);
  }
  grid_dependency_wait();
  if (a.weight && threadIdx.x < kRowThreads)
    stage_weights<T, VEC, kRowThreads, CPL>(a.weight, a.w32, d, tid, 1.f, shared);
  __syncthreads();
  const long long slots = static_cast<long long>(gridDim.x) * kRowsPerBlock;
  Raw8<T> xr[CPL], gr[CPL], xn[CPL], gn[CPL];
  float mean = 0.f, rstd = 0.f, mean_n = 0.f, rstd_n = 0.f;
  const auto fetch = [&](long long row, Raw8<T> (&x8)[CPL], Raw8<T> (&g8)[CPL], float& m, float& r) {
    if (row >= a.rows) return;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    m = a.mean[row];
    r = a.rstd[row];
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      x8[j] = Cols<VEC>::load(x, d, tid, kRowThreads, j);
      g8[j] = Cols<VEC>::load(dy, d, tid, kRowThreads, j);
    }
  };
  int turn = 0;
  long long row = static_cast<long long>(blockIdx.x) * kRowsPerBlock + threadIdx.x / kRowThreads;
  if (kAhead) fetch(row, xn, gn, mean_n, rstd_n);
  for (; row < a.rows; row += slots, turn ^= 1) {
    if constexpr (kAhead) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        xr[j] = xn[j];
        gr[j] = gn[j];
      }
      mean = mean_n;
      rstd = rstd_n;
      fetch(row + slots, xn, gn, mean_n, rstd_n);
    } else {
      fetch(row, xr, gr, mean, rstd);
    }
    // h = x r - mu r. Columns outside the row: dy reads as zero there, so g is zero
    // and they add nothing to any sum.
    const Pair r2 = both(rstd), shift = both(-mean * rstd);
    Pair s1 = both(0.f), s2 = both(0.f);
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Pair g = pair_at(gr[j], i);
        const Pair h = pair_fma(pair_at(xr[j], i), r2, shift);
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
        Raw8<T> out;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const Pair g = pair_at(gr[j], i);
          const Pair h = pair_fma(pair_at(xr[j], i), r2, shift);
          const Pair gw = a.weight ? pair_mul(g, weight_at<kRowThreads>(shared, tid, j, i)) : g;
          set_pair(out, i, pair_mul(r2, pair_add(gw, pair_fma(h, c2, c1))));
        }
        Cols<VEC>::store(dx, d, tid, kRowThreads, j, out);
      }
    }
  }
  grid_launch_dependents();
  if (a.partial == nullptr) return;
  float* block_out = a.partial + static_cast<size_t>(blockIdx.x) * 2 * d;
  float* sums = WARPS > 1 ? block_out : reinterpret_cast<float*>(shared) + static_cast<size_t>(threadIdx.x >> 5) * 2 * d;
  if constexpr (WARPS == 1) __syncthreads();  // the weights are no longer read
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

unsigned norm_grid(long long rows, int rows_per_block, int blocks) {
  return static_cast<unsigned>(std::max<long long>(1, std::min<long long>((rows + rows_per_block - 1) / rows_per_block, blocks)));
}

template <class T, bool VEC, int WARPS, int CPL>
cudaError_t launch_one(const NormArgs& a, bool backward, unsigned grid, cudaStream_t stream) {
  const size_t weights = static_cast<size_t>(CPL) * 4 * 32 * WARPS * sizeof(float2);
  const size_t sums = WARPS == 1 && a.partial ? static_cast<size_t>(kNormWarps) * 2 * a.d * 4 : 0;
  const size_t smem = backward ? std::max(weights, sums) : 2 * weights;
  auto kern = backward ? norm_backward_kernel<T, VEC, WARPS, CPL> : norm_forward_kernel<T, VEC, WARPS, CPL>;
  if (smem > 32 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
  }
  return launch_programmatic(kern, dim3(grid), dim3(kNormThreads), smem, stream, a);
}

template <class T, bool VEC>
cudaError_t launch_width(const NormArgs& a, bool backward, unsigned grid, cudaStream_t stream) {
  const int groups = (a.d + 255) / 256;  // groups of eight columns per lane of one warp
  if (groups <= 1) return launch_one<T, VEC, 1, 1>(a, backward, grid, stream);
  if (groups <= 2) return launch_one<T, VEC, 1, 2>(a, backward, grid, stream);
  if (groups <= 3) return launch_one<T, VEC, 1, 3>(a, backward, grid, stream);
  if (groups <= 4) return launch_one<T, VEC, 1, 4>(a, backward, grid, stream);
  if (groups <= 8) return launch_one<T, VEC, 8, 1>(a, backward, grid, stream);
  if (groups <= 16) return launch_one<T, VEC, 8, 2>(a, backward, grid, stream);
  return launch_one<T, VEC, 8, 4>(a, backward, grid, stream);
}

template <class T>
cudaError_t launch_type(const NormArgs& a, bool backward, unsigned grid, cudaStream_t stream) {
  const auto ok = [&](const void* p, long long stride, size_t es) {
    return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (stride * es) % 16 == 0);
  };
  const size_t es = sizeof(T), ws = a.w32 ? 4 : es;
  const bool vec = a.d % 8 == 0 && ok(a.x, a.x_stride, es) && ok(a.y, a.y_stride, es) && ok(a.dy, a.dy_stride, es) &&
                   ok(a.dx, a.dx_stride, es) && ok(a.weight, 0, ws) && ok(a.bias, 0, ws);
  return vec ? launch_width<T, true>(a, backward, grid, stream) : launch_width<T, false>(a, backward, grid, stream);
}

int row_warps(int d) { return d <= 1024 ? 1 : kNormWarps; }

}  // namespace

int norm_backward_blocks(long long rows, int d, int num_sms) {
  return static_cast<int>(norm_grid(rows, kNormWarps / row_warps(d), 2 * num_sms));
}

cudaError_t norm_launch(const NormArgs& a, int dtype, bool backward, int num_sms, cudaStream_t stream) {
  if (a.d < 1 || a.d > kNormMaxWidth || a.rows < 1) return cudaErrorInvalidValue;
  const unsigned grid = backward ? static_cast<unsigned>(norm_backward_blocks(a.rows, a.d, num_sms))
                                 : norm_grid(a.rows, kNormWarps / row_warps(a.d), 16 * num_sms);
  cudaError_t e;
  switch (dtype) {
    case kSrcF32: e = launch_type<float>(a, backward, grid, stream); break;
    case kSrcF16: e = launch_type<__half>(a, backward, grid, stream); break;
    case kSrcBF16: e = launch_type<__nv_bfloat16>(a, backward, grid, stream); break;
    default: return cudaErrorInvalidValue;
  }
  if (e != cudaSuccess || !backward || a.partial == nullptr) return e;
  return launch_programmatic(norm_finish_kernel, dim3(static_cast<unsigned>((2 * a.d + 31) / 32)), dim3(1024), 0, stream,
                             static_cast<const float*>(a.partial), static_cast<int>(grid), a.d, a.dweight, a.dbias,
                             a.w32 ? static_cast<int>(kSrcF32) : dtype);
}

}  // namespace cvs
