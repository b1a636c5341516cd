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
// A row belongs to one warp (width up to 1024: no shared memory, no barrier) or
// to one block of 8 warps (up to 8192). In the backward pass a block walks rows
// with a stride of the grid and every thread keeps the sums of dw and db for the
// columns it owns, so the weights' gradients cost no traffic per row; the blocks'
// sums go to the workspace and a second small kernel adds them in a fixed order,
// which makes the result the same on every run.
#include "cvs_device.cuh"
#include "cvs_elem.cuh"
#include "cvs_kernels.h"

#include <algorithm>

namespace cvs {

namespace {

constexpr int kNormThreads = 256;
constexpr int kNormWarps = kNormThreads / 32;

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

// One element of the weights: their own fp32, or the rows' type.
template <class T, bool VEC, int THREADS>
__device__ __forceinline__ void load_weights(const void* w, bool w32, int d, int tid, int j, float missing,
                                             float (&out)[8]) {
  if (w == nullptr) {
#pragma unroll
    for (int t = 0; t < 8; ++t) out[t] = missing;
  } else if (w32) {
    const Raw8<float> r = Cols<VEC>::load(static_cast<const float*>(w), d, tid, THREADS, j);
#pragma unroll
    for (int t = 0; t < 8; ++t) out[t] = r.v[t];
  } else {
    const Raw8<T> r = Cols<VEC>::load(static_cast<const T*>(w), d, tid, THREADS, j);
#pragma unroll
    for (int t = 0; t < 8; ++t) out[t] = to_f32(r.v[t]);
  }
}

template <class T, bool VEC, int WARPS, int CPL>
__global__ void __launch_bounds__(kNormThreads) norm_forward_kernel(const NormArgs a) {
  constexpr int kRowThreads = 32 * WARPS;
  constexpr int kRowsPerBlock = kNormThreads / kRowThreads;
  __shared__ float2 scratch[2][WARPS > 1 ? WARPS : 1];
  const int tid = threadIdx.x % kRowThreads;
  const int d = a.d;
  const float inv_d = 1.f / static_cast<float>(d);
  for (long long row = static_cast<long long>(blockIdx.x) * kRowsPerBlock + threadIdx.x / kRowThreads; row < a.rows;
       row += static_cast<long long>(gridDim.x) * kRowsPerBlock) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    Raw8<T> raw[CPL];
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      raw[j] = Cols<VEC>::load(x, d, tid, kRowThreads, j);
#pragma unroll
      for (int t = 0; t < 8; ++t) sum += to_f32(raw[j].v[t]);
    }
    const float mean = row_sum2<WARPS>(sum, 0.f, scratch[0]).x * inv_d;
    float sq = 0.f;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const float c = to_f32(raw[j].v[t]) - mean;
        if (Cols<VEC>::at(tid, kRowThreads, j, t) < d) sq = fmaf(c, c, sq);
      }
    }
    const float rstd = 1.f / sqrtf(row_sum2<WARPS>(sq, 0.f, scratch[1]).x * inv_d + a.eps);
    if (tid == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      float w[8], b[8];
      load_weights<T, VEC, kRowThreads>(a.weight, a.w32, d, tid, j, 1.f, w);
      load_weights<T, VEC, kRowThreads>(a.bias, a.w32, d, tid, j, 0.f, b);
      Raw8<T> out;
#pragma unroll
      for (int t = 0; t < 8; ++t) out.v[t] = from_f32<T>(fmaf((to_f32(raw[j].v[t]) - mean) * rstd, w[t], b[t]));
      Cols<VEC>::store(y, d, tid, kRowThreads, j, out);
    }
  }
}

template <class T, bool VEC, int WARPS, int CPL>
__global__ void __launch_bounds__(kNormThreads) norm_backward_kernel(const NormArgs a) {
  constexpr int kRowThreads = 32 * WARPS;
  constexpr int kRowsPerBlock = kNormThreads / kRowThreads;
  __shared__ float2 scratch[2][WARPS > 1 ? WARPS : 1];
  extern __shared__ float partial[];  // [2][d]: this block's dw and db (rows held by single warps)
  const int tid = threadIdx.x % kRowThreads;
  const int d = a.d;
  const float inv_d = 1.f / static_cast<float>(d);
  float dw[CPL][8], db[CPL][8];
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
#pragma unroll
    for (int t = 0; t < 8; ++t) dw[j][t] = db[j][t] = 0.f;
  }
  int turn = 0;
  for (long long row = static_cast<long long>(blockIdx.x) * kRowsPerBlock + threadIdx.x / kRowThreads; row < a.rows;
       row += static_cast<long long>(gridDim.x) * kRowsPerBlock, turn ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    const float mean = a.mean[row], rstd = a.rstd[row];
    Raw8<T> xr[CPL], gr[CPL];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      xr[j] = Cols<VEC>::load(x, d, tid, kRowThreads, j);
      gr[j] = Cols<VEC>::load(dy, d, tid, kRowThreads, j);
    }
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      float w[8];
      load_weights<T, VEC, kRowThreads>(a.weight, a.w32, d, tid, j, 1.f, w);
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const float g = to_f32(gr[j].v[t]);  // zero outside the row
        const float h = (to_f32(xr[j].v[t]) - mean) * rstd;
        const float gw = g * w[t];
        // Columns outside the row: dy reads as zero there, so they add nothing.
        s1 += Cols<VEC>::at(tid, kRowThreads, j, t) < d ? gw : 0.f;
        s2 += Cols<VEC>::at(tid, kRowThreads, j, t) < d ? gw * h : 0.f;
        dw[j][t] = fmaf(g, h, dw[j][t]);
        db[j][t] += g;
      }
    }
    const float2 s = row_sum2<WARPS>(s1, s2, scratch[turn]);
    if (a.dx) {
      const float c1 = s.x * inv_d, c2 = s.y * inv_d;
      T* dx = static_cast<T*>(a.dx) + row * a.dx_stride;
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        float w[8];
        load_weights<T, VEC, kRowThreads>(a.weight, a.w32, d, tid, j, 1.f, w);
        Raw8<T> out;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const float h = (to_f32(xr[j].v[t]) - mean) * rstd;
          out.v[t] = from_f32<T>(rstd * (to_f32(gr[j].v[t]) * w[t] - c1 - h * c2));
        }
        Cols<VEC>::store(dx, d, tid, kRowThreads, j, out);
      }
    }
  }
  if (a.partial == nullptr) return;
  float* block_out = a.partial + static_cast<size_t>(blockIdx.x) * 2 * d;
  if constexpr (WARPS > 1) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int c = Cols<VEC>::at(tid, kRowThreads, j, t);
        if (c < d) {
          block_out[c] = dw[j][t];
          block_out[d + c] = db[j][t];
        }
      }
    }
  } else {
    // The warps add their sums one after another: a fixed order.
    for (int w = 0; w < kNormWarps; ++w) {
      if ((threadIdx.x >> 5) == w) {
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            const int c = Cols<VEC>::at(tid, kRowThreads, j, t);
            if (c < d) {
              partial[c] = w == 0 ? dw[j][t] : partial[c] + dw[j][t];
              partial[d + c] = w == 0 ? db[j][t] : partial[d + c] + db[j][t];
            }
          }
        }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * d; i += kNormThreads) block_out[i] = partial[i];
  }
}

// out[c] = sum over blocks of partial[block][c], in a fixed order: 32 columns a
// block, 8 threads a column.
__global__ void __launch_bounds__(256) norm_finish_kernel(const float* partial, int blocks, int d, void* dweight,
                                                          void* dbias, int out_dtype) {
  __shared__ float sums[8][32];
  const int c = blockIdx.x * 32 + threadIdx.x % 32;  // column of [2][d]
  const int part = threadIdx.x / 32;
  float s = 0.f;
  if (c < 2 * d)
    for (int b = part; b < blocks; b += 8) s += partial[static_cast<size_t>(b) * 2 * d + c];
  sums[part][threadIdx.x % 32] = s;
  __syncthreads();
  if (part != 0 || c >= 2 * d) return;
  for (int p = 1; p < 8; ++p) s += sums[p][threadIdx.x];
  void* out = c < d ? dweight : dbias;
  const int i = c < d ? c : c - d;
  if (out == nullptr) return;
  if (out_dtype == kSrcF32) static_cast<float*>(out)[i] = s;
  else if (out_dtype == kSrcF16) static_cast<__half*>(out)[i] = __float2half_rn(s);
  else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(s);
}

unsigned norm_grid(long long rows, int warps_per_row, int blocks) {
  const int per_block = kNormWarps / warps_per_row;
  return static_cast<unsigned>(std::max<long long>(1, std::min<long long>((rows + per_block - 1) / per_block, blocks)));
}

template <class T, bool VEC, int WARPS, int CPL>
cudaError_t launch_one(const NormArgs& a, bool backward, unsigned grid, cudaStream_t stream) {
  if (backward) {
    const size_t smem = WARPS == 1 && a.partial ? static_cast<size_t>(a.d) * 8 : 0;
    norm_backward_kernel<T, VEC, WARPS, CPL><<<grid, kNormThreads, smem, stream>>>(a);
  } else {
    norm_forward_kernel<T, VEC, WARPS, CPL><<<grid, kNormThreads, 0, stream>>>(a);
  }
  return cudaGetLastError();
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

int row_warps(int d) { return d <= 1024 ? 1 : 8; }

}  // namespace

int norm_backward_blocks(long long rows, int d, int num_sms) {
  return static_cast<int>(norm_grid(rows, row_warps(d), 2 * num_sms));
}

cudaError_t norm_launch(const NormArgs& a, int dtype, bool backward, int num_sms, cudaStream_t stream) {
  if (a.d < 1 || a.d > kNormMaxWidth || a.rows < 1) return cudaErrorInvalidValue;
  const unsigned grid = backward ? static_cast<unsigned>(norm_backward_blocks(a.rows, a.d, num_sms))
                                 : norm_grid(a.rows, row_warps(a.d), 8 * num_sms);
  cudaError_t e;
  switch (dtype) {
    case kSrcF32: e = launch_type<float>(a, backward, grid, stream); break;
    case kSrcF16: e = launch_type<__half>(a, backward, grid, stream); break;
    case kSrcBF16: e = launch_type<__nv_bfloat16>(a, backward, grid, stream); break;
    default: return cudaErrorInvalidValue;
  }
  if (e != cudaSuccess || !backward || a.partial == nullptr) return e;
  norm_finish_kernel<<<(2 * a.d + 31) / 32, 256, 0, stream>>>(a.partial, static_cast<int>(grid), a.d, a.dweight,
                                                              a.dbias, a.w32 ? static_cast<int>(kSrcF32) : dtype);
  return cudaGetLastError();
}

}  // namespace cvs
