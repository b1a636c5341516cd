// Preference loss of queries over rows of the corpus, with its gradient.
//
// The scores s_i = scale u.x_i (u = q, or q / max(|q|, 1e-12) for cosine) define a
// choice p(i | q) = softmax_i(s_i) over the corpus. For a chosen row c and a
// rejected row r the log ratio log p(c) - log p(r) = s_c - s_r needs no sum over
// the corpus, and the margin against a reference query is
//
//   m = scale (u - u_ref) . (x_c - x_r)
//   loss = (1 - e) softplus(-m) + e softplus(m)          (e: label smoothing)
//   dloss/dm = e - sigmoid(-m)
//   dloss/du = sum over the query's pairs of (dloss/dm) scale (x_c - x_r)
//   dloss/dq = (dloss/du - u (u . dloss/du)) / |q|        (cosine)
//
// Bound by the gather of corpus rows from HBM: each row is read once, the chosen
// one stays in registers, and the gradient is accumulated in the same pass that
// computes the margins, in fp32 registers. The division by the number of pairs
// and by whatever scales the loss follows in preference_grad_kernel, which turns
// the kept fp32 sums into the queries' type: a half-precision gradient is
// rounded once, after its scaling.
//
// One warp takes a query, or 2, 4 or 8 warps share its rejected rows when there
// are too few queries to fill the GPU with one warp each; the shares are added
// through shared memory in a fixed order. Ids below zero mark absent rows (a query
// without a chosen row, a shorter list of rejected ones): their pairs give margin
// zero and do not count. An id that is not a row of the corpus reads nothing and
// makes its pair's margin NaN, and so the loss.
#include "cvs_device.cuh"
#include "cvs_elem.cuh"
#include "cvs_kernels.h"

#include <algorithm>
#include <cmath>

namespace cvs {

namespace {

constexpr int kPrefThreads = 256;
constexpr int kPrefWarps = kPrefThreads / 32;

// Group j of this lane's query columns as fp32 (zeros outside).
__device__ __forceinline__ void load_query(const void* q, int dtype, long long base, int d, bool vec, int lane, int j,
                                           float (&out)[8]) {
  const int c0 = (lane + 32 * j) * 8;
  if (vec && c0 < d) {
    if (dtype == kSrcF32) {
      const Raw8<float> r = load8(static_cast<const float*>(q) + base + c0);
#pragma unroll
      for (int t = 0; t < 8; ++t) out[t] = r.v[t];
    } else if (dtype == kSrcF16) {
      const Raw8<__half> r = load8(static_cast<const __half*>(q) + base + c0);
#pragma unroll
      for (int t = 0; t < 8; ++t) out[t] = to_f32(r.v[t]);
    } else {
      const Raw8<__nv_bfloat16> r = load8(static_cast<const __nv_bfloat16*>(q) + base + c0);
#pragma unroll
      for (int t = 0; t < 8; ++t) out[t] = to_f32(r.v[t]);
    }
    return;
  }
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const int c = c0 + t;
    float v = 0.f;
    if (c < d) {
      if (dtype == kSrcF32) v = static_cast<const float*>(q)[base + c];
      else if (dtype == kSrcF16) v = to_f32(static_cast<const __half*>(q)[base + c]);
      else v = to_f32(static_cast<const __nv_bfloat16*>(q)[base + c]);
    }
    out[t] = v;
  }
}

// Loads a query row, divides it by its clamped norm for cosine; returns the divisor.
template <int CPL>
__device__ __forceinline__ float load_unit(const void* q, int dtype, long long base, int d, bool vec, bool cosine,
                                           int lane, float (&u)[CPL][8]) {
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
    load_query(q, dtype, base, d, vec, lane, j, u[j]);
#pragma unroll
    for (int t = 0; t < 8; ++t) ss = fmaf(u[j][t], u[j][t], ss);
  }
  if (!cosine) return 1.f;
  const float norm = fmaxf(sqrtf(warp_sum(ss)), 1e-12f);
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
#pragma unroll
    for (int t = 0; t < 8; ++t) u[j][t] = __fdiv_rn(u[j][t], norm);
  }
  return norm;
}

template <int CPL>
__device__ __forceinline__ void load_row(const __half* x, int d_pad, int lane, Raw8<__half> (&r)[CPL]) {
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
    const int c = (lane + 32 * j) * 8;
    r[j] = c < d_pad ? load8(x + c) : zero8<__half>();
  }
}

template <int CPL>
__global__ void __launch_bounds__(kPrefThreads) preference_kernel(const PreferenceArgs a) {
  extern __shared__ float shares[];  // [warps][d_pad] gradient shares when several warps take one query
  __shared__ float2 totals[kPrefWarps];
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int share = warp % a.warps_per_query;
  const int qpb = kPrefWarps / a.warps_per_query;
  const long long q = static_cast<long long>(blockIdx.x) * qpb + warp / a.warps_per_query;
  const bool live = q < a.b;
  float g[CPL][8];
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
#pragma unroll
    for (int t = 0; t < 8; ++t) g[j][t] = 0.f;
  }
  float loss = 0.f;
  float count = 0.f;
  if (live) {
    const long long c = a.chosen[q];
    const bool bad_c = c >= a.n;
    float u[CPL][8];
    load_unit<CPL>(a.q, a.q_dtype, q * a.q_stride, a.d, a.q_vec, a.cosine, lane, u);
    if (a.ref) {
      float v[CPL][8];
      load_unit<CPL>(a.ref, a.ref_dtype, q * a.ref_stride, a.d, a.ref_vec, a.cosine, lane, v);
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
#pragma unroll
        for (int t = 0; t < 8; ++t) u[j][t] -= v[j][t];
      }
    }
    Raw8<__half> xc[CPL];
    if (c >= 0 && !bad_c) load_row<CPL>(a.x + static_cast<size_t>(c) * a.d_pad, a.d_pad, lane, xc);
    for (int r = share; r < a.r; r += a.warps_per_query) {
      const long long id = a.rejected[q * a.rejected_stride + r];
      float m = 0.f;
      if (c >= 0 && id >= 0) {
        count += 1.f;
        if (bad_c || id >= a.n) {
          m = __int_as_float(0x7fffffff);
          loss += m;
#pragma unroll
          for (int j = 0; j < CPL; ++j) {
#pragma unroll
            for (int t = 0; t < 8; ++t) g[j][t] += m;
          }
        } else {
          Raw8<__half> xr[CPL];
          load_row<CPL>(a.x + static_cast<size_t>(id) * a.d_pad, a.d_pad, lane, xr);
          float dot = 0.f;
#pragma unroll
          for (int j = 0; j < CPL; ++j) {
#pragma unroll
            for (int t = 0; t < 8; ++t) dot = fmaf(u[j][t], to_f32(xc[j].v[t]) - to_f32(xr[j].v[t]), dot);
          }
          m = a.scale * warp_sum(dot);
          const float tail = log1pf(expf(-fabsf(m)));
          loss += (1.f - a.smoothing) * (fmaxf(-m, 0.f) + tail) + a.smoothing * (fmaxf(m, 0.f) + tail);
          const float slope = (a.smoothing - 1.f / (1.f + expf(m))) * a.scale;
#pragma unroll
          for (int j = 0; j < CPL; ++j) {
#pragma unroll
            for (int t = 0; t < 8; ++t) g[j][t] = fmaf(slope, to_f32(xc[j].v[t]) - to_f32(xr[j].v[t]), g[j][t]);
          }
        }
      }
      if (lane == 0) a.margins[q * a.r + r] = m;
    }
  }
  if (lane == 0) totals[warp] = make_float2(loss, count);
  if (a.grad != nullptr && a.warps_per_query > 1) {
    if (live && share != 0) {
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const int col = (lane + 32 * j) * 8 + t;
          if (col < a.d) shares[static_cast<size_t>(warp) * a.d_pad + col] = g[j][t];
        }
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float2 s = make_float2(0.f, 0.f);
    for (int w = 0; w < kPrefWarps; ++w) {
      s.x += totals[w].x;
      s.y += totals[w].y;
    }
    a.partial[blockIdx.x] = s;
  }
  if (a.grad == nullptr || !live || share != 0) return;
  for (int w = 1; w < a.warps_per_query; ++w) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int col = (lane + 32 * j) * 8 + t;
        if (col < a.d) g[j][t] += shares[static_cast<size_t>(warp + w) * a.d_pad + col];
      }
    }
  }
  if (a.cosine) {
    float u[CPL][8];
    const float norm = load_unit<CPL>(a.q, a.q_dtype, q * a.q_stride, a.d, a.q_vec, true, lane, u);
    float along = 0.f;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
#pragma unroll
      for (int t = 0; t < 8; ++t) along = fmaf(u[j][t], g[j][t], along);
    }
    along = norm > 1e-12f ? warp_sum(along) : 0.f;  // below the clamp the divisor is a constant
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
#pragma unroll
      for (int t = 0; t < 8; ++t) g[j][t] = __fdiv_rn(g[j][t] - u[j][t] * along, norm);
    }
  }
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
    const int c0 = (lane + 32 * j) * 8;
    if (c0 + 8 <= a.grad_stride) {
      Raw8<float> out;
#pragma unroll
      for (int t = 0; t < 8; ++t) out.v[t] = g[j][t];
      store8(a.grad + q * a.grad_stride + c0, out);
    }
  }
}

// loss = (sum of the blocks' losses) * weight, weight = 1 / max(pairs, 1) (mean) or 1 (sum).
__global__ void __launch_bounds__(256) preference_finish_kernel(const float2* partial, int blocks, int mean,
                                                                float* loss, float* weight) {
  __shared__ float2 sums[256];
  float2 s = make_float2(0.f, 0.f);
  for (int i = threadIdx.x; i < blocks; i += 256) {
    s.x += partial[i].x;
    s.y += partial[i].y;
  }
  sums[threadIdx.x] = s;
  __syncthreads();
  for (int n = 128; n > 0; n >>= 1) {
    if (threadIdx.x < n) {
      sums[threadIdx.x].x += sums[threadIdx.x + n].x;
      sums[threadIdx.x].y += sums[threadIdx.x + n].y;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const float w = mean ? 1.f / fmaxf(sums[0].y, 1.f) : 1.f;
    *loss = sums[0].x * w;
    *weight = w;
  }
}

// dq = grad * weight * upstream, rounded once to the queries' type.
template <class T>
__global__ void __launch_bounds__(256) preference_grad_kernel(const float* grad, long long grad_stride, long long b,
                                                              int d, const float* weight, const float* upstream,
                                                              T* dq) {
  const float s = *weight * *upstream;
  const long long groups = grad_stride / 8;
  const bool vec = d % 8 == 0 && (reinterpret_cast<uintptr_t>(dq) & 15u) == 0;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < b * groups;
       i += static_cast<long long>(gridDim.x) * 256) {
    const long long row = i / groups;
    const int c = static_cast<int>(i - row * groups) * 8;
    if (c >= d) continue;
    const Raw8<float> g = load8(grad + row * grad_stride + c);
    Raw8<T> out;
#pragma unroll
    for (int t = 0; t < 8; ++t) out.v[t] = from_f32<T>(g.v[t] * s);
    T* p = dq + row * d + c;
    if (vec) {
      store8(p, out);
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t)
        if (c + t < d) p[t] = out.v[t];
    }
  }
}

int pref_warps(long long b, int r, int num_sms) {
  // One warp a query once the queries alone give every SM 16 warps; fewer
  // queries share their rejected rows among up to 8 warps.
  int w = 1;
  while (w < kPrefWarps && 2 * w <= r && b * w < 16LL * num_sms) w *= 2;
  return w;
}

template <int CPL>
cudaError_t pref_launch_one(const PreferenceArgs& a, unsigned grid, size_t smem, cudaStream_t stream) {
  if (smem > 32 * 1024) {  // static shared memory counts towards the default limit of 48 KB
    const cudaError_t e = cudaFuncSetAttribute(preference_kernel<CPL>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(smem));
    if (e != cudaSuccess) return e;
  }
  preference_kernel<CPL><<<grid, kPrefThreads, smem, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

int preference_blocks(long long b, int r, int num_sms) {
  const int qpb = kPrefWarps / pref_warps(b, r, num_sms);
  return static_cast<int>((b + qpb - 1) / qpb);
}

cudaError_t preference_launch(PreferenceArgs a, int mean, float* loss, float* weight, int num_sms, cudaStream_t stream) {
  a.warps_per_query = pref_warps(a.b, a.r, num_sms);
  const unsigned grid = static_cast<unsigned>(preference_blocks(a.b, a.r, num_sms));
  const size_t smem = a.grad && a.warps_per_query > 1 ? static_cast<size_t>(kPrefWarps) * a.d_pad * 4 : 0;
  const int cpl = (a.d_pad / 8 + 31) / 32;
  cudaError_t e;
  if (a.b == 0) e = cudaSuccess;
  else if (cpl <= 1) e = pref_launch_one<1>(a, grid, smem, stream);
  else if (cpl <= 2) e = pref_launch_one<2>(a, grid, smem, stream);
  else if (cpl <= 3) e = pref_launch_one<3>(a, grid, smem, stream);
  else if (cpl <= 4) e = pref_launch_one<4>(a, grid, smem, stream);
  else if (cpl <= 8) e = pref_launch_one<8>(a, grid, smem, stream);
  else return cudaErrorInvalidValue;
  if (e != cudaSuccess) return e;
  preference_finish_kernel<<<1, 256, 0, stream>>>(a.partial, static_cast<int>(grid), mean, loss, weight);
  return cudaGetLastError();
}

cudaError_t preference_grad_launch(const float* grad, long long grad_stride, long long b, int d, const float* weight,
                                   const float* upstream, int q_dtype, void* dq, int num_sms, cudaStream_t stream) {
  const long long items = b * (grad_stride / 8);
  const unsigned grid = static_cast<unsigned>(std::max<long long>(1, std::min<long long>((items + 255) / 256, 8LL * num_sms)));
  switch (q_dtype) {
    case kSrcF32:
      preference_grad_kernel<<<grid, 256, 0, stream>>>(grad, grad_stride, b, d, weight, upstream, static_cast<float*>(dq));
      break;
    case kSrcF16:
      preference_grad_kernel<<<grid, 256, 0, stream>>>(grad, grad_stride, b, d, weight, upstream, static_cast<__half*>(dq));
      break;
    case kSrcBF16:
      preference_grad_kernel<<<grid, 256, 0, stream>>>(grad, grad_stride, b, d, weight, upstream,
                                                       static_cast<__nv_bfloat16*>(dq));
      break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace cvs
