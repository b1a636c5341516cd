// Element access shared by the adapter kernels (layer norm, linear, preference
// loss): eight consecutive or eight strided elements of a row as fp32, from
// fp32, fp16 or bf16 storage.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <type_traits>

namespace cvs {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Base-2 exponential and reciprocal of the special-function unit (2 ulp and 1 ulp).
__device__ __forceinline__ float exp2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Two fp32 values in one register pair, for the instructions that work on both.
struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair pair_of(float lo, float hi) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ void split(Pair p, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p.v));
}
__device__ __forceinline__ Pair pair_fma(Pair a, Pair b, Pair c) {
  Pair p;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return p;
}
__device__ __forceinline__ Pair pair_mul(Pair a, Pair b) {
  Pair p;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
  return p;
}
__device__ __forceinline__ Pair pair_add(Pair a, Pair b) {
  Pair p;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
  return p;
}

// Eight elements as stored: 16 bytes (halves) or 32 bytes (fp32).
template <class T>
struct alignas(16) Raw8 {
  T v[8];
};

template <class T>
__device__ __forceinline__ Raw8<T> zero8() {
  Raw8<T> r;
#pragma unroll
  for (int t = 0; t < 8; ++t) r.v[t] = from_f32<T>(0.f);
  return r;
}

// Hides the elements' history from the compiler, which would otherwise keep their
// converted values in registers from one use to the next instead of converting again.
template <class T>
__device__ __forceinline__ void forget(Raw8<T>& r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(r) / 4); ++i) asm volatile("" : "+r"(u[i]));
}

// p must be 16-byte aligned.
template <class T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
  Raw8<T> r;
  const uint4* s = reinterpret_cast<const uint4*>(p);
  uint4* d = reinterpret_cast<uint4*>(&r);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(r) / 16); ++i) d[i] = s[i];
  return r;
}

template <class T>
__device__ __forceinline__ void store8(T* p, const Raw8<T>& r) {
  const uint4* s = reinterpret_cast<const uint4*>(&r);
  uint4* d = reinterpret_cast<uint4*>(p);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(r) / 16); ++i) d[i] = s[i];
}

// Elements 2 i and 2 i + 1 of eight, as fp32.
template <class T>
__device__ __forceinline__ Pair pair_at(const Raw8<T>& r, int i) {
  if constexpr (sizeof(T) == 4) {
    return pair_of(r.v[2 * i], r.v[2 * i + 1]);
  } else {
    const uint32_t u = reinterpret_cast<const uint32_t*>(&r)[i];
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return pair_of(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
      return pair_of(f.x, f.y);
    }
  }
}
template <class T>
__device__ __forceinline__ void set_pair(Raw8<T>& r, int i, Pair p) {
  float lo, hi;
  split(p, lo, hi);
  if constexpr (sizeof(T) == 4) {
    r.v[2 * i] = lo;
    r.v[2 * i + 1] = hi;
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    reinterpret_cast<__nv_bfloat162*>(&r)[i] = __floats2bfloat162_rn(lo, hi);
  } else {
    reinterpret_cast<__half2*>(&r)[i] = __floats2half2_rn(lo, hi);
  }
}
__device__ __forceinline__ float pair_total(Pair p) {
  float lo, hi;
  split(p, lo, hi);
  return lo + hi;
}
__device__ __forceinline__ Pair both(float v) { return pair_of(v, v); }

// The j-th group of eight columns that thread `tid` of `threads` owns in a row
// of d columns. Aligned rows (VEC): eight consecutive columns, one 16-byte (or
// two) access; d is a multiple of 8. Otherwise eight single columns `threads`
// apart, so that a warp's scalar accesses still cover consecutive elements.
template <bool VEC>
struct Cols {
  static __device__ __forceinline__ int at(int tid, int threads, int j, int t) {
    return VEC ? (tid + threads * j) * 8 + t : tid + threads * (8 * j + t);
  }
  template <class T>
  static __device__ __forceinline__ Raw8<T> load(const T* row, int d, int tid, int threads, int j) {
    if constexpr (VEC) {
      const int c = (tid + threads * j) * 8;
      return c < d ? load8(row + c) : zero8<T>();
    } else {
      Raw8<T> r = zero8<T>();
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int c = at(tid, threads, j, t);
        if (c < d) r.v[t] = row[c];
      }
      return r;
    }
  }
  template <class T>
  static __device__ __forceinline__ void store(T* row, int d, int tid, int threads, int j, const Raw8<T>& r) {
    if constexpr (VEC) {
      const int c = (tid + threads * j) * 8;
      if (c < d) store8(row + c, r);
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int c = at(tid, threads, j, t);
        if (c < d) row[c] = r.v[t];
      }
    }
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

}  // namespace cvs
