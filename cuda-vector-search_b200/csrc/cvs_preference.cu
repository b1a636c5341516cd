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
// Each warp has two stages of row buffers in shared memory, filled by bulk copies (one
// a row, a multiple of 128 bytes) ahead of the arithmetic and across its queries, so the
// bytes in flight do not depend on registers: with rows loaded into registers one or two
// ahead, 16384 queries x 4 rejected rows of 768 columns took 113 us at an occupancy of 8
// to 16 warps an SM. A stage's copies are issued together, a lane each, and waited for
// together, which keeps the arithmetic's share of the instructions up. That size takes 61
// us now (202 MB of rows, queries and results: 31 us at HBM rate), held by instructions
// and their latency at the two blocks an SM that the registers allow.
//
// One warp takes a query, or 2, 4 or 8 warps share its rejected rows when there
// are too few queries to fill the GPU with one warp each; the shares are added
// through shared memory in a fixed order. Ids below zero mark absent rows (a query
// without a chosen row, a shorter list of rejected ones): their pairs give margin
// zero and do not count, and no value that lies there (in a padded query, in a chosen row
// whose rejected rows are all absent) reaches a result, NaN and infinity included. An id that is not a row of the corpus reads nothing and
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
constexpr int kPrefStageRows = 8;  // most row buffers of a warp's stage
constexpr int kAbsent = -1, kOutside = -2;  // what a position may hold instead of a row
constexpr float kLog2E = 1.44269504088896341f, kLog2ELow = 1.92596299e-08f, kLn2 = 0.69314718056f;  // log2(e) = kLog2E + kLog2ELow

// This lane's columns of a query row as pairs of fp32 (zeros outside).
template <class T, int CPL>
__device__ __forceinline__ void load_pairs_of(const T* row, int d, bool vec, int lane, Pair (&u)[CPL][4]) {
  if (vec) {
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      const Raw8<T> r = Cols<true>::load(row, d, lane, 32, j);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[j][i] = pair_at(r, i);
    }
  } else {
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = (lane + 32 * j) * 8 + 2 * i;
        u[j][i] = pair_of(c < d ? to_f32(row[c]) : 0.f, c + 1 < d ? to_f32(row[c + 1]) : 0.f);
      }
    }
  }
}
template <int CPL>
__device__ __forceinline__ void load_pairs(const void* q, int dtype, long long base, int d, bool vec, int lane,
                                           Pair (&u)[CPL][4]) {
  if (dtype == kSrcF32) load_pairs_of(static_cast<const float*>(q) + base, d, vec, lane, u);
  else if (dtype == kSrcF16) load_pairs_of(static_cast<const __half*>(q) + base, d, vec, lane, u);
  else load_pairs_of(static_cast<const __nv_bfloat16*>(q) + base, d, vec, lane, u);
}

// Asks for a query row that is read later.
__device__ __forceinline__ void prefetch_row(const void* q, int dtype, long long base, int d, int lane) {
  const int es = dtype == kSrcF32 ? 4 : 2;
  const char* row = static_cast<const char*>(q) + base * es;
  for (int c = lane * 128; c < d * es; c += 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + c));
}

// What a cosine query is multiplied with: inv + lo = 1 / max(|q|, 1e-12) to about twice
// fp32's digits. A margin against a reference is a small difference of two unit vectors,
// and a rounding of the factor, unlike one of an element, moves all of the vector one
// way: lo is one Newton step's correction of inv, from the sum of squares itself.
struct UnitScale {
  float inv = 1.f, lo = 0.f;
  bool clamped = false;
};
template <int CPL>
__device__ __forceinline__ UnitScale unit_scale(const Pair (&u)[CPL][4]) {
  Pair sq = both(0.f), sq2 = both(0.f);
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      sq = pair_fma(u[j][i], u[j][i], sq);
      sq2 = pair_fma(u[j][i + 1], u[j][i + 1], sq2);
    }
  }
  const float ss = warp_sum(pair_total(pair_add(sq, sq2)));
  const float norm = sqrtf(ss);
  UnitScale s;
  s.clamped = norm <= 1e-12f;
  s.inv = __fdiv_rn(1.f, fmaxf(norm, 1e-12f));
  if (!s.clamped && norm < 1e18f) {  // (beyond, the sum of squares is near overflow)
    const float p = ss * s.inv, rest = fmaf(ss, s.inv, -p);
    s.lo = 0.5f * s.inv * (fmaf(-p, s.inv, 1.f) - rest * s.inv);
  }
  return s;
}

// Group j of a staged row (zeros behind the row, which only the last group can reach).
template <int CPL>
__device__ __forceinline__ Raw8<__half> staged(const uint8_t* row, int d_pad, int lane, int j) {
  const int c = (lane + 32 * j) * 8;
  return j < CPL - 1 || c < d_pad ? load8(reinterpret_cast<const __half*>(row) + c) : zero8<__half>();
}

// The rows a warp reads, in order (for each of its queries the chosen row, then this
// warp's rejected ones), through two stages of `rows` buffers each.
struct RowStream {
  const PreferenceArgs& a;
  long long query0, query_step;  // this warp's queries
  int per_query;                 // rows per query: 1 + rejected rows of this warp
  int share, lane, rows, total;
  uint32_t row_bytes;
  uint8_t* ring;
  uint64_t* bars;                // one per stage
  volatile int* abort;
  int asked = 0;                 // positions asked for, a multiple of `rows`
  int stage = 0, at = 0;         // the next row to read
  uint32_t parity = 0;           // bit per stage
  // Bit per buffer, of the stage being read and of the other one: its row was copied; no
  // row at all (neither: an id outside the corpus).
  uint32_t copied = 0, copied_next = 0, absent = 0, absent_next = 0;
  bool stopped = false;          // a wait ran out: nothing more is asked for
  int ahead = kAbsent;           // this lane's id of the stage asked for next

  // A row of the corpus, kAbsent or kOutside.
  __device__ __forceinline__ int id_at(int p) const {
    if (lane >= rows || p >= total) return kAbsent;
    const int k = p / per_query, e = p - k * per_query;
    const long long q = query0 + k * query_step;
    const long long id =
        e == 0 ? a.chosen[q] : a.rejected[q * a.rejected_stride + static_cast<long long>(e - 1) * a.warps_per_query + share];
    return id < 0 ? kAbsent : (id < a.n ? static_cast<int>(id) : kOutside);
  }
  // Copies the rows of the next `rows` positions into a stage, a lane each, and reads the
  // ids of those behind them.
  __device__ __forceinline__ void ask(int s) {
    const uint32_t have = __ballot_sync(0xffffffffu, ahead >= 0);
    absent_next = __ballot_sync(0xffffffffu, ahead == kAbsent);
    copied_next = have;
    if (have != 0 && lane == 0) mbar_arrive_expect_tx(bars + s, __popc(have) * row_bytes);
    __syncwarp();
    if (ahead >= 0)
      bulk_load(ring + (s * rows + lane) * row_bytes, a.x + static_cast<size_t>(ahead) * a.d_pad, row_bytes, bars + s);
    asked += rows;
    ahead = id_at(asked + lane);
  }
  __device__ __forceinline__ void init() {
    ahead = id_at(lane);
    ask(0);
    copied = copied_next;
    absent = absent_next;
    ask(1);
    arrive();
  }
  // Waits for the stage's copies (none: nothing to wait for).
  __device__ __forceinline__ void arrive() {
    if (copied == 0 || stopped) return;
    if (__all_sync(0xffffffffu, mbar_wait(bars + stage, parity >> stage & 1, abort, a.err, 40))) parity ^= 1u << stage;
    else stopped = true;
  }
  __device__ __forceinline__ bool gone() const { return absent >> at & 1; }
  __device__ __forceinline__ bool there() const { return !stopped && (copied >> at & 1); }
  __device__ __forceinline__ const uint8_t* row() const { return ring + (stage * rows + at) * row_bytes; }
  // The row has been read; after a stage's last one the stage is refilled.
  __device__ __forceinline__ void next() {
    if (++at < rows) return;
    __syncwarp();
    copied = copied_next;
    absent = absent_next;
    if (!stopped) ask(stage);
    at = 0;
    stage ^= 1;
    arrive();
  }
  // After a wait that ran out: lets copies under way land.
  __device__ __forceinline__ void drain() {
    if (!stopped || lane != 0) return;
    if (copied != 0) mbar_wait_drain(bars + stage, parity >> stage & 1);
    if (copied_next != 0) mbar_wait_drain(bars + (stage ^ 1), parity >> (stage ^ 1) & 1);
  }
};

// softplus(v) = log(1 + e^v), without overflow and without losing small values.
__device__ __forceinline__ float softplus_of(float v) { return fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))); }

template <int CPL>
__global__ void __launch_bounds__(kPrefThreads, CPL <= 4 ? 2 : 1) preference_kernel(const __grid_constant__ PreferenceArgs a) {
  // [warps][2 stages][rows] row buffers, then (several warps a query) the gradient's shares [warps][d_pad].
  extern __shared__ __align__(128) uint8_t rows_s[];
  __shared__ float2 totals[kPrefWarps];
  __shared__ int present[kPrefWarps];  // whether the warp's share of the query has a pair
  __shared__ __align__(8) uint64_t bars[kPrefWarps][2];
  __shared__ int abort_s;
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int wpq = a.warps_per_query;
  const int share = warp % wpq;
  const int qpb = kPrefWarps / wpq;
  const uint32_t row_bytes = static_cast<uint32_t>(a.d_pad) * 2;
  const size_t ring_bytes = static_cast<size_t>(2 * a.stage_rows) * row_bytes;
  float* shares = reinterpret_cast<float*>(rows_s + kPrefWarps * ring_bytes);
  if (lane == 0) {
    mbar_init(&bars[warp][0], 1);
    mbar_init(&bars[warp][1], 1);
    if (warp == 0) abort_s = 0;
    fence_barrier_init();
  }
  __syncthreads();
  grid_dependency_wait();

  const int mine = (a.r - share + wpq - 1) / wpq;  // rejected rows: share, share + wpq, ...
  const long long first = static_cast<long long>(blockIdx.x) * qpb + warp / wpq;
  const long long step = static_cast<long long>(gridDim.x) * qpb;
  const int total = first < a.b ? static_cast<int>((a.b - first + step - 1) / step) * (mine + 1) : 0;
  RowStream stream{a, first, step, mine + 1, share, lane, a.stage_rows, total, row_bytes, rows_s + warp * ring_bytes,
                   bars[warp], &abort_s};
  stream.init();
  float loss = 0.f, count = 0.f;  // per lane

  // Every warp of the block takes part in every round: the shares need barriers.
  const long long rounds = (a.b - static_cast<long long>(blockIdx.x) * qpb + step - 1) / step;
  for (long long round = 0; round < rounds; ++round) {
    const long long q = first + round * step;
    const bool live = q < a.b;
    Pair g[CPL][4];
    UnitScale unit;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) g[j][i] = both(0.f);
    }
    Raw8<__half> xc[CPL];
    float slopes = 0.f;  // sum of the slopes
    bool any = false;    // this warp has a pair
    if (live) {
      if (q + step < a.b) {
        prefetch_row(a.q, a.q_dtype, (q + step) * a.q_stride, a.d, lane);
        if (a.ref) prefetch_row(a.ref, a.ref_dtype, (q + step) * a.ref_stride, a.d, lane);
      }
      Pair u[CPL][4];
      load_pairs<CPL>(a.q, a.q_dtype, q * a.q_stride, a.d, a.q_vec, lane, u);
      if (a.ref) load_pairs<CPL>(a.ref, a.ref_dtype, q * a.ref_stride, a.d, a.ref_vec, lane, g);
      if (a.cosine) {
        unit = unit_scale<CPL>(u);
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) u[j][i] = pair_fma(u[j][i], both(unit.inv), pair_mul(u[j][i], both(unit.lo)));
        }
      }
      if (a.ref) {
        UnitScale r;
        if (a.cosine) r = unit_scale<CPL>(g);
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            u[j][i] = pair_fma(g[j][i], both(-r.inv), pair_fma(g[j][i], both(-r.lo), u[j][i]));
            g[j][i] = both(0.f);
          }
        }
      }
      const bool gone_c = stream.gone(), row_c = stream.there();
      // m = scale (u.x_c - u.x_r), and the gradient's sum is (sum of slopes) x_c - sum of
      // slope x_r: a rejected row is converted once and meets two multiply-adds an element.
      float dot_c = 0.f;
      {
        Pair dot = both(0.f), dot2 = both(0.f);
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          xc[j] = zero8<__half>();
          if (row_c) xc[j] = staged<CPL>(stream.row(), a.d_pad, lane, j);
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            dot = pair_fma(u[j][i], pair_at(xc[j], i), dot);
            dot2 = pair_fma(u[j][i + 1], pair_at(xc[j], i + 1), dot2);
          }
        }
        dot_c = warp_sum(pair_total(pair_add(dot, dot2)));
      }
      stream.next();
      float kept = 0.f;  // lane k holds the margin of row k of the last 32 ...
      bool counts = false;  // ... and whether its pair is there
      for (int k = 0; k < mine; ++k) {
        const bool gone = gone_c || stream.gone();
        const bool row = row_c && stream.there();
        any |= !gone;
        float m = gone ? 0.f : __int_as_float(0x7fffffff);
        if (row && !gone) {
          Pair x[CPL][4];
          Pair dot = both(0.f), dot2 = both(0.f);
#pragma unroll
          for (int j = 0; j < CPL; ++j) {
            const Raw8<__half> r = staged<CPL>(stream.row(), a.d_pad, lane, j);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              x[j][i] = pair_at(r, i);
              x[j][i + 1] = pair_at(r, i + 1);
              dot = pair_fma(u[j][i], x[j][i], dot);
              dot2 = pair_fma(u[j][i + 1], x[j][i + 1], dot2);
            }
          }
          m = a.scale * (dot_c - warp_sum(pair_total(pair_add(dot, dot2))));
          if (a.grad != nullptr) {
            // sigmoid(-m) from e^-|m| (exponential 2 ulp, reciprocal 1). The exponent is |m| / ln 2
            // to more than fp32's digits: p, and what p misses as a factor 1 + rest ln 2 -- the
            // rounding of p alone would cost a confident pair's slope |m| / 2 ulp.
            const float p = -kLog2E * fabsf(m);
            const float rest = fmaf(-kLog2E, fabsf(m), -p) - kLog2ELow * fabsf(m);
            const float e0 = exp2_approx(p);
            const float e = e0 == 0.f ? 0.f : fmaf(e0, rest * kLn2, e0);  // (an infinite margin: rest is NaN)
            const float below = (m > 0.f ? e : 1.f) * rcp_approx(1.f + e);
            const float slope = (a.smoothing - below) * a.scale;
            slopes += slope;
            const Pair less = both(-slope);
#pragma unroll
            for (int j = 0; j < CPL; ++j) {
#pragma unroll
              for (int i = 0; i < 4; ++i) g[j][i] = pair_fma(less, x[j][i], g[j][i]);
            }
          }
        } else if (!gone) {
          slopes = m;  // NaN, for every column below
        }
        stream.next();
        if (lane == (k & 31)) {
          kept = m;
          counts = !gone;
        }
        if ((k & 31) == 31 || k + 1 == mine) {
          // 32 margins, one per lane: their losses and the margins themselves.
          const int r = (k & ~31) + lane;
          if (r <= k) {
            if (counts) {
              loss += (1.f - a.smoothing) * softplus_of(-kept) + a.smoothing * softplus_of(kept);
              count += 1.f;
            }
            a.margins[q * a.r + static_cast<long long>(r) * wpq + share] = kept;
          }
        }
      }
    }
    if (a.grad == nullptr) continue;
    if (any) {  // else zeros
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) g[j][i] = pair_fma(both(slopes), pair_at(xc[j], i), g[j][i]);
      }
    }
    if (wpq > 1) {
      if (lane == 0) present[warp] = any;
      if (live && share != 0) {
        float4* out = reinterpret_cast<float4*>(shares + static_cast<size_t>(warp) * a.d_pad);
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
          const int col = (lane + 32 * j) * 8;
          if (col < a.d_pad) {
            float4 lo, hi;
            split(g[j][0], lo.x, lo.y);
            split(g[j][1], lo.z, lo.w);
            split(g[j][2], hi.x, hi.y);
            split(g[j][3], hi.z, hi.w);
            out[col / 4] = lo;
            out[col / 4 + 1] = hi;
          }
        }
      }
      __syncthreads();
      if (live && share == 0) {
        for (int w = 1; w < wpq; ++w) {
          any |= present[warp + w] != 0;
          const float4* in = reinterpret_cast<const float4*>(shares + static_cast<size_t>(warp + w) * a.d_pad);
#pragma unroll
          for (int j = 0; j < CPL; ++j) {
            const int col = (lane + 32 * j) * 8;
            if (col < a.d_pad) {
              const float4 lo = in[col / 4], hi = in[col / 4 + 1];
              g[j][0] = pair_add(g[j][0], pair_of(lo.x, lo.y));
              g[j][1] = pair_add(g[j][1], pair_of(lo.z, lo.w));
              g[j][2] = pair_add(g[j][2], pair_of(hi.x, hi.y));
              g[j][3] = pair_add(g[j][3], pair_of(hi.z, hi.w));
            }
          }
        }
      }
      __syncthreads();  // the shares are read before the next round writes them
    }
    if (!live || share != 0) continue;
    if (a.cosine && any) {
      Pair u[CPL][4];
      load_pairs<CPL>(a.q, a.q_dtype, q * a.q_stride, a.d, a.q_vec, lane, u);
      Pair dot = both(0.f);
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u[j][i] = pair_mul(u[j][i], both(unit.inv));
          dot = pair_fma(u[j][i], g[j][i], dot);
        }
      }
      const float along_all = warp_sum(pair_total(dot));
      const float along = unit.clamped ? 0.f : along_all;  // below the clamp the divisor is a constant
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) g[j][i] = pair_mul(pair_fma(u[j][i], both(-along), g[j][i]), both(unit.inv));
      }
    }
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      const int c0 = (lane + 32 * j) * 8;
      if (c0 + 8 <= a.grad_stride) {
        Raw8<float> out;
#pragma unroll
        for (int i = 0; i < 4; ++i) set_pair(out, i, g[j][i]);
        store8(a.grad + q * a.grad_stride + c0, out);
      }
    }
  }
  loss = warp_sum(loss);
  count = warp_sum(count);
  if (lane == 0) totals[warp] = make_float2(loss, count);
  stream.drain();
  __syncthreads();
  if (threadIdx.x == 0) {
    float2 s = make_float2(0.f, 0.f);
    for (int w = 0; w < kPrefWarps; ++w) {
      s.x += totals[w].x;
      s.y += totals[w].y;
    }
    a.partial[blockIdx.x] = s;
  }
}

// loss = (sum of the blocks' losses) * weight, weight = 1 / max(pairs, 1) (mean) or 1 (sum).
__global__ void __launch_bounds__(256) preference_finish_kernel(const float2* partial, int blocks, int mean,
                                                                float* loss, float* weight) {
  __shared__ float2 sums[256];
  grid_dependency_wait();
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
  grid_dependency_wait();
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

// Shared memory of a block: two blocks an SM up to 1024 columns, one block beyond.
constexpr int pref_shared(int cpl) { return cpl <= 4 ? 108 * 1024 : 216 * 1024; }

// Rows of a stage.
int pref_stage_rows(int d_pad, int cpl, size_t shares) {
  const size_t per = static_cast<size_t>(2 * kPrefWarps) * d_pad * 2;
  return static_cast<int>(std::max<size_t>(1, std::min<size_t>(kPrefStageRows, (pref_shared(cpl) - shares) / per)));
}

template <int CPL>
cudaError_t pref_launch_one(const PreferenceArgs& a, unsigned grid, size_t smem, cudaStream_t stream) {
  static std::atomic<unsigned long long> allowed{0};
  const cudaError_t e = allow_smem(preference_kernel<CPL>, pref_shared(CPL), allowed);
  if (e != cudaSuccess) return e;
  return launch_programmatic(preference_kernel<CPL>, dim3(grid), dim3(kPrefThreads), smem, stream, a);
}

}  // namespace

int preference_blocks(long long b, int r, int num_sms) {
  const int qpb = kPrefWarps / pref_warps(b, r, num_sms);
  return static_cast<int>(std::min<long long>((b + qpb - 1) / qpb, 2LL * num_sms));
}

cudaError_t preference_launch(PreferenceArgs a, int mean, float* loss, float* weight, int num_sms, cudaStream_t stream) {
  a.warps_per_query = pref_warps(a.b, a.r, num_sms);
  const unsigned grid = static_cast<unsigned>(preference_blocks(a.b, a.r, num_sms));
  const size_t shares = a.grad && a.warps_per_query > 1 ? static_cast<size_t>(kPrefWarps) * a.d_pad * 4 : 0;
  const int cpl = (a.d_pad / 8 + 31) / 32;
  a.stage_rows = pref_stage_rows(a.d_pad, cpl, shares);
  const size_t smem = static_cast<size_t>(2 * kPrefWarps) * a.stage_rows * a.d_pad * 2 + shares;
  cudaError_t e;
  if (a.b == 0) {
    e = cudaSuccess;
  } else {
    switch (cpl) {
      case 1: e = pref_launch_one<1>(a, grid, smem, stream); break;
      case 2: e = pref_launch_one<2>(a, grid, smem, stream); break;
      case 3: e = pref_launch_one<3>(a, grid, smem, stream); break;
      case 4: e = pref_launch_one<4>(a, grid, smem, stream); break;
      case 5: e = pref_launch_one<5>(a, grid, smem, stream); break;
      case 6: e = pref_launch_one<6>(a, grid, smem, stream); break;
      case 7: e = pref_launch_one<7>(a, grid, smem, stream); break;
      case 8: e = pref_launch_one<8>(a, grid, smem, stream); break;
      default: return cudaErrorInvalidValue;
    }
  }
  if (e != cudaSuccess) return e;
  return launch_programmatic(preference_finish_kernel, dim3(1), dim3(256), 0, stream, static_cast<const float2*>(a.partial),
                             static_cast<int>(grid), mean, loss, weight);
}

cudaError_t preference_grad_launch(const float* grad, long long grad_stride, long long b, int d, const float* weight,
                                   const float* upstream, int q_dtype, void* dq, int num_sms, cudaStream_t stream) {
  const long long items = b * (grad_stride / 8);
  const dim3 grid(static_cast<unsigned>(std::max<long long>(1, std::min<long long>((items + 255) / 256, 8LL * num_sms))));
  switch (q_dtype) {
    case kSrcF32:
      return launch_programmatic(preference_grad_kernel<float>, grid, dim3(256), 0, stream, grad, grad_stride, b, d, weight,
                                 upstream, static_cast<float*>(dq));
    case kSrcF16:
      return launch_programmatic(preference_grad_kernel<__half>, grid, dim3(256), 0, stream, grad, grad_stride, b, d, weight,
                                 upstream, static_cast<__half*>(dq));
    case kSrcBF16:
      return launch_programmatic(preference_grad_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, grad, grad_stride, b, d,
                                 weight, upstream, static_cast<__nv_bfloat16*>(dq));
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace cvs
