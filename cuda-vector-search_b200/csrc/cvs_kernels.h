// Launch-side declarations shared by the kernel translation units and the
// C-ABI host code (cvs_capi.cu). Nothing here is part of the public ABI; the
// public entry points are declared in include/cvs.h.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <atomic>
#include <cstddef>
#include <cstdint>

namespace cvs {

// ---- tcgen05 fused score + top-k / score-store kernel ----------------------
constexpr int kTcM = 128;          // queries per tile (MMA M; TMEM lanes)
constexpr int kTcN = 256;          // corpus rows per tile (MMA N; TMEM columns)
constexpr int kTcK = 64;           // halves per K slice (one 128-byte swizzled row)
// Ring stages of the tcgen05 kernels: as many as the shared memory left after
// the resident queries, barriers, iteration log and (buffer epilogues) radix
// histograms and compaction buffers holds, at most this many (the barrier
// arrays are sized for it).
constexpr int kTcMaxStages = 8;
constexpr int kSmemLimit = 232448;          // dynamic shared memory per CTA
constexpr int kSmemBudget = kSmemLimit - 1024;  // less the alignment slack
constexpr int kTcMaxResidentSlices = 7;  // queries stay in smem when d_pad <= 448
// Dry tiles of the top-k epilogues (see cvs_epilogue.cuh): at most this many
// (TileSource in cvs_sched.cuh keeps two).
constexpr int kDryTiles = 2;

enum TcEpilogue : int {
  kEpiTopkReg16 = 0,   // k <= 16: per-query sorted list in registers
  kEpiTopkReg32 = 1,   // k <= 32
  kEpiTopkBuf = 2,     // k  > 32: per-query candidate buffer in global memory
  kEpiStoreF32 = 3,    // write the score matrix as fp32
  kEpiStoreF16 = 4,    // write the score matrix as fp16
  kEpiTopkBuf8 = 5,    // k > 32 with fewer lists: candidate buffers, 8 ranks tracked in registers
};

// Rank J of the per-list value a buffer list (k > 32) publishes (its J-th best)
// and how many lists m must reach a value for it to bound the query's k-th best
// (m lists x J rows >= k rows). Aim: J = ceil(2k / lists), so m is about half
// the lists; but J is held to regj (the ranks the epilogue tracks in registers,
// which is what lets it publish from the first tile on) whenever m = ceil(k / J)
// still fits in the lists. The merge uses the same pair.
__host__ __device__ inline int tops_j(int k, int lists, int regj) {
  lists = lists < 1 ? 1 : lists;
  int j = (2 * k + lists - 1) / lists;
  const int jmin = (k + lists - 1) / lists;  // smallest J with m <= lists
  if (j > regj) j = jmin > regj ? jmin : regj;
  return j < 1 ? 1 : (j > k ? k : j);
}
__host__ __device__ inline int tops_m(int k, int lists, int regj) {
  const int j = tops_j(k, lists, regj);
  return (k + j - 1) / j;
}

// Ranks a buffer epilogue tracks in registers (kEpiTopkBuf: 4, kEpiTopkBuf8: 8;
// more ranks cost registers in the drain loop, so 8 only where 4 cannot serve).
__host__ __device__ inline int buf_reg_ranks(int epi) { return epi == kEpiTopkBuf8 ? 8 : 4; }
__host__ __device__ inline bool is_buf_epi(int epi) { return epi == kEpiTopkBuf || epi == kEpiTopkBuf8; }


struct TcArgs {
  int b;              // queries
  int n;              // corpus rows
  int d_pad;          // row width in halves (multiple of 64)
  int ksl;            // d_pad / 64
  int qtiles;         // ceil(b / 128)
  int segs;           // corpus segments (each a contiguous run of 256-row tiles)
  int tiles_per_seg;
  int ntiles;         // ceil(n / 256)
  int k;              // candidates kept per (query, segment)
  int cap;            // slots per candidate list; cap >= k
  uint64_t* part;     // [b][segs * lists per segment][cap] ordered keys
  uint32_t* gthr;     // [b] shared per-query lower bounds (ordered bits), zeroed per call
  uint32_t* tops;     // [b][segs * lists per segment] each list's published score (ordered bits), zeroed per call
  int* counts;        // [b][segs * lists per segment] keys each buffer list ends with (buffer epilogue)
  int* tile_counter;  // [qtiles] next unclaimed corpus tile per query tile, zeroed per call;
                      // null: CTA s works on the fixed tiles [s*tiles_per_seg, (s+1)*tiles_per_seg)
  int dry;            // tiles each CTA reads dry first (0 or kDryTiles)
  void* scores_out;   // [b][n] fp32/fp16 for the store epilogues
  int* err;           // device error word
  // Failure-path test hook (one-CTA kernel only; cvs_debug_stall_next_search):
  // stall != 0 makes the producer claim and load nothing, and wait_cycles > 0
  // replaces the ~1 s limit of the kernel's waits, so every wait runs out.
  long long wait_cycles;
  int stall;
};

// Candidate lists each (query, segment) produces with this epilogue (one per
// epilogue column stripe); the workspace holds b * segs * lists * cap keys.
int tc_lists_per_segment(int epi);
// Whether the query tile can stay resident in shared memory next to the stage
// ring and this epilogue's scratch (one-CTA kernel).
bool tc_resident_queries(int epi, int ksl);
cudaError_t tc_launch(int epi, bool resident_queries, const CUtensorMap* qmap,
                      const CUtensorMap* xmap, const TcArgs& a, cudaStream_t stream);

// CTA-pair variant (batches > 128): a.qtiles counts 256-query pair tiles, the
// corpus tensor map uses 128-row boxes, the grid is 2 * qtiles * segs CTAs.
bool tc_pair_resident_queries(int epi, int ksl);
int tc_pair_max_clusters(int epi, bool resident_queries, int ksl);
cudaError_t tc_pair_launch(int epi, bool resident_queries, const CUtensorMap* qmap,
                           const CUtensorMap* xmap, const TcArgs& a, cudaStream_t stream);

// ---- CUDA-core GEMV + top-k for one to eight queries -----------------------
constexpr int kGemvThreads = 256;
constexpr int kGemvMaxK = 32;
constexpr int kGemvMaxBatch = 8;  // queries per GEMV launch (small corpora only from 2 on)

struct GemvArgs {
  const __half* x;    // [n][d_pad]
  const __half* q;    // [b][d_pad]
  int b;
  int n;
  int d_pad;
  int k;
  int segs;           // grid size; segment s covers rows [s*rows_per_seg, ...)
  int rows_per_seg;
  uint64_t* part;     // [b][segs][k]
  uint32_t* bounds;   // [b] per-query lower bounds on the k-th best (ordered bits), zeroed per call
  uint32_t* tops;     // [b][segs] each CTA's best score (ordered bits)
  int* err;
};

bool gemv_supported(int b, int k, int d_pad);
cudaError_t gemv_launch(const GemvArgs& a, cudaStream_t stream);
int gemv_blocks_per_sm(int b, int d_pad);

// ---- merge of per-segment candidate lists into the final sorted top-k ------
struct MergeKeysArgs {
  const uint64_t* part;  // [b][lists][stride], first per_list entries of each used
  const int* counts;     // [b][lists] entries used per list (then per_list is ignored) or null
  int b;
  int lists;
  int stride;
  int per_list;
  int k;
  long long id_offset;   // added to every returned row id
  const uint32_t* bounds;  // [b] lower bounds on each query's k-th best (ordered bits) or null
  const uint32_t* tops;    // [b][tops_n] per-list published scores (ordered bits, 0 = none) or null
  int tops_n;
  int tops_m;              // the tops_m-th largest published score bounds the k-th best
  float* out_v;          // [b][k]
  long long* out_i;      // [b][k]
  int* err;
};
cudaError_t merge_keys_launch(const MergeKeysArgs& a, cudaStream_t stream);

// Zeroes `bytes` bytes at p (4-byte aligned); if q_dst is given, also copies the
// b x d_pad fp16 queries q_src into q_dst and zeroes its rows b..rows_pad-1. Lets
// the next kernel, launched programmatically, start its prologue meanwhile.
cudaError_t prepare_launch(void* p, size_t bytes, const void* q_src, void* q_dst, int b, int d_pad,
                           int rows_pad, cudaStream_t stream);

// Launches `kernel` with programmatic stream serialisation: it may start while
// the previous kernel on the stream finishes and must call
// grid_dependency_wait() before touching that kernel's results.
template <class... Params, class... Args>
cudaError_t launch_programmatic(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem,
                                cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Args&&>(args)...);
}

// Sets a kernel's dynamic shared memory limit, once per device. The limit belongs to the
// kernel, not to a launch, so `smem` is the most that any call of it asks for: one that
// followed the call's own size could be lowered by another thread before the launch.
template <class K>
cudaError_t allow_smem(K kern, int smem, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

struct MergeListsArgs {
  const float* v;        // [lists] x [b][len] scores, lists v_stride floats apart
  const long long* ids;  // [lists] x [b][len] ids (must lie in [0, 2^31)), lists i_stride apart
  long long v_stride;
  long long i_stride;
  int b;
  int lists;
  int len;
  int k;
  float* out_v;          // [b][k]
  long long* out_i;      // [b][k]
  int* err;
};
cudaError_t merge_lists_launch(const MergeListsArgs& a, cudaStream_t stream);

// ---- ingest: dtype conversion, optional L2 normalisation, width padding ----
enum SrcDtype : int { kSrcF32 = 0, kSrcF16 = 1, kSrcBF16 = 2, kSrcF64 = 3 };
// With `clear` given, the same launch also zeroes clear_words 32-bit words there,
// and rows n .. rows_pad-1 of dst are written as zeros (a search's workspace
// preparation folded into its query ingest).
cudaError_t ingest_launch(const void* src, int src_dtype, long long n, int d, long long src_stride,
                          int d_pad, int cosine, __half* dst, int num_sms, cudaStream_t stream,
                          uint32_t* clear = nullptr, size_t clear_words = 0, long long rows_pad = 0);

// ---- layer norm -------------------------------------------------------------
constexpr int kNormMaxWidth = 8192;

struct NormArgs {
  const void* x;       // [rows][d], rows x_stride elements apart
  const void* weight;  // [d] or null (ones); fp32 if w32, else the rows' type
  const void* bias;    // [d] or null (zeros), same type as weight
  int w32;
  long long rows;
  int d;
  long long x_stride;
  float eps;
  void* y;             // forward result
  long long y_stride;
  float* mean;         // [rows]: forward writes them (or null), backward reads them
  float* rstd;
  const void* dy;      // backward only
  long long dy_stride;
  void* dx;            // null: not wanted
  long long dx_stride;
  void* dweight;       // null: not wanted
  void* dbias;
  float* partial;      // [blocks][2][d] or null when neither dweight nor dbias is wanted
  int* err;            // device error word (the rings' waits are bounded)
  int slots;           // set by norm_launch: row pairs in a warp's ring
  // Failure-path test hook (kernels with a ring; cvs_debug_stall_next_norm): stall != 0
  // copies no row, and wait_cycles > 0 replaces the waits' usual limit.
  int stall;
  long long wait_cycles;
};
// Blocks of the backward kernel, each with its own row of `partial`.
int norm_backward_blocks(long long rows, int d, int num_sms);
cudaError_t norm_launch(const NormArgs& a, int dtype, bool backward, int num_sms, cudaStream_t stream);

// ---- linear layer -------------------------------------------------------------
enum Activation : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3 };
constexpr int kLinearSmallRows = 8;  // rows of any alignment up to which CUDA cores stream the weights

// One product out[m][n] = A B^T over kblocks slices of 64 along K, cut into
// `splits` parts of kper slices. All pointers hold halves of the call's type
// except z (fp16) and partial (fp32).
struct GemmProblem {
  int work;              // work items: tiles_m * tiles_n * splits (0: no such product)
  int tiles_m, tiles_n;
  int splits, kblocks, kper;
  int m, n;
  int a_mn, b_mn;        // operand stored with K as its outer dimension
  void* out;
  long long ld_out;
  const void* bias;      // [n] or null
  const void* residual;  // [m][n] or null
  long long ld_res;
  void* z;               // pre-activation, fp16, rows 16-byte aligned, or null
  long long ld_z;
  int vec_out, vec_res;  // rows the tensor-memory accelerator can address
  float* partial;        // splits > 1: fp32 parts instead of all of the above
};
// Only p[0] may have a residual or z.
struct GemmArgs {
  GemmProblem p[2];
  int act;               // of p[0]; kActNone where there are two
  int bf16;
  int* err;
};
// Tensor maps: both products' operands (boxes as the tile shape needs them) and, in
// boxes of 64 columns x 32 rows, what the epilogue moves: results (where vec_out),
// z and the residual (where vec_res).
struct GemmMaps {
  CUtensorMap a[2], b[2], out[2], z, residual;
};
// Tile shapes: cg CTAs (128 rows each) x bn columns. One translation unit per activation.
cudaError_t gemm_launch_none(int cg, int bn, const GemmMaps& maps, const GemmArgs& a, int ctas, cudaStream_t stream);
cudaError_t gemm_launch_relu(int cg, int bn, const GemmMaps& maps, const GemmArgs& a, int ctas, cudaStream_t stream);
cudaError_t gemm_launch_gelu(int cg, int bn, const GemmMaps& maps, const GemmArgs& a, int ctas, cudaStream_t stream);
cudaError_t gemm_launch_silu(int cg, int bn, const GemmMaps& maps, const GemmArgs& a, int ctas, cudaStream_t stream);
cudaError_t gemm_launch(int cg, int bn, const GemmMaps& maps, const GemmArgs& a, int ctas, cudaStream_t stream);

// One product of few 128 x 64 tiles, its K slices shared by the 2, 4 or 8 CTAs of a
// cluster. amap: boxes of 64 columns x a_rows rows, bmap: 64 x 64.
struct SplitArgs {
  int m, n;
  int tiles_m;
  int kblocks, kper;     // slices of 64 along K, per CTA
  int a_rows;
  int act, bf16;
  const void* bias;
  const void* residual;
  void* out;
  void* z;
  long long ld_res, ld_out, ld_z;
  int vec_res, vec_out;  // rows 16-byte aligned
  int* err;
};
cudaError_t split_launch(int splits, const CUtensorMap& amap, const CUtensorMap& bmap, const SplitArgs& a, int tiles,
                         cudaStream_t stream);

struct LinearSmallArgs {
  const void* x;
  const void* w;
  const void* bias;
  const void* residual;
  void* out;
  void* z;
  long long ld_x, ld_w, ld_res, ld_out, ld_z;
  int m, n, k;
  int act, bf16;
  int vec;  // x and w rows 16-byte aligned and k a multiple of 8
};
cudaError_t linear_small_launch(const LinearSmallArgs& a, cudaStream_t stream);

cudaError_t pad_rows_launch(const void* src, long long rows, int cols, long long ld_src, void* dst, long long ld_dst,
                            int num_sms, cudaStream_t stream);

struct LinearDzArgs {
  const void* dy;
  const void* z;     // null: no activation
  void* dz;          // null: dy is used as it is
  float* partial;    // [parts][n] column sums, or null
  long long ld_dy, ld_z, ld_dz;
  long long m;
  int n;
  int act, bf16, vec_dy;
};
int linear_dz_parts(long long m, int n, int num_sms);
cudaError_t linear_dz_launch(const LinearDzArgs& a, int parts, cudaStream_t stream);

struct LinearFinishArgs {
  const float* db_partial;
  int db_parts, db_blocks;  // db_blocks: ceil(n / 32), 0 when dbias is not wanted
  void* dbias;
  const float* dw_partial;  // null when dw was written by the product itself
  int splits, tiles_m, tiles_n, cg, bn;
  void* dw;
  long long ld_dw;
  int vec_dw;               // rows 16-byte aligned
  int n, k;                 // dw is [n][k]
  int bf16;
};
cudaError_t linear_finish_launch(const LinearFinishArgs& a, cudaStream_t stream);

// ---- preference loss ------------------------------------------------------------
struct PreferenceArgs {
  const void* q;            // [b][d]
  const void* ref;          // [b][d] or null
  int q_dtype, ref_dtype;
  long long q_stride, ref_stride;
  int q_vec, ref_vec;       // rows 16-byte aligned and d a multiple of 8
  int cosine;
  const __half* x;          // [n][d_pad]
  long long n;
  int d, d_pad;
  const long long* chosen;  // [b]
  const long long* rejected;  // [b][r], rows rejected_stride apart
  long long rejected_stride;
  long long b;
  int r;
  float scale, smoothing;
  float* margins;           // [b][r]
  float* grad;              // [b][grad_stride] sums of the loss's gradient, or null
  long long grad_stride;    // d rounded up to a multiple of 8
  float2* partial;          // [blocks] (loss, pairs)
  int* err;
  int warps_per_query;      // set by preference_launch, as is
  int stage_rows;           // row buffers of each of a warp's two stages
};
int preference_blocks(long long b, int r, int num_sms);
cudaError_t preference_launch(PreferenceArgs a, int mean, float* loss, float* weight, int num_sms, cudaStream_t stream);
cudaError_t preference_grad_launch(const float* grad, long long grad_stride, long long b, int d, const float* weight,
                                   const float* upstream, int q_dtype, void* dq, int num_sms, cudaStream_t stream);

}  // namespace cvs
