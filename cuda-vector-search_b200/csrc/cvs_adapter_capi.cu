// Host side of the adapter operators' C ABI (include/cvs.h): argument contracts,
// tile plans and tensor maps of the linear layer's products, kernel launches.
#include <algorithm>
#include <climits>
#include <cstdint>

#include "cvs.h"
#include "cvs_host.h"
#include "cvs_kernels.h"

namespace cvs {
namespace {

static_assert(CVS_MAX_NORM_WIDTH == kNormMaxWidth, "public limit");
static_assert(CVS_LINEAR_SMALL_ROWS == kLinearSmallRows, "public limit");

constexpr size_t kAlign = 256;
size_t up(size_t v) { return (v + kAlign - 1) / kAlign * kAlign; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool float_type(int t) { return t == CVS_F32 || t == CVS_F16 || t == CVS_BF16; }

cvs_status check_workspace(const void* ws, size_t have, size_t need) {
  if (need == 0) return CVS_OK;
  if (!ws || have < need || (reinterpret_cast<uintptr_t>(ws) % kAlign) != 0)
    return fail(CVS_ERR_WORKSPACE, "workspace of %zu bytes (256-byte aligned) required, got %zu at %p", need, have, ws);
  return CVS_OK;
}

// ---- layer norm -----------------------------------------------------------------
thread_local int64_t g_norm_stall = 0;  // armed failure-path test (cvs_debug_stall_next_norm)

// Launches, with the device error word that the kernels' bounded waits report to.
cvs_status run_norm(NormArgs& a, int dtype, bool backward, const DeviceInfo& dev, cudaStream_t s) {
  a.err = dev.err;
  a.wait_cycles = g_norm_stall;
  a.stall = g_norm_stall > 0;
  g_norm_stall = 0;  // one call only
  const cudaError_t e = norm_launch(a, dtype, backward, dev.sms, s);
  if (a.stall && e == cudaErrorNotSupported)
    return fail(CVS_ERR_INVALID_ARGUMENT, "the stall test hook needs aligned rows of up to 1024 columns (forward: halves, more than 2^22 of them)");
  return e == cudaSuccess ? CVS_OK : cuda_fail(e, backward ? "layer norm backward launch" : "layer norm launch");
}

cvs_status check_norm(int dtype, int64_t rows, int d, int64_t x_stride, int weight_dtype) {
  if (rows < 0) return fail(CVS_ERR_INVALID_ARGUMENT, "row count must be >= 0");
  if (d < 1 || d > CVS_MAX_NORM_WIDTH)
    return fail(CVS_ERR_INVALID_ARGUMENT, "layer norm width must be in 1 .. %d (got %d)", CVS_MAX_NORM_WIDTH, d);
  if (!float_type(dtype)) return fail(CVS_ERR_INVALID_ARGUMENT, "unsupported dtype %d", dtype);
  if (weight_dtype != dtype && weight_dtype != CVS_F32)
    return fail(CVS_ERR_INVALID_ARGUMENT, "weight dtype must be the rows' dtype or float32");
  if (rows > 1 && x_stride < 0) return fail(CVS_ERR_INVALID_ARGUMENT, "negative row stride");
  return CVS_OK;
}

// ---- linear ---------------------------------------------------------------------
cvs_status check_linear(int activation, int dtype, int64_t m, int n, int k) {
  if (m < 0 || m >= INT_MAX) return fail(CVS_ERR_INVALID_ARGUMENT, "row count %lld out of range", (long long)m);
  if (n < 1 || k < 1 || n > CVS_MAX_LAYER_WIDTH || k > CVS_MAX_LAYER_WIDTH)
    return fail(CVS_ERR_INVALID_ARGUMENT, "layer widths must be in 1 .. 2^24 (got %d x %d)", n, k);
  if (activation < CVS_ACT_NONE || activation > CVS_ACT_SILU)
    return fail(CVS_ERR_INVALID_ARGUMENT, "unknown activation %d", activation);
  if (dtype != CVS_F16 && dtype != CVS_BF16)
    return fail(CVS_ERR_INVALID_ARGUMENT, "linear takes float16 or bfloat16 (got dtype %d)", dtype);
  return CVS_OK;
}

cvs_status check_operand(const void* p, int64_t stride, int64_t width, const char* name) {
  if (!p || !aligned16(p) || stride % 8 != 0 || stride < width)
    return fail(CVS_ERR_INVALID_ARGUMENT, "%s must be non-null and 16-byte aligned with a row stride that is a multiple of 8 and "
                "at least its width", name);
  return CVS_OK;
}

// A product's operand: stored [mn][k] (K-major) or [k][mn] (MN-major).
struct Operand {
  const void* p;
  int64_t stride;
  bool mn_major;
};

cvs_status operand_map(CUtensorMap* map, const Operand& o, int dtype, int64_t mn, int64_t k, int box_mn) {
  return o.mn_major ? make_half_map(map, o.p, dtype, k, mn, o.stride, 64)
                    : make_half_map(map, o.p, dtype, mn, k, o.stride, box_mn);
}

// Rows a tensor map can describe, and the map of what the epilogue moves. A store writes
// whole 16-byte units (zeros behind the width), so only whole rows of them are stored
// through a map; loads read zeros behind the width.
bool mappable(const void* p, int64_t stride, int64_t width) {
  return p && aligned16(p) && stride % 8 == 0 && stride >= width;
}
bool storable(const void* p, int64_t stride, int64_t width) { return mappable(p, stride, width) && width % 8 == 0; }
cvs_status block_map(CUtensorMap* map, const void* p, int dtype, int64_t rows, int64_t cols, int64_t stride) {
  return make_half_map(map, p, dtype, rows, cols, stride, 32);
}

struct Tile {
  int cg, bn;
  int slots(int sms) const { return sms / cg; }
};
constexpr Tile kTiles[3] = {{2, 256}, {1, 128}, {1, 64}};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Time of one round of work items, in units of half the smallest tile's: larger tiles keep the
// tensor cores busier per byte of shared memory read. Measured (us, tiles of 256 x 256 by a CTA
// pair / 128 x 128 / 128 x 64, K = 768, rounds in brackets): 18944 x 128 10.8 [1] / 8.4 [1] /
// 10.1 [2]; 18944 x 256 12.0 [1] / 12.4 [2] / 16.0 [4]; 4096 x 768 10.4 [1] / 11.2 [2] / 13.7
// [3]; 16384 x 768 23.5 [3] / 30.3 [6] / 42.1 [11]; 131072 x 768 131 [21] / 221 [42] / 349
// [84]: 6.2 : 4.2-5.3 : 3.4-4.2 us a round in the larger ones.
double tile_cost(const Tile& t) { return t.cg == 2 ? 4.0 : (t.bn == 128 ? 2.7 : 2.0); }

// The tile shape whose rounds of work items over the SMs take least: large tiles
// for large products, small ones where large ones would leave SMs idle.
Tile pick_tile(int64_t m, int64_t n, int sms) {
  Tile best = kTiles[0];
  double best_time = 0;
  for (const Tile& t : kTiles) {
    const int64_t tiles = ceil_div(m, 128 * t.cg) * ceil_div(n, t.bn);
    const double time = static_cast<double>(ceil_div(tiles, t.slots(sms))) * tile_cost(t);
    if (best_time == 0 || time < best_time) {
      best = t;
      best_time = time;
    }
  }
  return best;
}

// CTAs that share a 128 x 64 tile's K dimension (0: the persistent kernel). Eight as long
// as one round of SMs holds them, four as long as two rounds do (two CTAs fit on an SM),
// two where one round does or K is long. Measured (us, persistent / 2 / 4 / 8): 64 rows,
// 768 -> 1536 (24 tiles): 7.7 / 6.6 / 5.2 / 5.7; 16 rows, 1536 -> 768 (12): 10.2 / 7.5 /
// 5.5 / 4.8; 32 rows, 4096 -> 4096 (64): 19.4 / 12.5 / 9.9 / 15.1; 512 rows, 768 -> 1536
// (96): 8.5 / 9.0 / 12.2 / 17.3; 256 rows, 4096 -> 4096 (128): 20.9 / 16.9 / 21.7 / 31.7.
int pick_splits(int64_t m, int64_t n, int64_t k, int sms) {
  const int64_t tiles = ceil_div(m, 128) * ceil_div(n, 64), kblocks = ceil_div(k, 64);
  if (8 * tiles <= sms && kblocks >= 6) return 8;
  if (4 * tiles <= 2 * sms && kblocks >= 4) return 4;
  if (2 * tiles <= (kblocks >= 32 ? 2 * sms : sms) && kblocks >= 2) return 2;
  return 0;
}

void set_shape(GemmProblem* p, const Tile& t, int64_t m, int64_t n, int64_t k, int splits) {
  p->m = static_cast<int>(m);
  p->n = static_cast<int>(n);
  p->tiles_m = static_cast<int>(ceil_div(m, 128 * t.cg));
  p->tiles_n = static_cast<int>(ceil_div(n, t.bn));
  p->kblocks = static_cast<int>(ceil_div(k, 64));
  p->kper = static_cast<int>(ceil_div(p->kblocks, splits));
  p->splits = static_cast<int>(ceil_div(p->kblocks, p->kper));
  p->work = p->tiles_m * p->tiles_n * p->splits;
}

int grid_ctas(const Tile& t, int work, int sms) { return t.cg * std::max(1, std::min(t.slots(sms), work)); }

// Backward: the tile shape, dw's parts along K (= rows), and the workspace, whose end
// holds dz (bytes_dz; not needed where the products read dy itself).
struct BackwardPlan {
  Tile tile;
  int splits;
  int db_parts;
  size_t dz_offset, db_offset, dw_offset, bytes, bytes_dz;
  int64_t dz_stride;
};

BackwardPlan plan_backward(int64_t m, int n, int k, int sms) {
  BackwardPlan b;
  // Both products run in one launch, with one tile shape, dw's work items first; item
  // i goes to CTA (pair) i mod slots. dw's K dimension (the rows) is cut into as many
  // parts as give the shortest of the longest queues, in slices of 64 along K plus one
  // an item; parts also cost the writing and reading of their fp32 sums, about three
  // slices' time a round of them.
  b.tile = pick_tile(std::max<int64_t>(m, n), k, sms);
  const int slots = b.tile.slots(sms);
  const int64_t tiles = ceil_div(n, 128 * b.tile.cg) * ceil_div(k, b.tile.bn);
  const int64_t dx_items = ceil_div(m, 128 * b.tile.cg) * ceil_div(k, b.tile.bn);
  const int64_t dx_len = ceil_div(n, 64) + 1, kblocks = ceil_div(m, 64);
  int64_t best = 0;
  b.splits = 1;
  for (int s : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32}) {
    if (s > kblocks) break;
    const int64_t kper = ceil_div(kblocks, s), parts = ceil_div(kblocks, kper);
    const int64_t dw_items = tiles * parts, dw_len = kper + 1;
    // Queue of slot 0, and of the first slot past dw's last round, which gets one dw item less.
    const int64_t total = dw_items + dx_items;
    const auto queue = [&](int64_t slot) {
      const int64_t dw = slot < dw_items ? (dw_items - slot + slots - 1) / slots : 0;
      const int64_t all = slot < total ? (total - slot + slots - 1) / slots : 0;
      return dw * dw_len + (all - dw) * dx_len;
    };
    int64_t time = std::max(queue(0), queue(dw_items % slots));
    if (parts > 1) time += 2 + 3 * parts * tiles / slots;
    if (best == 0 || time < best) {
      best = time;
      b.splits = static_cast<int>(parts);
    }
  }
  GemmProblem p{};
  set_shape(&p, b.tile, n, k, m, b.splits);
  b.splits = p.splits;
  b.db_parts = linear_dz_parts(m, n, sms);
  b.dz_stride = (static_cast<int64_t>(n) + 7) / 8 * 8;
  size_t at = 0;
  b.db_offset = at;
  at += up(static_cast<size_t>(b.db_parts) * n * 4);
  b.dw_offset = at;
  if (b.splits > 1) at += up(static_cast<size_t>(p.work) * b.tile.cg * 128 * b.tile.bn * 4);
  b.dz_offset = at;
  b.bytes_dz = up(static_cast<size_t>(m) * b.dz_stride * 2);
  b.bytes = at + b.bytes_dz;
  return b;
}

}  // namespace
}  // namespace cvs

using namespace cvs;

extern "C" {

cvs_status cvs_layer_norm(const void* x, int dtype, int64_t rows, int d, int64_t x_stride, const void* weight,
                          const void* bias, int weight_dtype, float eps, void* y, int64_t y_stride, float* mean,
                          float* rstd, void* stream) {
  cvs_status st = check_norm(dtype, rows, d, x_stride, weight_dtype);
  if (st != CVS_OK) return st;
  if (rows == 0) return CVS_OK;
  if (!x || !y) return fail(CVS_ERR_INVALID_ARGUMENT, "null pointer");
  if (rows > 1 && y_stride < d) return fail(CVS_ERR_INVALID_ARGUMENT, "output row stride smaller than the width");
  DeviceInfo dev;
  if ((st = device_info(&dev)) != CVS_OK) return st;
  NormArgs a{};
  a.x = x;
  a.weight = weight;
  a.bias = bias;
  a.w32 = weight_dtype == CVS_F32;
  a.rows = rows;
  a.d = d;
  a.x_stride = x_stride;
  a.eps = eps;
  a.y = y;
  a.y_stride = y_stride;
  a.mean = mean;
  a.rstd = rstd;
  return run_norm(a, dtype, false, dev, static_cast<cudaStream_t>(stream));
}

cvs_status cvs_layer_norm_backward_workspace_size(int64_t rows, int d, size_t* bytes) {
  if (!bytes) return fail(CVS_ERR_INVALID_ARGUMENT, "bytes must not be null");
  *bytes = 0;
  cvs_status st = check_norm(CVS_F32, rows, d, d, CVS_F32);
  if (st != CVS_OK) return st;
  if (rows == 0) return CVS_OK;
  DeviceInfo dev;
  if ((st = device_info(&dev)) != CVS_OK) return st;
  *bytes = up(static_cast<size_t>(norm_backward_blocks(rows, d, dev.sms)) * 2 * d * 4);
  return CVS_OK;
}

cvs_status cvs_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int dtype, int64_t rows, int d,
                                   int64_t x_stride, const void* weight, int weight_dtype, const float* mean,
                                   const float* rstd, void* dx, int64_t dx_stride, void* dweight, void* dbias,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  cvs_status st = check_norm(dtype, rows, d, x_stride, weight_dtype);
  if (st != CVS_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t ws = weight_dtype == CVS_F32 ? 4 : 2;
  if (rows == 0) {  // sums over no rows
    cudaError_t e = cudaSuccess;
    if (dweight) e = cudaMemsetAsync(dweight, 0, ws * d, s);
    if (e == cudaSuccess && dbias) e = cudaMemsetAsync(dbias, 0, ws * d, s);
    return e == cudaSuccess ? CVS_OK : cuda_fail(e, "clearing the weights' gradients");
  }
  if (!dy || !x || !mean || !rstd) return fail(CVS_ERR_INVALID_ARGUMENT, "null pointer");
  if (rows > 1 && dy_stride < 0) return fail(CVS_ERR_INVALID_ARGUMENT, "negative row stride");
  if (dx && rows > 1 && dx_stride < d) return fail(CVS_ERR_INVALID_ARGUMENT, "gradient row stride smaller than the width");
  if (!dx && !dweight && !dbias) return CVS_OK;
  DeviceInfo dev;
  if ((st = device_info(&dev)) != CVS_OK) return st;
  const bool sums = dweight || dbias;
  if (sums) {
    const size_t need = up(static_cast<size_t>(norm_backward_blocks(rows, d, dev.sms)) * 2 * d * 4);
    if ((st = check_workspace(workspace, workspace_bytes, need)) != CVS_OK) return st;
  }
  NormArgs a{};
  a.x = x;
  a.weight = weight;
  a.w32 = weight_dtype == CVS_F32;
  a.rows = rows;
  a.d = d;
  a.x_stride = x_stride;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.dy = dy;
  a.dy_stride = dy_stride;
  a.dx = dx;
  a.dx_stride = dx_stride;
  a.dweight = dweight;
  a.dbias = dbias;
  a.partial = sums ? static_cast<float*>(workspace) : nullptr;
  return run_norm(a, dtype, true, dev, s);
}

cvs_status cvs_debug_stall_next_norm(int64_t wait_cycles) {
  if (wait_cycles < 1000 || wait_cycles > (int64_t{1} << 40))
    return fail(CVS_ERR_INVALID_ARGUMENT, "wait_cycles must be in 1000 .. 2^40 (got %lld)", (long long)wait_cycles);
  g_norm_stall = wait_cycles;
  return CVS_OK;
}

cvs_status cvs_align_rows(const void* src, int64_t src_stride, int dtype, int64_t rows, int cols, void* dst,
                          int64_t dst_stride, void* stream) {
  if (dtype != CVS_F16 && dtype != CVS_BF16) return fail(CVS_ERR_INVALID_ARGUMENT, "float16 or bfloat16 (got dtype %d)", dtype);
  if (rows < 0 || cols < 1) return fail(CVS_ERR_INVALID_ARGUMENT, "bad matrix shape [%lld][%d]", (long long)rows, cols);
  if (rows == 0) return CVS_OK;
  if (!src || (rows > 1 && src_stride < 0)) return fail(CVS_ERR_INVALID_ARGUMENT, "bad source");
  cvs_status st = check_operand(dst, dst_stride, cols, "dst");
  if (st != CVS_OK) return st;
  DeviceInfo dev;
  if ((st = device_info(&dev)) != CVS_OK) return st;
  const cudaError_t e = pad_rows_launch(src, rows, cols, src_stride, dst, dst_stride, dev.sms, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? CVS_OK : cuda_fail(e, "row alignment launch");
}

cvs_status cvs_linear(const void* x, int64_t x_stride, const void* w, int64_t w_stride, const void* bias,
                      const void* residual, int64_t residual_stride, int activation, int dtype, int64_t m, int n,
                      int k, void* y, int64_t y_stride, void* z, int64_t z_stride, void* stream) {
  cvs_status st = check_linear(activation, dtype, m, n, k);
  if (st != CVS_OK) return st;
  if (m == 0) return CVS_OK;
  if (!x || !w || !y) return fail(CVS_ERR_INVALID_ARGUMENT, "null pointer");
  if (m > 1 && y_stride < n) return fail(CVS_ERR_INVALID_ARGUMENT, "output row stride smaller than the width");
  if (z && (!aligned16(z) || z_stride % 8 != 0 || z_stride < n))
    return fail(CVS_ERR_INVALID_ARGUMENT, "z must be 16-byte aligned with a row stride that is a multiple of 8 and at least n");
  if (residual && m > 1 && residual_stride < 0) return fail(CVS_ERR_INVALID_ARGUMENT, "negative row stride");
  if (activation == CVS_ACT_NONE) z = nullptr;  // only an activation's derivative reads it
  DeviceInfo dev;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  // One row, and two of up to 2048 columns, the CUDA cores take fastest, streaming the weights.
  // Rows 1 / 2 / 3 on CUDA cores against any of them on the tensor cores, us: 256 -> 256 1.6 /
  // 1.9 / 2.3, 4.3; 768 -> 1536 2.1 / 3.0 / 3.8, 4.8; 1024 -> 16384 8.4 / 11.4 / 15.2, 12.6;
  // 2048 -> 2048 2.6 / 5.2 / 7.2, 6.1; 2048 -> 8192 8.8 / 10.9 / 14.9, 13.2; 4096 -> 1024 3.3 /
  // 8.6 / 12.3, 7.2; 4096 -> 4096 8.0 / 17.7 / 24.4, 12.8. Rows of any alignment stay there up
  // to kLinearSmallRows rather than have the weights copied.
  const bool tiles = mappable(x, m > 1 ? x_stride : ceil_div(k, 8) * 8, k) && mappable(w, w_stride, k);
  if (m == 1 || (m == 2 && k <= 2048) || (m <= kLinearSmallRows && !tiles)) {
    if ((m > 1 && x_stride < 0) || w_stride < k)
      return fail(CVS_ERR_INVALID_ARGUMENT, "bad row stride");
    if ((st = device_info(&dev)) != CVS_OK) return st;
    LinearSmallArgs a{};
    a.x = x;
    a.w = w;
    a.bias = bias;
    a.residual = residual;
    a.out = y;
    a.z = z;
    a.ld_x = x_stride;
    a.ld_w = w_stride;
    a.ld_res = residual_stride;
    a.ld_out = y_stride;
    a.ld_z = z_stride;
    a.m = static_cast<int>(m);
    a.n = n;
    a.k = k;
    a.act = activation;
    a.bf16 = dtype == CVS_BF16;
    a.vec = aligned16(x) && aligned16(w) && x_stride % 8 == 0 && w_stride % 8 == 0 && k % 8 == 0;
    if ((e = linear_small_launch(a, s)) != cudaSuccess) return cuda_fail(e, "linear launch");
    return CVS_OK;
  }
  if ((st = check_operand(x, x_stride, k, "x")) != CVS_OK) return st;
  if ((st = check_operand(w, w_stride, k, "w")) != CVS_OK) return st;
  if ((st = device_info(&dev)) != CVS_OK) return st;
  if (const int splits = pick_splits(m, n, k, dev.sms)) {
    SplitArgs a{};
    a.m = static_cast<int>(m);
    a.n = n;
    a.tiles_m = static_cast<int>(ceil_div(m, 128));
    a.kblocks = static_cast<int>(ceil_div(k, 64));
    a.kper = static_cast<int>(ceil_div(a.kblocks, splits));
    a.a_rows = static_cast<int>(std::min<int64_t>(128, (m + 7) / 8 * 8));
    a.act = activation;
    a.bf16 = dtype == CVS_BF16;
    a.bias = bias;
    a.residual = residual;
    a.out = y;
    a.z = z;
    a.ld_res = residual_stride;
    a.ld_out = y_stride;
    a.ld_z = z_stride;
    a.vec_res = aligned16(residual) && residual_stride % 8 == 0;
    a.vec_out = aligned16(y) && y_stride % 8 == 0;
    a.err = dev.err;
    CUtensorMap amap, bmap;
    if ((st = operand_map(&amap, {x, x_stride, false}, dtype, m, k, a.a_rows)) != CVS_OK) return st;
    if ((st = operand_map(&bmap, {w, w_stride, false}, dtype, n, k, 64)) != CVS_OK) return st;
    e = split_launch(splits, amap, bmap, a, a.tiles_m * static_cast<int>(ceil_div(n, 64)), s);
    return e == cudaSuccess ? CVS_OK : cuda_fail(e, "linear launch");
  }
  const Tile t = pick_tile(m, n, dev.sms);
  GemmMaps maps{};
  if ((st = operand_map(&maps.a[0], {x, x_stride, false}, dtype, m, k, 128)) != CVS_OK) return st;
  if ((st = operand_map(&maps.b[0], {w, w_stride, false}, dtype, n, k, t.bn / t.cg)) != CVS_OK) return st;
  GemmArgs a{};
  GemmProblem& p = a.p[0];
  set_shape(&p, t, m, n, k, 1);
  a.act = activation;
  p.out = y;
  p.ld_out = y_stride;
  p.vec_out = storable(y, y_stride, n);
  p.bias = bias;
  p.residual = residual;
  p.ld_res = residual_stride;
  p.vec_res = mappable(residual, residual_stride, n);
  p.z = z;
  p.ld_z = z_stride;
  if (p.vec_out && (st = block_map(&maps.out[0], y, dtype, m, n, y_stride)) != CVS_OK) return st;
  if (p.vec_res && (st = block_map(&maps.residual, residual, dtype, m, n, residual_stride)) != CVS_OK) return st;
  if (z && (st = block_map(&maps.z, z, CVS_F16, m, n, z_stride)) != CVS_OK) return st;
  a.bf16 = dtype == CVS_BF16;
  a.err = dev.err;
  e = gemm_launch(t.cg, t.bn, maps, a, grid_ctas(t, p.work, dev.sms), s);
  return e == cudaSuccess ? CVS_OK : cuda_fail(e, "linear launch");
}

cvs_status cvs_linear_backward_workspace_size(int activation, int64_t m, int n, int k, size_t* bytes) {
  if (!bytes) return fail(CVS_ERR_INVALID_ARGUMENT, "bytes must not be null");
  *bytes = 0;
  cvs_status st = check_linear(activation, CVS_F16, m, n, k);
  if (st != CVS_OK) return st;
  if (m == 0) return CVS_OK;
  DeviceInfo dev;
  if ((st = device_info(&dev)) != CVS_OK) return st;
  *bytes = plan_backward(m, n, k, dev.sms).bytes;
  return CVS_OK;
}

cvs_status cvs_linear_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* w,
                               int64_t w_stride, const void* z, int64_t z_stride, int activation, int dtype,
                               int64_t m, int n, int k, void* dx, int64_t dx_stride, void* dw, int64_t dw_stride,
                               void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  cvs_status st = check_linear(activation, dtype, m, n, k);
  if (st != CVS_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (dw && n > 1 && dw_stride < k) return fail(CVS_ERR_INVALID_ARGUMENT, "dw row stride smaller than its width");
  if (m == 0) {  // sums over no rows
    if (dw) e = cudaMemset2DAsync(dw, static_cast<size_t>(std::max<int64_t>(dw_stride, k)) * 2, 0, static_cast<size_t>(k) * 2, n, s);
    if (e == cudaSuccess && dbias) e = cudaMemsetAsync(dbias, 0, static_cast<size_t>(n) * 2, s);
    return e == cudaSuccess ? CVS_OK : cuda_fail(e, "clearing the weights' gradients");
  }
  if (!dx && !dw && !dbias) return CVS_OK;
  if (!dy) return fail(CVS_ERR_INVALID_ARGUMENT, "null pointer");
  if (m > 1 && dy_stride < 0) return fail(CVS_ERR_INVALID_ARGUMENT, "negative row stride");
  if (dx && m > 1 && dx_stride < k) return fail(CVS_ERR_INVALID_ARGUMENT, "dx row stride smaller than its width");
  if (dw && (st = check_operand(x, x_stride, k, "x")) != CVS_OK) return st;
  if (dx && (st = check_operand(w, w_stride, k, "w")) != CVS_OK) return st;
  const bool act = activation != CVS_ACT_NONE;
  if (act && (!z || !aligned16(z) || z_stride % 8 != 0 || z_stride < n))
    return fail(CVS_ERR_INVALID_ARGUMENT, "z must be 16-byte aligned with a row stride that is a multiple of 8 and at least n");
  DeviceInfo dev;
  if ((st = device_info(&dev)) != CVS_OK) return st;
  const BackwardPlan plan = plan_backward(m, n, k, dev.sms);
  const bool dy_tiles = mappable(dy, dy_stride, n);  // TMA can read dy itself
  const size_t need_bytes = plan.bytes - (act || !dy_tiles ? 0 : plan.bytes_dz);
  if ((st = check_workspace(workspace, workspace_bytes, need_bytes)) != CVS_OK) return st;
  char* base = static_cast<char*>(workspace);
  const bool bf16 = dtype == CVS_BF16;
  Operand dz{dy, dy_stride, false};
  if (act || !dy_tiles) dz = {base + plan.dz_offset, plan.dz_stride, false};
  const bool needs_dz = act || (!dy_tiles && (dx || dw));
  const auto launch_dz = [&]() {
    LinearDzArgs a{};
    a.dy = dy;
    a.ld_dy = dy_stride;
    a.vec_dy = aligned16(dy) && dy_stride % 8 == 0;
    a.z = act ? z : nullptr;
    a.ld_z = z_stride;
    a.dz = dz.p == dy || !(dx || dw) ? nullptr : const_cast<void*>(dz.p);
    a.ld_dz = plan.dz_stride;
    a.partial = dbias ? reinterpret_cast<float*>(base + plan.db_offset) : nullptr;
    a.m = m;
    a.n = n;
    a.act = activation;
    a.bf16 = bf16;
    return linear_dz_launch(a, plan.db_parts, s);
  };
  if (needs_dz && (e = launch_dz()) != cudaSuccess) return cuda_fail(e, "linear backward launch");
  const Tile& t = plan.tile;
  if (dx || dw) {
    GemmMaps maps{};
    GemmArgs a{};
    a.bf16 = bf16;
    a.err = dev.err;
    int i = 0;
    if (dw) {  // dw[n][k] = dz^T x: both operands have K (the rows) as their outer dimension
      GemmProblem& p = a.p[i];
      set_shape(&p, t, n, k, m, plan.splits);
      p.a_mn = p.b_mn = 1;
      p.out = dw;
      p.ld_out = dw_stride;
      p.vec_out = storable(dw, dw_stride, k);
      p.partial = p.splits > 1 ? reinterpret_cast<float*>(base + plan.dw_offset) : nullptr;
      if ((st = operand_map(&maps.a[i], {dz.p, dz.stride, true}, dtype, n, m, 64)) != CVS_OK) return st;
      if ((st = operand_map(&maps.b[i], {x, x_stride, true}, dtype, k, m, 64)) != CVS_OK) return st;
      if (p.vec_out && (st = block_map(&maps.out[i], dw, dtype, n, k, dw_stride)) != CVS_OK) return st;
      ++i;
    }
    if (dx) {  // dx[m][k] = dz w: w has K (its n rows) as its outer dimension
      GemmProblem& p = a.p[i];
      set_shape(&p, t, m, k, n, 1);
      p.b_mn = 1;
      p.out = dx;
      p.ld_out = dx_stride;
      p.vec_out = storable(dx, dx_stride, k);
      if ((st = operand_map(&maps.a[i], dz, dtype, m, n, 128)) != CVS_OK) return st;
      if ((st = operand_map(&maps.b[i], {w, w_stride, true}, dtype, k, n, 64)) != CVS_OK) return st;
      if (p.vec_out && (st = block_map(&maps.out[i], dx, dtype, m, k, dx_stride)) != CVS_OK) return st;
      ++i;
    }
    const int work = a.p[0].work + a.p[1].work;
    if ((e = gemm_launch(t.cg, t.bn, maps, a, grid_ctas(t, work, dev.sms), s)) != cudaSuccess)
      return cuda_fail(e, "linear backward launch");
  }
  // Without dz only dbias needs dy's columns: after the products, which leave part of dy in L2.
  if (!needs_dz && dbias && (e = launch_dz()) != cudaSuccess) return cuda_fail(e, "linear backward launch");
  LinearFinishArgs f{};
  f.db_partial = reinterpret_cast<const float*>(base + plan.db_offset);
  f.db_parts = plan.db_parts;
  f.db_blocks = dbias ? (n + 31) / 32 : 0;
  f.dbias = dbias;
  f.dw_partial = dw && plan.splits > 1 ? reinterpret_cast<const float*>(base + plan.dw_offset) : nullptr;
  f.splits = plan.splits;
  f.tiles_m = static_cast<int>(ceil_div(n, 128 * t.cg));
  f.tiles_n = static_cast<int>(ceil_div(k, t.bn));
  f.cg = t.cg;
  f.bn = t.bn;
  f.dw = dw;
  f.ld_dw = dw_stride;
  f.vec_dw = dw && aligned16(dw) && dw_stride % 8 == 0;
  f.n = n;
  f.k = k;
  f.bf16 = bf16;
  if ((e = linear_finish_launch(f, s)) != cudaSuccess) return cuda_fail(e, "linear backward launch");
  return CVS_OK;
}

cvs_status cvs_preference_loss_workspace_size(int64_t b, int r, size_t* bytes) {
  if (!bytes) return fail(CVS_ERR_INVALID_ARGUMENT, "bytes must not be null");
  *bytes = 0;
  if (b < 0 || b >= INT_MAX) return fail(CVS_ERR_INVALID_ARGUMENT, "query count out of range");
  if (r < 1 || r > CVS_MAX_REJECTED)
    return fail(CVS_ERR_INVALID_ARGUMENT, "rejected rows per query must be in 1 .. %d (got %d)", CVS_MAX_REJECTED, r);
  if (b == 0) return CVS_OK;
  DeviceInfo dev;
  const cvs_status st = device_info(&dev);
  if (st != CVS_OK) return st;
  *bytes = up(static_cast<size_t>(preference_blocks(b, r, dev.sms)) * 8);
  return CVS_OK;
}

cvs_status cvs_preference_loss(const void* q, int q_dtype, int64_t q_stride, const void* ref, int ref_dtype,
                               int64_t ref_stride, int64_t b, int d, int cosine, const void* x_f16, int64_t n,
                               int d_pad, const int64_t* chosen, const int64_t* rejected, int64_t rejected_stride,
                               int r, float scale, float label_smoothing, int mean, float* loss, float* weight,
                               float* margins, float* grad, int64_t grad_stride, void* workspace,
                               size_t workspace_bytes, void* stream) {
  if (b < 0 || b >= INT_MAX) return fail(CVS_ERR_INVALID_ARGUMENT, "query count %lld out of range", (long long)b);
  if (r < 1 || r > CVS_MAX_REJECTED)
    return fail(CVS_ERR_INVALID_ARGUMENT, "rejected rows per query must be in 1 .. %d (got %d)", CVS_MAX_REJECTED, r);
  if (n < 1 || n >= INT_MAX)
    return fail(CVS_ERR_INVALID_ARGUMENT, "corpus must have 1 .. 2^31-1 rows (got %lld)", (long long)n);
  if (d_pad < CVS_PAD || d_pad % CVS_PAD != 0 || d_pad > 2048)
    return fail(CVS_ERR_INVALID_ARGUMENT, "corpus width must be a multiple of 64 up to 2048 (got %d)", d_pad);
  if (d < 1 || d > d_pad) return fail(CVS_ERR_INVALID_ARGUMENT, "query width %d exceeds the corpus width %d", d, d_pad);
  if (!float_type(q_dtype) || (ref && !float_type(ref_dtype)))
    return fail(CVS_ERR_INVALID_ARGUMENT, "queries must be float32, float16 or bfloat16");
  if (!(label_smoothing >= 0.f && label_smoothing <= 1.f))
    return fail(CVS_ERR_INVALID_ARGUMENT, "label smoothing must be in 0 .. 1");
  if (!x_f16 || !aligned16(x_f16)) return fail(CVS_ERR_INVALID_ARGUMENT, "corpus must be a non-null 16-byte aligned pointer");
  if (!loss || !weight) return fail(CVS_ERR_INVALID_ARGUMENT, "null output pointer");
  if (b > 0 && (!q || !chosen || !rejected || !margins)) return fail(CVS_ERR_INVALID_ARGUMENT, "null pointer");
  if (b > 1 && (q_stride < 0 || (ref && ref_stride < 0) || rejected_stride < 0))
    return fail(CVS_ERR_INVALID_ARGUMENT, "negative row stride");
  if (grad && (!aligned16(grad) || grad_stride % 8 != 0 || grad_stride < d))
    return fail(CVS_ERR_INVALID_ARGUMENT, "grad must be 16-byte aligned with a row stride that is a multiple of 8 and at least d");
  DeviceInfo dev;
  cvs_status st = device_info(&dev);
  if (st != CVS_OK) return st;
  const size_t need = b == 0 ? 0 : up(static_cast<size_t>(preference_blocks(b, r, dev.sms)) * 8);
  if ((st = check_workspace(workspace, workspace_bytes, need)) != CVS_OK) return st;
  const auto vec = [d](const void* p, int dtype, int64_t stride) {
    return d % 8 == 0 && aligned16(p) && (stride * (dtype == CVS_F32 ? 4 : 2)) % 16 == 0;
  };
  PreferenceArgs a{};
  a.q = q;
  a.ref = ref;
  a.q_dtype = q_dtype;
  a.ref_dtype = ref_dtype;
  a.q_stride = q_stride;
  a.ref_stride = ref_stride;
  a.q_vec = vec(q, q_dtype, q_stride);
  a.ref_vec = ref && vec(ref, ref_dtype, ref_stride);
  a.cosine = cosine;
  a.x = static_cast<const __half*>(x_f16);
  a.n = n;
  a.d = d;
  a.d_pad = d_pad;
  a.chosen = reinterpret_cast<const long long*>(chosen);
  a.rejected = reinterpret_cast<const long long*>(rejected);
  a.rejected_stride = rejected_stride;
  a.b = b;
  a.r = r;
  a.scale = scale;
  a.smoothing = label_smoothing;
  a.margins = margins;
  a.grad = grad;
  a.grad_stride = grad_stride;
  a.partial = static_cast<float2*>(workspace);
  a.err = dev.err;
  const cudaError_t e = preference_launch(a, mean, loss, weight, dev.sms, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? CVS_OK : cuda_fail(e, "preference loss launch");
}

cvs_status cvs_preference_grad(const float* grad, int64_t grad_stride, int64_t b, int d, const float* weight,
                               const float* upstream, int dtype, void* dq, void* stream) {
  if (b < 0 || b >= INT_MAX) return fail(CVS_ERR_INVALID_ARGUMENT, "query count out of range");
  if (b == 0) return CVS_OK;
  if (d < 1 || grad_stride < d || grad_stride % 8 != 0)
    return fail(CVS_ERR_INVALID_ARGUMENT, "grad's row stride must be a multiple of 8 and at least d");
  if (!grad || !aligned16(grad) || !weight || !upstream || !dq)
    return fail(CVS_ERR_INVALID_ARGUMENT, "null or misaligned pointer");
  if (!float_type(dtype)) return fail(CVS_ERR_INVALID_ARGUMENT, "unsupported dtype %d", dtype);
  DeviceInfo dev;
  const cvs_status st = device_info(&dev);
  if (st != CVS_OK) return st;
  const cudaError_t e = preference_grad_launch(grad, grad_stride, b, d, weight, upstream, dtype, dq, dev.sms,
                                               static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? CVS_OK : cuda_fail(e, "preference gradient launch");
}

}  // extern "C"
