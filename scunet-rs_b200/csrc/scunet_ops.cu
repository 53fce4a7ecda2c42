// The block operators' C entries (include/scunet_b200.h): argument checks, the choice of
// kernel and launch shape, the launches. Context-free: they work on the caller's device
// pointers, on the caller's stream and in the caller's workspace, and allocate nothing.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdio>
#include <initializer_list>
#include <string>

#include "../../include/scunet_b200.h"
#include "host_logic.h"
#include "op_attn.cuh"
#include "op_attn_tc.cuh"
#include "op_norm.cuh"
#include "op_rotary.cuh"

using namespace scb;

namespace {

int refuse(const char* op, const std::string& msg) { return global_error(SCB_EINVAL, std::string(op) + ": " + msg); }

int launched(const char* op) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return global_error(SCB_ECUDA, std::string(op) + ": " + cudaGetErrorString(e));
  return SCB_OK;
}

// No C++ exception leaves a C entry (std::string may fail to allocate).
template <typename F>
int guarded(F&& f) noexcept {
  try {
    return f();
  } catch (...) {
    return SCB_ENOMEM;
  }
}

int elem_size(int dtype) { return dtype == SCB_F32 ? 4 : dtype == SCB_F16 || dtype == SCB_BF16 ? 2 : 0; }

uint64_t addr(const void* p) { return (uint64_t)reinterpret_cast<uintptr_t>(p); }

int sm_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return sms;
}

// ---------------------------------------------------------------------------- group norm
const long kMaxBlocks = 0x7fffffffl;

// Vectors per row, block tiling and splits of a group norm. `vec`: elements per access.
void norm_plan(NormGeom& g, int vec, int sms) {
  g.cpg = g.c / g.groups;
  g.cols = g.c / vec;
  g.tc = g.cols < NORM_THREADS ? g.cols : NORM_THREADS;
  g.rp = NORM_THREADS / g.tc;
  const long chunks = (g.cols + g.tc - 1) / g.tc;
  // about four blocks an SM over all pictures, each with at least four rows a thread
  long s = (4L * sms + g.n * chunks - 1) / (g.n * chunks);
  const long most = (g.l + 4L * g.rp - 1) / (4L * g.rp);
  s = s < most ? s : most;
  g.splits = (int)(s < 1 ? 1 : s);
}

// Workspace: one (mean, M2) or (sum, sum) per picture, split and channel, the pictures'
// joined sums, and mean and rstd for callers that do not ask for them. Sized for any
// vector width: a narrower one has fewer splits, never more.
long norm_most_splits(long n, long l, int sms) {
  long s = (4L * sms + n - 1) / n;
  const long most = (l + 3) / 4;
  s = s < most ? s : most;
  return s < 1 ? 1 : s;
}
size_t norm_work_bytes(long n, long l, int c, int groups, int sms) {
  return (size_t)n * norm_most_splits(n, l, sms) * c * 8 + (size_t)n * c * 8 + (size_t)n * groups * 8 + 256;
}

int norm_check(const char* op, int dtype, int64_t n, int64_t l, int c, int groups, int act) {
  if (!elem_size(dtype)) return refuse(op, "the element type must be SCB_F32, SCB_F16 or SCB_BF16");
  if (n < 0 || l < 0 || c < 1) return refuse(op, "n and l must not be negative, c must be positive");
  if (groups < 1 || c % groups)
    return refuse(op, std::to_string(c) + " channels do not split into " + std::to_string(groups) + " groups");
  if (act < 0 || act > 3) return refuse(op, "unknown activation");
  return SCB_OK;
}

// The widest access that every row of every tensor allows.
int norm_vec(int es, int c, std::initializer_list<uint64_t> bytes) {
  const int a = common_alignment(16, bytes);
  int v = a / es;
  if (v < 1) return 0;
  while (v > 1 && c % v) v /= 2;
  return v == 16 / es ? v : v >= 2 ? 2 : 1;
}

template <typename T, int V, int ACT>
void norm_apply(const NormGeom& g, dim3 grid, const void* x, void* y, const float* mean, const float* rstd,
                const float* w, const float* b, cudaStream_t st) {
  norm_apply_kernel<T, V, ACT><<<grid, NORM_THREADS, 0, st>>>(static_cast<const T*>(x), static_cast<T*>(y), mean, rstd,
                                                              w, b, g);
}

template <typename T, int V>
void norm_forward(const NormGeom& g, const void* x, void* y, const float* w, const float* b, float* mean, float* rstd,
                  float2* part, cudaStream_t st) {
  const dim3 grid((unsigned)(g.n * g.splits), (unsigned)((g.cols + g.tc - 1) / g.tc));
  const int smem = NORM_THREADS * 4 * (2 * V + 1);
  norm_stats_kernel<T, V><<<grid, NORM_THREADS, smem, st>>>(static_cast<const T*>(x), part, g);
  norm_join_kernel<<<(unsigned)(g.n * g.groups), NORM_THREADS, 0, st>>>(part, mean, rstd, g);
  if (V * sizeof(T) < 16)
    norm_apply<T, V, ACT_ANY>(g, grid, x, y, mean, rstd, w, b, st);
  else if (g.act == ACT_RELU)
    norm_apply<T, V, ACT_RELU>(g, grid, x, y, mean, rstd, w, b, st);
  else if (g.act == ACT_GELU)
    norm_apply<T, V, ACT_GELU>(g, grid, x, y, mean, rstd, w, b, st);
  else if (g.act == ACT_SILU)
    norm_apply<T, V, ACT_SILU>(g, grid, x, y, mean, rstd, w, b, st);
  else
    norm_apply<T, V, ACT_NONE>(g, grid, x, y, mean, rstd, w, b, st);
}

template <typename T, int V, int ACT>
void norm_backward_act(const NormGeom& g, const void* dy, const void* x, void* dx, const float* mean,
                       const float* rstd, const float* w, const float* b, float* dw, float* db, float2* part,
                       float2* sums, cudaStream_t st) {
  const dim3 grid((unsigned)(g.n * g.splits), (unsigned)((g.cols + g.tc - 1) / g.tc));
  const T *d = static_cast<const T*>(dy), *p = static_cast<const T*>(x);
  norm_grad_sums_kernel<T, V, ACT><<<grid, NORM_THREADS, NORM_THREADS * 8 * V, st>>>(d, p, mean, rstd, w, b, part, g);
  norm_grad_join_kernel<<<(unsigned)g.c, 32, 0, st>>>(part, sums, dw, db, g);
  norm_grad_apply_kernel<T, V, ACT><<<grid, NORM_THREADS, 0, st>>>(d, p, static_cast<T*>(dx), mean, rstd, w, b, sums, g);
}

template <typename T, int V>
void norm_backward(const NormGeom& g, const void* dy, const void* x, void* dx, const float* mean, const float* rstd,
                   const float* w, const float* b, float* dw, float* db, float2* part, float2* sums, cudaStream_t st) {
  if (V * sizeof(T) < 16)
    norm_backward_act<T, V, ACT_ANY>(g, dy, x, dx, mean, rstd, w, b, dw, db, part, sums, st);
  else if (g.act == ACT_RELU)
    norm_backward_act<T, V, ACT_RELU>(g, dy, x, dx, mean, rstd, w, b, dw, db, part, sums, st);
  else if (g.act == ACT_GELU)
    norm_backward_act<T, V, ACT_GELU>(g, dy, x, dx, mean, rstd, w, b, dw, db, part, sums, st);
  else if (g.act == ACT_SILU)
    norm_backward_act<T, V, ACT_SILU>(g, dy, x, dx, mean, rstd, w, b, dw, db, part, sums, st);
  else
    norm_backward_act<T, V, ACT_NONE>(g, dy, x, dx, mean, rstd, w, b, dw, db, part, sums, st);
}

// ---------------------------------------------------------------------------- attention
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
    return reinterpret_cast<EncodeTiledFn>(e == cudaSuccess && q == cudaDriverEntryPointSuccess ? p : nullptr);
  }();
  return fn;
}

// K or V as [picture][head][key][channel]: boxes of 128 keys x 64 channels, 128-byte
// swizzle; channels past d and keys past lk read zeros. A dimension that is broadcast
// (stride 0) or single has extent 1.
bool attn_map(CUtensorMap* m, const scb_rows& t, int dtype, int64_t b, int64_t lk, int hk, int d) {
  const EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const bool hs = hk > 1 && t.sh, bs = b > 1 && t.sb;
  cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)lk, (cuuint64_t)(hs ? hk : 1), (cuuint64_t)(bs ? b : 1)};
  cuuint64_t strides[3] = {lk > 1 ? (cuuint64_t)t.sl * 2 : 16, hs ? (cuuint64_t)t.sh * 2 : 16,
                           bs ? (cuuint64_t)t.sb * 2 : 16};
  cuuint32_t box[4] = {64, AT_KEYS, 1, 1}, one[4] = {1, 1, 1, 1};
  return fn(m, dtype == SCB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, t.x, dims,
            strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether TMA can read the tensor: 16-byte aligned rows, strides in its range.
bool attn_tma_ok(const scb_rows& t, int64_t b, int64_t lk, int hk) {
  const int64_t most = 1ll << 38;  // elements: strides below 2^40 bytes, with room
  if (addr(t.x) % 16 || lk > 0x7fffff00) return false;
  if (lk > 1 && (t.sl <= 0 || t.sl % 8 || t.sl > most)) return false;
  if (hk > 1 && (t.sh % 8 || t.sh > most)) return false;
  return !(b > 1 && (t.sb % 8 || t.sb > most));
}

// How the tensor-core kernel cuts the work (op_attn_tc.cuh).
struct AttnPlan {
  int twin, unit_rows, share;
  long rows, row_units, units, tiles, total;
  int grid;
  bool cut;
  size_t work;
};
AttnPlan attn_plan(int64_t b, int64_t lq, int64_t lk, int h, int hk, int d, int sms) {
  AttnPlan p{};
  p.share = h / hk;
  p.rows = lq * p.share;
  p.tiles = (lk + AT_KEYS - 1) / AT_KEYS;
  p.twin = p.rows <= 128 && p.tiles > 1;
  p.unit_rows = p.twin ? 128 : 256;
  p.row_units = (p.rows + p.unit_rows - 1) / p.unit_rows;
  p.units = b * hk * p.row_units;
  p.total = p.units * p.tiles;
  long grid = p.units;
  const long waves = (p.units + sms - 1) / sms;
  if (p.units < sms) {
    const long most = p.total / 4;  // at least four tiles a CTA
    grid = most < p.units ? p.units : most < sms ? most : sms;
  } else if (!p.twin && p.units < waves * sms * 95 / 100) {
    grid = sms;
  }
  p.grid = (int)(grid < kMaxBlocks ? grid : kMaxBlocks);
  p.cut = p.grid != p.units;
  p.work = p.cut || p.twin ? (size_t)p.grid * 2 * 256 * (d + 2) * sizeof(float) : 0;
  return p;
}

template <typename T, int Boxes>
int attn_tc_launch(const AttnTcArgs& g, const AttnPlan& p, const CUtensorMap& tk, const CUtensorMap& tv,
                   cudaStream_t st) {
  const auto kernel = attn_tc_kernel<T, Boxes>;
  constexpr int smem = AtLayout<Boxes>::kSmem;
  // the kernel's shared memory limit is raised once on each device
  static std::atomic<uint64_t> raised{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (!(raised.load() & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return global_error(SCB_ECUDA, std::string("scb_attention: ") + cudaGetErrorString(e));
    raised.fetch_or(bit);
  }
  kernel<<<p.grid, AT_THREADS, smem, st>>>(tk, tv, g);
  if (p.cut || p.twin) attn_join_kernel<T><<<(unsigned)(p.units * (p.unit_rows / 32)), AT_JOIN, 0, st>>>(g, p.grid);
  return launched("scb_attention");
}

// f<T, V>() for the element type and vector width.
#define NORM_DISPATCH(dtype, vec, F, ...)                                        \
  do {                                                                           \
    if (dtype == SCB_F32)                                                        \
      vec == 4 ? F<float, 4>(__VA_ARGS__) : vec == 2 ? F<float, 2>(__VA_ARGS__) : F<float, 1>(__VA_ARGS__); \
    else if (dtype == SCB_F16)                                                   \
      vec == 8 ? F<__half, 8>(__VA_ARGS__) : vec == 2 ? F<__half, 2>(__VA_ARGS__) : F<__half, 1>(__VA_ARGS__); \
    else                                                                         \
      vec == 8 ? F<__nv_bfloat16, 8>(__VA_ARGS__)                                \
               : vec == 2 ? F<__nv_bfloat16, 2>(__VA_ARGS__) : F<__nv_bfloat16, 1>(__VA_ARGS__); \
  } while (0)

}  // namespace

extern "C" {

int scb_group_norm_workspace(int64_t n, int64_t l, int c, int groups, size_t* bytes) {
  return guarded([&]() -> int {
    const char* op = "scb_group_norm_workspace";
    if (!bytes) return refuse(op, "bytes is NULL");
    *bytes = 0;
    if (int r = norm_check(op, SCB_F32, n, l, c, groups, 0)) return r;
    if (n == 0) return SCB_OK;
    const int sms = sm_count();
    if (!sms) return global_error(SCB_ECUDA, "no CUDA device");
    *bytes = norm_work_bytes(n, l, c, groups, sms);
    return SCB_OK;
  });
}

int scb_group_norm(const void* x, int64_t x_sn, int64_t x_sl, int dtype, int64_t n, int64_t l, int c, int groups,
                   const float* weight, const float* bias, float eps, int act, void* y, int64_t y_sn, int64_t y_sl,
                   float* mean, float* rstd, void* work, size_t work_bytes, void* stream) {
  return guarded([&]() -> int {
    const char* op = "scb_group_norm";
    if (int r = norm_check(op, dtype, n, l, c, groups, act)) return r;
    if (n == 0) return SCB_OK;
    if (l && (!x || !y)) return refuse(op, "NULL data pointer");
    if (x_sn < 0 || x_sl < 0 || !distinct_elements(c, {{l, y_sl}, {n, y_sn}}))
      return refuse(op, "negative input strides or overlapping output rows");
    if (!(eps >= 0.f)) return refuse(op, "eps must not be negative");
    const int es = elem_size(dtype), sms = sm_count();
    if (!sms) return global_error(SCB_ECUDA, "no CUDA device");
    if (!work || work_bytes < norm_work_bytes(n, l, c, groups, sms) || addr(work) % 16)
      return refuse(op, "the workspace is too small or not 16-byte aligned (scb_group_norm_workspace)");
    if ((mean && addr(mean) % 4) || (rstd && addr(rstd) % 4) || addr(weight) % 4 || addr(bias) % 4)
      return refuse(op, "misaligned float pointer");
    const int vec = norm_vec(es, c, {addr(x), addr(y), (uint64_t)(x_sn * es), (uint64_t)(x_sl * es),
                                     (uint64_t)(y_sn * es), (uint64_t)(y_sl * es)});
    if (!vec) return refuse(op, "data not aligned to its element size");
    NormGeom g{};
    g.n = n; g.l = l; g.c = c; g.groups = groups; g.eps = eps; g.act = act;
    g.x_sn = x_sn; g.x_sl = x_sl; g.y_sn = y_sn; g.y_sl = y_sl;
    norm_plan(g, vec, sms);
    if (g.n * g.splits > kMaxBlocks || n * groups > kMaxBlocks) return refuse(op, "too many pictures");
    float2* part = static_cast<float2*>(work);
    float* own = reinterpret_cast<float*>(part + (size_t)n * g.splits * c);
    if (!mean) mean = own;
    if (!rstd) rstd = own + (size_t)n * groups;
    NORM_DISPATCH(dtype, vec, norm_forward, g, x, y, weight, bias, mean, rstd, part, static_cast<cudaStream_t>(stream));
    return launched(op);
  });
}

int scb_group_norm_backward(const void* dy, int64_t d_sn, int64_t d_sl, const void* x, int64_t x_sn, int64_t x_sl,
                            int dtype, int64_t n, int64_t l, int c, int groups, const float* mean, const float* rstd,
                            const float* weight, const float* bias, int act, void* dx, int64_t dx_sn, int64_t dx_sl,
                            float* dweight, float* dbias, void* work, size_t work_bytes, void* stream) {
  return guarded([&]() -> int {
    const char* op = "scb_group_norm_backward";
    if (int r = norm_check(op, dtype, n, l, c, groups, act)) return r;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (addr(mean) % 4 || addr(rstd) % 4 || addr(weight) % 4 || addr(bias) % 4 || addr(dweight) % 4 || addr(dbias) % 4)
      return refuse(op, "misaligned float pointer");
    if (n == 0 || l == 0) {
      if (dweight) cudaMemsetAsync(dweight, 0, sizeof(float) * c, st);
      if (dbias) cudaMemsetAsync(dbias, 0, sizeof(float) * c, st);
      return launched(op);
    }
    if (!dy || !x || !dx || !mean || !rstd) return refuse(op, "NULL data pointer");
    if (d_sn < 0 || d_sl < 0 || x_sn < 0 || x_sl < 0 || !distinct_elements(c, {{l, dx_sl}, {n, dx_sn}}))
      return refuse(op, "negative input strides or overlapping output rows");
    const int es = elem_size(dtype), sms = sm_count();
    if (!sms) return global_error(SCB_ECUDA, "no CUDA device");
    if (!work || work_bytes < norm_work_bytes(n, l, c, groups, sms) || addr(work) % 16)
      return refuse(op, "the workspace is too small or not 16-byte aligned (scb_group_norm_workspace)");
    const int vec = norm_vec(es, c, {addr(x), addr(dy), addr(dx), (uint64_t)(x_sn * es), (uint64_t)(x_sl * es),
                                     (uint64_t)(d_sn * es), (uint64_t)(d_sl * es), (uint64_t)(dx_sn * es),
                                     (uint64_t)(dx_sl * es)});
    if (!vec) return refuse(op, "data not aligned to its element size");
    NormGeom g{};
    g.n = n; g.l = l; g.c = c; g.groups = groups; g.act = act;
    g.x_sn = x_sn; g.x_sl = x_sl; g.y_sn = dx_sn; g.y_sl = dx_sl; g.d_sn = d_sn; g.d_sl = d_sl;
    norm_plan(g, vec, sms);
    if (g.n * g.splits > kMaxBlocks) return refuse(op, "too many pictures");
    float2* part = static_cast<float2*>(work);
    float2* sums = part + (size_t)n * g.splits * c;
    NORM_DISPATCH(dtype, vec, norm_backward, g, dy, x, dx, mean, rstd, weight, bias, dweight, dbias, part, sums, st);
    return launched(op);
  });
}

int scb_rotate_axes(const scb_heads* q, const scb_heads* k, int dtype, int64_t b, int64_t l, int d, const void* pos,
                    int pos_dtype, int64_t pos_sb, int64_t pos_sl, int64_t pos_sa, const float* inv_freq,
                    const int* sections, int axes, int layout, int inverse, void* stream) {
  return guarded([&]() -> int {
    const char* op = "scb_rotate_axes";
    const int es = elem_size(dtype);
    if (!es) return refuse(op, "the element type must be SCB_F32, SCB_F16 or SCB_BF16");
    if (b < 0 || l < 0 || d < 2) return refuse(op, "b and l must not be negative, d must be at least 2");
    if (axes < 1 || axes > ROT_AXES || !sections) return refuse(op, "1 to 4 position axes");
    if (layout < 0 || layout > 2) return refuse(op, "unknown layout");
    if (!q || !inv_freq || (!pos && b && l)) return refuse(op, "NULL pointer");
    RotGeom g{};
    for (int a = 0; a < axes; ++a) {
      if (sections[a] < 0 || sections[a] > d / 2) return refuse(op, "a section is negative or too wide");
      g.first[a] = g.pairs;
      g.pairs += sections[a];
    }
    for (int a = axes; a <= ROT_AXES; ++a) g.first[a] = g.pairs;
    if (g.pairs < 1 || 2 * g.pairs > d)
      return refuse(op, "the sections' " + std::to_string(g.pairs) + " pairs must be 1 to " + std::to_string(d / 2));
    if (pos_dtype == SCB_I32)
      g.pos_type = POS_I32;
    else if (pos_dtype == SCB_I64)
      g.pos_type = POS_I64;
    else if (pos_dtype == SCB_F32)
      g.pos_type = POS_F32;
    else
      return refuse(op, "positions must be SCB_I32, SCB_I64 or SCB_F32");
    if (addr(pos) % (pos_dtype == SCB_I64 ? 8 : 4) || addr(inv_freq) % 4) return refuse(op, "misaligned positions");
    if (pos_sb < 0 || pos_sl < 0 || pos_sa < 0) return refuse(op, "negative position strides");
    const scb_heads* in[2] = {q, k};
    for (int w = 0; w < 2; ++w) {
      if (!in[w] || in[w]->heads == 0) continue;
      const scb_heads& t = *in[w];
      if (t.heads < 0) return refuse(op, "negative number of heads");
      if (b && l && (!t.x || !t.y)) return refuse(op, "NULL data pointer");
      if (addr(t.x) % es || addr(t.y) % es) return refuse(op, "data not aligned to its element size");
      if (t.x_sb < 0 || t.x_sl < 0 || t.x_sh < 0 ||
          !distinct_elements(d, {{b, t.y_sb}, {l, t.y_sl}, {t.heads, t.y_sh}}))
        return refuse(op, "negative input strides or overlapping outputs");
      g.t[w] = RotTensor{t.x, t.y, t.heads, t.x_sb, t.x_sl, t.x_sh, t.y_sb, t.y_sl, t.y_sh};
    }
    if (b == 0 || l == 0) return SCB_OK;
    g.b = b; g.l = l; g.tokens = b * l; g.d = d; g.axes = axes;
    g.pos = pos; g.pos_sb = pos_sb; g.pos_sl = pos_sl; g.pos_sa = pos_sa;
    g.freq = inv_freq;
    g.sign = inverse ? -1.f : 1.f;
    g.per_block = 8;
    while (g.per_block > 1 && g.per_block * g.pairs > 4096) g.per_block /= 2;
    if (g.pairs > 4096) return refuse(op, "heads wider than 8192 channels");
    const long blocks = (g.tokens + g.per_block - 1) / g.per_block;
    if (blocks > kMaxBlocks) return refuse(op, "too many tokens");
    const int smem = g.per_block * g.pairs * (int)sizeof(float2);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define ROT_LAYOUTS(T)                                                                            \
  (layout == ROT_HALF ? rotary_kernel<T, ROT_HALF><<<(unsigned)blocks, ROT_THREADS, smem, st>>>(g) \
   : layout == ROT_INTERLEAVED                                                                    \
       ? rotary_kernel<T, ROT_INTERLEAVED><<<(unsigned)blocks, ROT_THREADS, smem, st>>>(g)        \
       : rotary_kernel<T, ROT_AXIAL><<<(unsigned)blocks, ROT_THREADS, smem, st>>>(g))
    if (dtype == SCB_F32)
      ROT_LAYOUTS(float);
    else if (dtype == SCB_F16)
      ROT_LAYOUTS(__half);
    else
      ROT_LAYOUTS(__nv_bfloat16);
#undef ROT_LAYOUTS
    return launched(op);
  });
}

int scb_attention_workspace(int64_t b, int64_t lq, int64_t lk, int h, int hk, int d, size_t* bytes) {
  return guarded([&]() -> int {
    if (!bytes) return refuse("scb_attention_workspace", "bytes is NULL");
    *bytes = 0;
    if (b < 0 || lq < 0 || lk < 0 || h < 1 || hk < 1 || h % hk || d < 1)
      return refuse("scb_attention_workspace", "bad sizes");
    if (!b || !lq || !lk || d > 128) return SCB_OK;
    const int sms = sm_count();
    if (!sms) return global_error(SCB_ECUDA, "no CUDA device");
    *bytes = attn_plan(b, lq, lk, h, hk, d, sms).work;
    return SCB_OK;
  });
}

int scb_attention(const scb_rows* q, const scb_rows* k, const scb_rows* v, const scb_rows* o, int dtype, int64_t b,
                  int64_t lq, int64_t lk, int h, int hk, int d, const unsigned char* key_mask, int64_t mask_sb,
                  float scale, void* work, size_t work_bytes, void* stream) {
  return guarded([&]() -> int {
    const char* op = "scb_attention";
    if (dtype != SCB_F16 && dtype != SCB_BF16) return refuse(op, "the element type must be SCB_F16 or SCB_BF16");
    if (b < 0 || lq < 0 || lk < 0) return refuse(op, "negative size");
    if (h < 1 || hk < 1 || h % hk)
      return refuse(op, std::to_string(h) + " query heads cannot share " + std::to_string(hk) + " key heads");
    if (d < 1 || d > ATTN_ANY_D) return refuse(op, "heads must be 1 to 256 channels wide");
    if (!q || !k || !v || !o) return refuse(op, "NULL pointer");
    if (!std::isfinite(scale)) return refuse(op, "the scale must be finite");
    if (b == 0 || lq == 0) return SCB_OK;
    if (!q->x || !o->x || (lk && (!k->x || !v->x))) return refuse(op, "NULL data pointer");
    for (const scb_rows* t : {q, k, v, o}) {
      if (addr(t->x) % 2) return refuse(op, "data not aligned to its element size");
      if (t->sb < 0 || t->sl < 0 || t->sh < 0) return refuse(op, "negative strides");
    }
    if (!distinct_elements(d, {{b, o->sb}, {lq, o->sl}, {h, o->sh}})) return refuse(op, "overlapping output");
    if (key_mask && mask_sb < 0) return refuse(op, "negative strides");
    AttnArgs a{};
    a.q = q->x; a.k = k->x; a.v = v->x; a.o = o->x;
    a.mask = key_mask; a.m_sb = mask_sb;
    a.b = (int)b; a.h = h; a.hk = hk; a.d = d; a.lq = lq; a.lk = lk;
    a.q_sb = q->sb; a.q_sl = q->sl; a.q_sh = q->sh;
    a.k_sb = k->sb; a.k_sl = k->sl; a.k_sh = k->sh;
    a.v_sb = v->sb; a.v_sl = v->sl; a.v_sh = v->sh;
    a.o_sb = o->sb; a.o_sl = o->sl; a.o_sh = o->sh;
    a.scale_log2 = scale * 1.4426950408889634f;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (lk && d <= 128 && attn_tma_ok(*k, b, lk, hk) && attn_tma_ok(*v, b, lk, hk)) {
      const int sms = sm_count();
      if (!sms) return global_error(SCB_ECUDA, "no CUDA device");
      const AttnPlan p = attn_plan(b, lq, lk, h, hk, d, sms);
      if (p.units <= kMaxBlocks / 256) {
        if (p.work && (!work || work_bytes < p.work || addr(work) % 16))
          return refuse(op, "the workspace is too small or not 16-byte aligned (scb_attention_workspace)");
        AttnTcArgs g{};
        g.a = a;
        g.share = p.share; g.rows = p.rows; g.twin = p.twin; g.unit_rows = p.unit_rows; g.row_units = p.row_units;
        g.units = p.units; g.tiles = p.tiles; g.total = p.total;
        g.kv_b = (b > 1 && k->sb ? 1 : 0) | (b > 1 && v->sb ? 2 : 0);
        g.kv_h = (hk > 1 && k->sh ? 1 : 0) | (hk > 1 && v->sh ? 2 : 0);
        g.qneg = scale < 0 ? 1 : a.scale_log2 == 0 ? 2 : 0;
        g.a.scale_log2 = g.qneg == 2 ? 1.f : std::fabs(a.scale_log2);
        g.part = static_cast<float*>(work);
        g.part_ml = reinterpret_cast<float2*>(g.part + (size_t)p.grid * 2 * 256 * d);
        const auto wide = [&](const scb_rows* t) {
          return addr(t->x) % 16 == 0 && t->sb % 8 == 0 && t->sl % 8 == 0 && t->sh % 8 == 0;
        };
        g.q_wide = wide(q);
        g.o_wide = wide(o);
        CUtensorMap tk, tv;
        if (!attn_map(&tk, *k, dtype, b, lk, hk, d) || !attn_map(&tv, *v, dtype, b, lk, hk, d))
          return global_error(SCB_ECUDA, "scb_attention: no tensor map for k or v");
        if (dtype == SCB_F16)
          return d <= 64 ? attn_tc_launch<__half, 1>(g, p, tk, tv, st) : attn_tc_launch<__half, 2>(g, p, tk, tv, st);
        return d <= 64 ? attn_tc_launch<__nv_bfloat16, 1>(g, p, tk, tv, st)
                       : attn_tc_launch<__nv_bfloat16, 2>(g, p, tk, tv, st);
      }
    }
    const long blocks = (lq + ATTN_ANY_WARPS - 1) / ATTN_ANY_WARPS;
    if (b > kMaxBlocks / h || blocks > kMaxBlocks / (b * h)) return refuse(op, "too many queries");
    if (dtype == SCB_F16)
      attn_any_kernel<__half><<<(unsigned)(blocks * b * h), 32 * ATTN_ANY_WARPS, 0, st>>>(a);
    else
      attn_any_kernel<__nv_bfloat16><<<(unsigned)(blocks * b * h), 32 * ATTN_ANY_WARPS, 0, st>>>(a);
    return launched(op);
  });
}

int scb_op_status(void* stream) {
  return guarded([&]() -> int {
    cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
    unsigned v = 0;
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, g_device_error, sizeof v);
    if (e != cudaSuccess) return global_error(SCB_ECUDA, std::string("scb_op_status: ") + cudaGetErrorString(e));
    if (!v) return SCB_OK;
    const unsigned zero = 0;
    cudaMemcpyToSymbol(g_device_error, &zero, sizeof zero);
    return global_error(SCB_EDEVICE,
                        "a kernel gave up on a bounded wait (device error code " + std::to_string(v) + ")");
  });
}

}  // extern "C"
