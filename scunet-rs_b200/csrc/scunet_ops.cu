// The block operators' C entries (include/scunet_b200.h): argument checks, the choice of
// kernel and launch shape, the launches. Context-free: they work on the caller's device
// pointers, on the caller's stream and in the caller's workspace, and allocate nothing.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <initializer_list>
#include <string>
#include <type_traits>

#include "../../include/scunet_b200.h"
#include "host_logic.h"
#include "op_attn.cuh"
#include "op_attn_tc.cuh"
#include "op_norm.cuh"
#include "op_rotary.cuh"

using namespace scb;

namespace {

int refuse(const char* op, const std::string& msg) { return global_error(SCB_EINVAL, std::string(op) + ": " + msg); }

// What the runtime calls and launches of an operator came to. A failure is taken back from the
// runtime's memory of it, or the next call would report it as its own.
int finished(const char* op, cudaError_t e) {
  if (e == cudaSuccess) return SCB_OK;
  cudaGetLastError();
  return global_error(SCB_ECUDA, std::string(op) + ": " + cudaGetErrorString(e));
}

// No C++ exception leaves a C entry (std::string may fail to allocate).
template <typename F>
int guarded(F&& f) noexcept {
  try {
    return f();
  } catch (...) {
    try {
      return global_error(SCB_ENOMEM, "out of memory");  // short enough to need none
    } catch (...) {
      return SCB_ENOMEM;
    }
  }
}

int elem_size(int dtype) { return dtype == SCB_F32 ? 4 : dtype == SCB_F16 || dtype == SCB_BF16 ? 2 : 0; }

uint64_t addr(const void* p) { return (uint64_t)reinterpret_cast<uintptr_t>(p); }

int sm_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) == cudaSuccess &&
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess)
    return sms;
  cudaGetLastError();
  return 0;
}

// A launch, which returns its own error (cudaGetLastError after it would return one that was
// left from before). `with`: one attribute, or null.
template <typename... P, typename... A>
cudaError_t launch_with(cudaLaunchAttribute* with, void (*kernel)(P...), dim3 grid, int threads, size_t smem,
                        cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = with;
  cfg.numAttrs = with ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
  return launch_with(nullptr, kernel, grid, threads, smem, st, args...);
}
// Launch `kernel` so that it may start while the launch before it in the stream ends
// (it waits for that launch's results itself).
template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchAttribute a;
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
  return launch_with(&a, kernel, grid, threads, smem, st, args...);
}

// ---------------------------------------------------------------------------- group norm
const long kMaxBlocks = 0x7fffffffl;

// What a group norm's launches look like.
struct NormPlan {
  NormGeom g;
  bool small;
  int threads;        // of the small form
  size_t smem;        // of the small form
  size_t part, cpart; // float2 of the workspace: the groups' partials, the channels'
};

// `vec` elements per access of `es` bytes. The two-pass form takes all pictures in one pair of
// launches: a pair for each picture, so that the second pass might find the first one's reads
// in L2, measured 180 us against 119 us for the gradient of 4 x 136 x 240 x 512 fp16.
NormPlan norm_plan(NormGeom g, int vec, int es, bool grad, int sms) {
  NormPlan p{};
  g.cpg = g.c / g.groups;
  g.cols = g.c / vec;
  g.whole = g.cpg % vec == 0;
  const int bufs = grad ? 2 : 1;
  // ---- small: whole groups whose values fit; at least 64 bytes of a row (two sectors), and
  // some work for a block
  int unit = g.cpg;
  while (unit % vec) unit += g.cpg;
  // sums and segments, K, six floats a group; then the values
  const auto keep = [&](long cc, int threads) {
    const long segs = cc > threads ? cc : threads;
    return (2L * vec * threads + 2 * segs + (cc + 1) / 2 * 2 + 6 * (cc / g.cpg) + 3) / 4 * 4;
  };
  const auto bytes = [&](long cc, int parts) { return (double)((g.l + parts - 1) / parts) * cc * es * bufs; };
  const auto fits = [&](long cc, int parts) {
    return cc <= 512L * vec && 4.0 * keep(cc, 512) + bytes(cc, parts) <= 226 * 1024;
  };
  if (fits(unit, 8)) {
    long cc = unit;
    while (cc < g.c && fits(cc + unit, 8) && (cc * es < 64 || bytes(cc, 1) < 8192)) cc += unit;
    g.chunks = (int)((g.c + cc - 1) / cc);
    // blocks of a cluster: as many as the values need; more while a block holds over 16 KB and
    // SMs are free
    int parts = 1;
    while (!fits(cc, parts) || (parts < 8 && bytes(cc, parts) > 16384 && 2 * parts * g.n * g.chunks <= sms)) parts *= 2;
    p.small = true;
    p.threads = bytes(cc, parts) <= 16384 && cc <= 128L * vec ? 128 : 512;
    g.tc = (int)(cc / vec);
    g.rp = p.threads / g.tc;
    g.splits = parts;
    g.range = (g.l + parts - 1) / parts;
    g.keep = (int)keep(cc, p.threads);
    p.smem = 4 * (size_t)g.keep + (size_t)g.range * cc * es * bufs;
    p.cpart = grad && g.n * parts > 1 ? (size_t)g.n * parts * g.c : 0;
    p.g = g;
    return p;
  }
  // ---- two passes
  g.tc = g.cols < NORM_THREADS ? g.cols : NORM_THREADS;
  g.rp = NORM_THREADS / g.tc;
  g.chunks = (g.cols + g.tc - 1) / g.tc;
  g.slots = g.groups + g.chunks - 1;
  // the blocks of one launch just fill the SMs; four rows a thread or more
  long s = (grad ? norm_grad_blocks(vec) : 2) * sms / (g.n * g.chunks);
  const long most = (g.l + 4L * g.rp - 1) / (4L * g.rp);
  s = s < most ? s : most;
  g.splits = (int)(s < 1 ? 1 : s);
  g.cycles = g.l / ((long)g.rp * g.splits);
  p.part = (size_t)g.n * g.splits * g.slots;
  p.cpart = grad ? (size_t)g.n * g.splits * g.c : 0;
  p.g = g;
  return p;
}

// Workspace for either direction, any element type and vector width.
size_t norm_work_bytes(long n, long l, int c, int groups, int sms) {
  size_t most = 0;
  for (int es = 2; es <= 4; es += 2)
    for (int vec = 1; vec <= 16 / es; vec *= 2) {
      if (c % vec) break;
      for (int grad = 0; grad < 2; ++grad) {
        NormGeom g{};
        g.n = n;
        g.l = l;
        g.c = c;
        g.groups = groups;
        const NormPlan p = norm_plan(g, vec, es, grad, sms);
        if (p.part + p.cpart > most) most = p.part + p.cpart;
      }
    }
  return most * sizeof(float2);
}

int norm_check(const char* op, int dtype, int64_t n, int64_t l, int c, int groups, int act) {
  if (!elem_size(dtype)) return refuse(op, "the element type must be SCB_F32, SCB_F16 or SCB_BF16");
  if (n < 0 || l < 0 || c < 1) return refuse(op, "n and l must not be negative, c must be positive");
  if (groups < 1 || c % groups)
    return refuse(op, std::to_string(c) + " channels do not split into " + std::to_string(groups) + " groups");
  if (act < 0 || act > 3) return refuse(op, "unknown activation");
  return SCB_OK;
}

// Elements of the widest access, `most` bytes at most, that every row of every tensor allows.
int norm_vec(int es, int c, int most, std::initializer_list<uint64_t> bytes) {
  const int a = common_alignment(most, bytes);
  int v = a / es;
  if (v < 1) return 0;
  while (v > 1 && c % v) v /= 2;
  return v;
}

// Raises a kernel's shared memory limit, once on each device (`raised`: one per kernel).
cudaError_t allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& raised) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (raised.load() & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) raised.fetch_or(bit);
  return e;
}

struct NormArgs {
  const void *dy, *x;
  void* y;
  float *mean, *rstd;
  const float *weight, *bias;
  float *dweight, *dbias;
  float2 *part, *cpart;
  cudaStream_t st;
};

template <typename T, int V, bool GRAD, int kT>
cudaError_t norm_small(const NormPlan& p, const NormArgs& a) {
  const auto kernel = norm_small_kernel<T, V, GRAD, kT>;
  static std::atomic<uint64_t> raised{0};
  const cudaError_t e = allow_smem((const void*)kernel, 227 * 1024, raised);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = (unsigned)p.g.splits;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  return launch_with(p.g.splits > 1 ? &cluster : nullptr, kernel,
                     dim3((unsigned)(p.g.n * p.g.splits), (unsigned)p.g.chunks), kT, p.smem, a.st,
                     static_cast<const T*>(a.dy), static_cast<const T*>(a.x), static_cast<T*>(a.y), a.mean, a.rstd,
                     a.weight, a.bias, a.dweight, a.dbias, p.cpart ? a.cpart : nullptr, p.g);
}

// Floats, rounded up to 16 bytes.
int ring_at(size_t floats) { return (int)((floats + 3) / 4 * 4); }

template <typename T, int V, int ACT>
cudaError_t norm_two_pass(const NormPlan& p, const NormArgs& a) {
  NormGeom gs = p.g, ga = p.g;
  const T* x = static_cast<const T*>(a.x);
  constexpr int ring = RowStream<T, V, 1, NORM_THREADS>::kSmem;
  gs.keep = std::max(ring / 4, ring_at(BlockSums<V, NORM_THREADS>::floats(gs.tc)));
  const int smem_s = 4 * (gs.keep + gs.tc * V);                                              // and K
  ga.keep = ring_at(2 * ((size_t)ga.tc * V / ga.cpg + 2));                                   // statistics
  static std::atomic<uint64_t> raised_s{0}, raised_a{0};
  cudaError_t e = allow_smem((const void*)norm_stats_kernel<T, V>, 113 * 1024, raised_s);
  if (e == cudaSuccess) e = allow_smem((const void*)norm_apply_kernel<T, V, ACT>, 113 * 1024, raised_a);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)(gs.n * gs.splits), (unsigned)gs.chunks);
  e = launch(norm_stats_kernel<T, V>, grid, NORM_THREADS, smem_s, a.st, x, a.part, gs);
  if (e != cudaSuccess) return e;
  return launch_after(norm_apply_kernel<T, V, ACT>, grid, NORM_THREADS, 4 * ga.keep + ring, a.st, x,
                      static_cast<T*>(a.y), a.part, a.mean, a.rstd, a.weight, a.bias, ga);
}

template <typename T, int V, int ACT>
cudaError_t norm_two_pass_grad(const NormPlan& p, const NormArgs& a) {
  NormGeom gs = p.g, ga = p.g;
  const T *x = static_cast<const T*>(a.x), *dy = static_cast<const T*>(a.dy);
  constexpr int ring = RowStream<T, V, 2, NORM_THREADS>::kSmem;
  const size_t stat = 2 * ((size_t)gs.tc * V / gs.cpg + 2);
  gs.keep = std::max(ring / 4, ring_at(BlockSums<V, NORM_THREADS>::floats(gs.tc)));
  const int smem_s = 4 * (gs.keep + (int)stat);
  ga.keep = ring_at(2 * stat);
  static std::atomic<uint64_t> raised_s{0}, raised_a{0};
  cudaError_t e = allow_smem((const void*)norm_grad_sums_kernel<T, V, ACT>, 113 * 1024, raised_s);
  if (e == cudaSuccess) e = allow_smem((const void*)norm_grad_apply_kernel<T, V, ACT>, 113 * 1024, raised_a);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)(gs.n * gs.splits), (unsigned)gs.chunks);
  e = launch(norm_grad_sums_kernel<T, V, ACT>, grid, NORM_THREADS, smem_s, a.st, dy, x, a.mean, a.rstd, a.weight,
             a.bias, a.part, a.cpart, gs);
  if (e != cudaSuccess) return e;
  return launch_after(norm_grad_apply_kernel<T, V, ACT>, grid, NORM_THREADS, 4 * ga.keep + ring, a.st, dy, x,
                      static_cast<T*>(a.y), a.mean, a.rstd, a.weight, a.bias, a.part, ga);
}

template <typename T, int V>
cudaError_t norm_forward(const NormPlan& p, const NormArgs& a) {
  if (p.small) return p.threads == 128 ? norm_small<T, V, false, 128>(p, a) : norm_small<T, V, false, 512>(p, a);
  if (V * sizeof(T) < 16) return norm_two_pass<T, V, ACT_ANY>(p, a);
  if (p.g.act == ACT_RELU) return norm_two_pass<T, V, ACT_RELU>(p, a);
  if (p.g.act == ACT_GELU) return norm_two_pass<T, V, ACT_GELU>(p, a);
  if (p.g.act == ACT_SILU) return norm_two_pass<T, V, ACT_SILU>(p, a);
  return norm_two_pass<T, V, ACT_NONE>(p, a);
}

template <typename T, int V>
cudaError_t norm_grad_x(const NormPlan& p, const NormArgs& a) {
  if (p.small) return p.threads == 128 ? norm_small<T, V, true, 128>(p, a) : norm_small<T, V, true, 512>(p, a);
  if (V < 4) return norm_two_pass_grad<T, V, ACT_ANY>(p, a);
  if (p.g.act == ACT_RELU) return norm_two_pass_grad<T, V, ACT_RELU>(p, a);
  if (p.g.act == ACT_GELU) return norm_two_pass_grad<T, V, ACT_GELU>(p, a);
  if (p.g.act == ACT_SILU) return norm_two_pass_grad<T, V, ACT_SILU>(p, a);
  return norm_two_pass_grad<T, V, ACT_NONE>(p, a);
}

template <typename T, int V>
cudaError_t norm_backward(const NormPlan& p, const NormArgs& a) {
  const cudaError_t e = norm_grad_x<T, V>(p, a);
  if (e != cudaSuccess || !p.cpart || !(a.dweight || a.dbias)) return e;
  return launch(norm_grad_params_kernel, dim3((unsigned)((p.g.c + 31) / 32)), 1024, 0, a.st, a.cpart,
                p.g.n * p.g.splits, p.g.c, a.dweight, a.dbias);
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
  int grid, cuts, pieces;  // pieces: of a unit, at most
  bool cut;
  size_t places, work;  // pieces of all units (places for them), the workspace's bytes
};
AttnPlan attn_plan(int64_t b, int64_t lq, int64_t lk, int h, int hk, int d, int sms) {
  AttnPlan p{};
  p.share = h / hk;
  p.rows = lq * p.share;
  p.tiles = (lk + AT_KEYS - 1) / AT_KEYS;
  // Twin units always leave pieces, whose cost grows with the rows, so they need some tiles.
  // Heads of 64 fp16, us without and with twin:
  //   140 pictures x 8 rows, 500 keys: 17 / 21; 1000 keys: 35 / 24; 128 rows, 1000 keys: 39 / 30
  //   2000 x 8, 300: 156 / 158; 500: 175 / 159; 2040: 413 / 275;  2000 x 128, 1000: 301 / 352; 2040: 462 / 448
  // and with very few units the join of many pieces of each (4 x 1 row, 32640 keys: 56 / 65;
  // 16 x 1: 69 / 54). Past a GB of workspace the units are whole, without any.
  const long keys_of_heads = b * hk, least = keys_of_heads <= sms ? 5 : p.rows <= 32 ? 4 : p.rows / 8;
  p.twin = p.rows <= 128 && p.tiles >= least && keys_of_heads >= 8 &&
           (keys_of_heads <= sms || keys_of_heads <= (1L << 30) / (256 * (d + 2) * (long)sizeof(float)));
  p.unit_rows = p.twin ? 128 : 256;
  p.row_units = (p.rows + p.unit_rows - 1) / p.unit_rows;
  p.units = b * hk * p.row_units;
  p.total = p.units * p.tiles;
  long grid = p.units;
  const long waves = (p.units + sms - 1) / sms;
  if (p.twin) {
    // as many pieces as one round of CTAs holds (a second round measured 50 % slower), each
    // of eight tiles or more (16 pictures x 1 row, 2040 keys: 29 us from two tiles on, 22 so)
    const long most = p.tiles / 8, s = sms / p.units;
    p.cuts = (int)std::max(1L, std::min(s, most));
    grid = p.units * p.cuts;
  } else if (p.units < sms) {
    const long most = p.total / 4;  // at least four tiles a CTA
    grid = most < p.units ? p.units : most < sms ? most : sms;
  } else if (p.units < waves * sms * 95 / 100) {
    grid = sms;
  }
  p.grid = (int)(grid < kMaxBlocks ? grid : kMaxBlocks);
  p.cut = p.grid != p.units && p.tiles > 1;  // units of one tile are whole wherever the ranges end
  p.pieces = p.twin ? 2 * p.cuts : (int)(p.grid / p.units + 2);
  p.places = p.twin ? p.grid : p.cut ? 2 * (size_t)p.grid : 0;
  p.work = p.places * 256 * (d + 2) * sizeof(float);
  return p;
}

template <typename T, int Boxes, bool Twin>
int attn_tc_launch(const AttnTcArgs& g, const AttnPlan& p, const CUtensorMap& tk, const CUtensorMap& tv,
                   cudaStream_t st) {
  const char* op = "scb_attention";
  const auto kernel = attn_tc_kernel<T, Boxes, Twin>;
  const auto join = attn_join_kernel<T>;
  constexpr int smem = AtLayout<Boxes, Twin>::kSmem;
  static std::atomic<uint64_t> raised{0}, raised_join{0};
  if (!raised.load()) {
    // the kernel's register split draws on what it is launched with: less would wait forever
    cudaFuncAttributes fa;
    const cudaError_t e = cudaFuncGetAttributes(&fa, (const void*)kernel);
    if (e != cudaSuccess) return finished(op, e);
    if (fa.numRegs != AT_REGS)
      return global_error(SCB_ECUDA, "scb_attention: built with " + std::to_string(fa.numRegs) +
                                         " registers a thread, not " + std::to_string(AT_REGS));
  }
  const bool joined = p.cut || p.twin;
  cudaError_t e = allow_smem((const void*)kernel, smem, raised);
  if (e == cudaSuccess && joined) e = allow_smem((const void*)join, 128 * 1024, raised_join);
  if (e == cudaSuccess) e = launch(kernel, dim3((unsigned)p.grid), AT_THREADS, smem, st, tk, tv, g);
  if (e == cudaSuccess && joined)
    e = launch_after(join, dim3((unsigned)(p.units * (p.unit_rows / 32))), AT_JOIN, (size_t)256 * p.pieces, st, g,
                     p.grid);
  return finished(op, e);
}

// F<T, V>() for the element type and vector width.
#define NORM_16(T, vec, F, ...)                                                                              \
  (vec == 8   ? F<T, 8>(__VA_ARGS__)                                                                         \
   : vec == 4 ? F<T, 4>(__VA_ARGS__)                                                                         \
   : vec == 2 ? F<T, 2>(__VA_ARGS__)                                                                         \
              : F<T, 1>(__VA_ARGS__))
#define NORM_DISPATCH(dtype, vec, F, ...)                                                                    \
  (dtype == SCB_F16    ? NORM_16(__half, vec, F, __VA_ARGS__)                                                \
   : dtype == SCB_BF16 ? NORM_16(__nv_bfloat16, vec, F, __VA_ARGS__)                                         \
   : vec == 4          ? F<float, 4>(__VA_ARGS__)                                                            \
   : vec == 2          ? F<float, 2>(__VA_ARGS__)                                                            \
                       : F<float, 1>(__VA_ARGS__))

// scb_attention; `lose` as in AttnTcArgs.
int attention(const scb_rows* q, const scb_rows* k, const scb_rows* v, const scb_rows* o, int dtype, int64_t b,
              int64_t lq, int64_t lk, int h, int hk, int d, const unsigned char* key_mask, int64_t mask_sb,
              float scale, void* work, size_t work_bytes, void* stream, uint32_t lose) {
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
      if (p.units <= kMaxBlocks / 256 && p.grid > 0) {
        if (p.work && (!work || work_bytes < p.work || addr(work) % 16))
          return refuse(op, "the workspace is too small or not 16-byte aligned (scb_attention_workspace)");
        AttnTcArgs g{};
        g.a = a;
        g.share = p.share; g.rows = p.rows; g.twin = p.twin; g.unit_rows = p.unit_rows; g.cuts = p.cuts;
        g.row_units = p.row_units;
        g.units = p.units; g.tiles = p.tiles; g.total = p.total;
        g.turns = p.rows > 64;  // fewer rows leave the special function units idle anyway
        g.kv_b = (b > 1 && k->sb ? 1 : 0) | (b > 1 && v->sb ? 2 : 0);
        g.kv_h = (hk > 1 && k->sh ? 1 : 0) | (hk > 1 && v->sh ? 2 : 0);
        g.qneg = scale < 0 ? 1 : a.scale_log2 == 0 ? 2 : 0;
        g.a.scale_log2 = g.qneg == 2 ? 1.f : std::fabs(a.scale_log2);
        g.lose = lose;
        g.part = static_cast<float*>(work);
        g.part_ml = reinterpret_cast<float2*>(g.part + p.places * 256 * d);
        const auto wide = [&](const scb_rows* t) {
          return addr(t->x) % 16 == 0 && t->sb % 8 == 0 && t->sl % 8 == 0 && t->sh % 8 == 0;
        };
        g.q_wide = wide(q);
        g.o_wide = wide(o);
        CUtensorMap tk, tv;
        if (!attn_map(&tk, *k, dtype, b, lk, hk, d) || !attn_map(&tv, *v, dtype, b, lk, hk, d))
          return global_error(SCB_ECUDA, "scb_attention: no tensor map for k or v");
        const auto boxes = [&](auto type, auto twin) {
          using T = decltype(type);
          return d <= 64 ? attn_tc_launch<T, 1, decltype(twin)::value>(g, p, tk, tv, st)
                         : attn_tc_launch<T, 2, decltype(twin)::value>(g, p, tk, tv, st);
        };
        const auto typed = [&](auto type) {
          return p.twin ? boxes(type, std::true_type{}) : boxes(type, std::false_type{});
        };
        return dtype == SCB_F16 ? typed(__half{}) : typed(__nv_bfloat16{});
      }
    }
    const long blocks = (lq + ATTN_ANY_WARPS - 1) / ATTN_ANY_WARPS;
    if (b > kMaxBlocks / h || blocks > kMaxBlocks / (b * h)) return refuse(op, "too many queries");
    return finished(op, launch(dtype == SCB_F16 ? attn_any_kernel<__half> : attn_any_kernel<__nv_bfloat16>,
                               dim3((unsigned)(blocks * b * h)), 32 * ATTN_ANY_WARPS, 0, st, a));
  });
}

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
    if ((mean && addr(mean) % 4) || (rstd && addr(rstd) % 4) || addr(weight) % 4 || addr(bias) % 4)
      return refuse(op, "misaligned float pointer");
    const int vec = norm_vec(es, c, 16, {addr(x), addr(y), (uint64_t)(x_sn * es), (uint64_t)(x_sl * es),
                                     (uint64_t)(y_sn * es), (uint64_t)(y_sl * es)});
    if (!vec) return refuse(op, "data not aligned to its element size");
    NormGeom g{};
    g.n = n; g.l = l; g.c = c; g.groups = groups; g.eps = eps; g.act = act;
    g.x_sn = x_sn; g.x_sl = x_sl; g.y_sn = y_sn; g.y_sl = y_sl;
    const NormPlan p = norm_plan(g, vec, es, false, sms);
    const size_t need = (p.part + p.cpart) * sizeof(float2);
    if (need && (!work || work_bytes < need || addr(work) % 16))
      return refuse(op, "the workspace is too small or not 16-byte aligned (scb_group_norm_workspace)");
    if (n * p.g.splits > kMaxBlocks || p.g.chunks > 65535) return refuse(op, "too many pictures or channels");
    NormArgs a{};
    a.x = x; a.y = y; a.mean = mean; a.rstd = rstd; a.weight = weight; a.bias = bias;
    a.part = static_cast<float2*>(work);
    a.st = static_cast<cudaStream_t>(stream);
    return finished(op, NORM_DISPATCH(dtype, vec, norm_forward, p, a));
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
      cudaError_t e = cudaSuccess;
      if (dweight) e = cudaMemsetAsync(dweight, 0, sizeof(float) * c, st);
      if (dbias && e == cudaSuccess) e = cudaMemsetAsync(dbias, 0, sizeof(float) * c, st);
      return finished(op, e);
    }
    if (!dy || !x || !dx || !mean || !rstd) return refuse(op, "NULL data pointer");
    if (d_sn < 0 || d_sl < 0 || x_sn < 0 || x_sl < 0 || !distinct_elements(c, {{l, dx_sl}, {n, dx_sn}}))
      return refuse(op, "negative input strides or overlapping output rows");
    const int es = elem_size(dtype), sms = sm_count();
    if (!sms) return global_error(SCB_ECUDA, "no CUDA device");
    // vectors of 8 only within one group (op_norm.cuh, Hats)
    const int vec = norm_vec(es, c, es == 2 && c / groups % 8 ? 8 : 16,
                             {addr(x), addr(dy), addr(dx), (uint64_t)(x_sn * es), (uint64_t)(x_sl * es),
                              (uint64_t)(d_sn * es), (uint64_t)(d_sl * es), (uint64_t)(dx_sn * es),
                              (uint64_t)(dx_sl * es)});
    if (!vec) return refuse(op, "data not aligned to its element size");
    NormGeom g{};
    g.n = n; g.l = l; g.c = c; g.groups = groups; g.act = act;
    g.x_sn = x_sn; g.x_sl = x_sl; g.y_sn = dx_sn; g.y_sl = dx_sl; g.d_sn = d_sn; g.d_sl = d_sl;
    const NormPlan p = norm_plan(g, vec, es, true, sms);
    const size_t need = (p.part + p.cpart) * sizeof(float2);
    if (need && (!work || work_bytes < need || addr(work) % 16))
      return refuse(op, "the workspace is too small or not 16-byte aligned (scb_group_norm_workspace)");
    if (n * p.g.splits > kMaxBlocks || p.g.chunks > 65535) return refuse(op, "too many pictures or channels");
    NormArgs a{};
    a.dy = dy; a.x = x; a.y = dx; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
    a.weight = weight; a.bias = bias; a.dweight = dweight; a.dbias = dbias;
    a.part = static_cast<float2*>(work);
    a.cpart = a.part + p.part;
    a.st = st;
    return finished(op, NORM_DISPATCH(dtype, vec, norm_backward, p, a));
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
    if (l >= 0x7fff0000) return refuse(op, "too many tokens");
    if (g.pairs > 4096) return refuse(op, "heads wider than 8192 channels");
    // the widest vector that the sections, the strides and the addresses allow
    int vec = 16 / es;
    uint64_t bytes = 0;
    for (const RotTensor& t : g.t) {
      if (!t.heads) continue;
      bytes |= addr(t.x) | addr(t.y);
      for (int64_t s : {t.x_sb, t.x_sl, t.x_sh, t.y_sb, t.y_sl, t.y_sh}) bytes |= (uint64_t)s * es;
    }
    const auto splits = [&](int v) {
      if (layout == ROT_INTERLEAVED) return d % (2 * v) == 0;
      if (d % v || g.pairs % v) return false;
      if (layout == ROT_AXIAL)
        for (int a = 1; a <= axes; ++a)
          if (g.first[a] % v) return false;
      return true;
    };
    while (vec > 1 && (bytes % (uint64_t)(vec * es) || !splits(vec))) vec /= 2;
    g.vecs = layout == ROT_INTERLEAVED && vec > 1 ? d / 2 / vec : (d - g.pairs) / vec;
    g.items = (unsigned)g.vecs * (unsigned)(g.t[0].heads + g.t[1].heads);
    if (!g.items) return SCB_OK;
    if ((uint64_t)g.vecs * (uint64_t)(g.t[0].heads + g.t[1].heads) > 1u << 24)
      return refuse(op, "heads too many or too wide");
    // tokens of a block: eight items a thread (4 and 16 measured 3 and 5 % slower on wide heads), but
    // blocks for every SM; angles of at most 32 KB
    long per = (8L * ROT_THREADS + g.items - 1) / g.items;
    const int sms = sm_count();
    if (!sms) return global_error(SCB_ECUDA, "no CUDA device");
    const long share = (g.tokens + 2L * sms - 1) / (2L * sms);
    per = per < share ? per : share;
    per = per * g.pairs > 4096 ? 4096 / g.pairs : per;
    g.per_block = (int)(per < 1 ? 1 : per);
    g.by_items = Divide::by(g.items);
    g.by_vecs = Divide::by((unsigned)g.vecs);
    g.by_l = Divide::by((unsigned)l);
    g.by_pairs = Divide::by((unsigned)g.pairs);
    const long blocks = (g.tokens + g.per_block - 1) / g.per_block;
    if (blocks > kMaxBlocks) return refuse(op, "too many tokens");
    const int smem = g.per_block * g.pairs * (int)sizeof(float2);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    const auto turn = [&](auto kernel) { e = launch(kernel, dim3((unsigned)blocks), ROT_THREADS, smem, st, g); };
#define ROT_VECS(T, L)                                        \
  switch (vec) {                                              \
    case 8: turn(rotary_kernel<T, L, 16 / sizeof(T)>); break; \
    case 4: turn(rotary_kernel<T, L, 4>); break;              \
    case 2: turn(rotary_kernel<T, L, 2>); break;              \
    default: turn(rotary_kernel<T, L, 1>);                    \
  }
#define ROT_LAYOUTS(T)                                              \
  if (layout == ROT_HALF) {                                         \
    ROT_VECS(T, ROT_HALF)                                           \
  } else if (layout == ROT_INTERLEAVED) {                           \
    ROT_VECS(T, ROT_INTERLEAVED)                                    \
  } else {                                                          \
    ROT_VECS(T, ROT_AXIAL)                                          \
  }
    if (dtype == SCB_F32) {
      ROT_LAYOUTS(float)
    } else if (dtype == SCB_F16) {
      ROT_LAYOUTS(__half)
    } else {
      ROT_LAYOUTS(__nv_bfloat16)
    }
#undef ROT_LAYOUTS
#undef ROT_VECS
    return finished(op, e);
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
  return attention(q, k, v, o, dtype, b, lq, lk, h, hk, d, key_mask, mask_sb, scale, work, work_bytes, stream, AT_NONE);
}

int scb_probe_attention_lost(const scb_rows* q, const scb_rows* k, const scb_rows* v, const scb_rows* o, int dtype,
                             int64_t b, int64_t lq, int64_t lk, int h, int hk, int d, const unsigned char* key_mask,
                             int64_t mask_sb, float scale, void* work, size_t work_bytes, void* stream,
                             unsigned load) {
  return attention(q, k, v, o, dtype, b, lq, lk, h, hk, d, key_mask, mask_sb, scale, work, work_bytes, stream, load);
}

int scb_op_status(void* stream) {
  return guarded([&]() -> int {
    cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
    unsigned v = 0;
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, g_device_error, sizeof v);
    const unsigned zero = 0;
    if (e == cudaSuccess && v) e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof zero);
    if (e != cudaSuccess || !v) return finished("scb_op_status", e);
    return global_error(SCB_EDEVICE,
                        "a kernel gave up on a bounded wait (device error code " + std::to_string(v) + ")");
  });
}

}  // extern "C"
