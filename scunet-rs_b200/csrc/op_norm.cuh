// Group norm with an activation over channels-last maps, and its gradient.
//
//   x [N][L][C], G groups of C / G neighbouring channels; per picture n and group g
//   mean = E[x], var = E[(x - mean)^2] over the L rows and the group's channels,
//   xh = (x - mean) / sqrt(var + eps),  z = w_c xh + b_c,  y = act(z).
// Gradient, with gz = dy act'(z) and h = gz w_c:
//   db_c = sum gz,  dw_c = sum gz xh  (over n and L),
//   dx = rstd (h - E_g[h] - xh E_g[h xh]).
//
// Two forms, each with its gradient:
//  * norm_small_kernel: a picture's rows of a few whole groups fit in the shared memory of a
//    block, or of a cluster of up to eight that share the rows and read one another's sums
//    there; the values are read once, one launch.
//  * norm_stats_kernel, then norm_apply_kernel (norm_grad_sums_kernel, then
//    norm_grad_apply_kernel): blocks take rows of all pictures and leave one partial per
//    group; the second launch starts while the first one ends and every block joins its
//    picture's partials itself. (Walking the second pass backwards, to meet what the first
//    read last in L2, measured 3 to 9 % slower than forwards.)
// A thread keeps its channels (a vector of up to 16 bytes) and steps over rows.
//
// Bound by memory. The two passes of 2 x 1088 x 1920 x 64 fp16 (267 MB a picture, more than
// the chip holds) run at 5.5 TB/s of reading and 5.3 of reading and writing: 300 to 330 us
// where reading twice and writing once costs 248 us at the copy rate; 3 x 135 x 241 x 320 bf16
// 57 us, of which the second pass finds about half of x in L2 (27 to 37 of 62 MB from DRAM); the
// gradient of 4 x 136 x 240 x 512 fp16 126 us (104 us likewise). About 6 us of each pass are its
// start and its sums. The small form takes 6 us for 8 x 8 x 512.
//
// Precision: fp32 throughout; exponentials, reciprocals and quotients of the activations are the
// fast ones (2 ulp or so), which in fp32 shows: 1.3e-7 off where exact functions leave 1.0e-7
// to 1.2e-7 (gradient of 33 x 47 x 96), 1.4e-7 and 7e-8 on some small maps.
//
// Statistics are fp32: a block sums x - K and (x - K)^2 with K the median of the channel's
// values in its first, middle and last row, so that the sum of squares loses nothing to a
// large mean or to one value far from the rest. Two of those three rows may be far from the
// rest, as where a map has a border of its own: a block whose K lies more than eight spreads
// from its mean (NORM_FAR) sums once more, about that mean (rstd 2.5e-3 off before, 1e6 at both
// ends of 1088 x 1920 rows). (count, mean, M2) triples are joined,
//   M2 = M2a + M2b + (mb - ma)^2 na nb / (na + nb).
// No atomics: the order of every sum is fixed by the sizes.
#pragma once
#include "ops_common.cuh"

namespace scb {

struct NormGeom {
  long n, l;          // pictures, rows of each
  int c, groups, cpg; // channels, groups, channels per group
  int cols;           // vectors of a row
  int tc, rp;         // vectors of a row that one block takes (a chunk), rows it takes at once
  int chunks, slots;  // chunks of a row; groups + chunks - 1 partials of a split: a chunk's
                      // part of a group is slot group + chunk (a group may span chunks)
  int splits;         // parts of a picture's rows
  long cycles;        // l / (rp * splits)
  long range;         // small form: rows of a block
  int whole;          // a vector never spans two groups
  long x_sn, x_sl;    // element strides of pictures and rows
  long y_sn, y_sl;
  long d_sn, d_sl;    // dy
  float eps;
  int act;            // read by the kernels compiled for ACT_ANY
  int keep;           // floats of shared memory before the values (small form), the ring (second
                      // pass) or what lies behind the ring (first pass)
};

constexpr int NORM_THREADS = 512;  // two blocks an SM: every block reads its picture's partials

constexpr float NORM_FAR = 64.f;   // of a group: sum of (x - K)^2 over M2 that a block accepts

// Blocks of the gradient an SM: vectors of 8 take more than the 64 registers that two leave.
__host__ __device__ constexpr int norm_grad_blocks(int vec) { return vec == 8 ? 1 : 2; }

struct Moments {
  float n, mean, m2;
};
__device__ __forceinline__ Moments join(const Moments& a, const Moments& b) {
  const float n = a.n + b.n;
  if (a.n == 0.f) return b;
  if (b.n == 0.f) return a;
  const float d = b.mean - a.mean, f = __fdividef(b.n, n);
  return {n, a.mean + d * f, a.m2 + b.m2 + d * d * a.n * f};
}
__device__ __forceinline__ Moments shfl_xor(const Moments& m, int d) {
  return {__shfl_xor_sync(0xffffffffu, m.n, d), __shfl_xor_sync(0xffffffffu, m.mean, d),
          __shfl_xor_sync(0xffffffffu, m.m2, d)};
}
__device__ __forceinline__ float2 shfl_xor(const float2& v, int d) {
  return make_float2(__shfl_xor_sync(0xffffffffu, v.x, d), __shfl_xor_sync(0xffffffffu, v.y, d));
}
__device__ __forceinline__ float2 join(const float2& a, const float2& b) { return make_float2(a.x + b.x, a.y + b.y); }
// The join over a warp, the same in every lane (operands ordered by lane).
template <typename S>
__device__ __forceinline__ S warp_join(S v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const S o = shfl_xor(v, d);
    v = lane & d ? join(o, v) : join(v, o);
  }
  return v;
}

// V values in fp32 and back.
template <typename T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V>& a, float* v) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = to_f32(a.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> repack(const float* v) {
  Pack<T, V> a;
#pragma unroll
  for (int i = 0; i < V; ++i) a.v[i] = from_f32<T>(v[i]);
  return a;
}

// 1 / (1 + e^-z) of two values: e^-z overflows to inf below z = -88, whose reciprocal is 0.
__device__ __forceinline__ float2 sigmoid2(float2 z) {
  const float2 t = __fmul2_rn(z, make_float2(-1.4426950408889634f, -1.4426950408889634f));
  const float2 d = __fadd2_rn(make_float2(ex2_approx(t.x), ex2_approx(t.y)), make_float2(1.f, 1.f));
  return make_float2(rcp_approx(d.x), rcp_approx(d.y));
}

// The activation, and its slope, of V values; SiLU two at a time (packed arithmetic halves
// the instructions, which bound these passes before memory does).
template <int ACT, int V>
__device__ __forceinline__ void act_all(const NormGeom& g, float* z) {
  if constexpr (ACT == ACT_ANY) {
    if (g.act == ACT_SILU) return act_all<ACT_SILU, V>(g, z);
    if (g.act == ACT_GELU) return act_all<ACT_GELU, V>(g, z);
    if (g.act == ACT_RELU) return act_all<ACT_RELU, V>(g, z);
  } else if constexpr (ACT == ACT_SILU && V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 v = make_float2(z[i], z[i + 1]), r = __fmul2_rn(v, sigmoid2(v));
      z[i] = r.x;
      z[i + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = act_fwd<ACT>(z[i]);
  }
}
template <int ACT, int V>
__device__ __forceinline__ void slope_all(const NormGeom& g, float* z) {
  if constexpr (ACT == ACT_ANY) {
    if (g.act == ACT_SILU) return slope_all<ACT_SILU, V>(g, z);
    if (g.act == ACT_GELU) return slope_all<ACT_GELU, V>(g, z);
    if (g.act == ACT_RELU) return slope_all<ACT_RELU, V>(g, z);
    return slope_all<ACT_NONE, V>(g, z);
  } else if constexpr (ACT == ACT_SILU && V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      // s (1 + z (1 - s)) = s + (z s) (1 - s)
      const float2 v = make_float2(z[i], z[i + 1]), s = sigmoid2(v);
      const float2 zs = __fmul2_rn(v, s);
      const float2 r = __ffma2_rn(make_float2(-s.x, -s.y), zs, __fadd2_rn(s, zs));
      z[i] = r.x;
      z[i + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = act_slope<ACT>(z[i]);
  }
}

// r = a b + c of V values; Nb, Nc: 1 where b, c are one value for all
template <int V, int Nb = V, int Nc = V>
__device__ __forceinline__ void fma_all(const float* a, const float* b, const float* c, float* r) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const int j = Nb == 1 ? 0 : i, j1 = Nb == 1 ? 0 : i + 1, k = Nc == 1 ? 0 : i, k1 = Nc == 1 ? 0 : i + 1;
      const float2 t = __ffma2_rn(make_float2(a[i], a[i + 1]), make_float2(b[j], b[j1]), make_float2(c[k], c[k1]));
      r[i] = t.x;
      r[i + 1] = t.y;
    }
  } else {
    r[0] = fmaf(a[0], b[0], c[0]);
  }
}
template <int V>
__device__ __forceinline__ void mul_all(const float* a, const float* b, float* r) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 t = __fmul2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
      r[i] = t.x;
      r[i + 1] = t.y;
    }
  } else {
    r[0] = a[0] * b[0];
  }
}

// The group of channel c0 + i: one division for a thread's vector when the groups are whole
// vectors.
__device__ __forceinline__ int group_of(const NormGeom& g, int c0, int i) {
  return g.whole ? c0 / g.cpg : (c0 + i) / g.cpg;
}

// What a thread needs of its channels: z = x sc + sh (one rounding; sh holds b - mean sc,
// whose rounding is that of the mean itself).
template <int V>
struct Channels {
  float sc[V], sh[V];
  __device__ __forceinline__ void load(const NormGeom& g, const float2* stats, int first_group, int c0,
                                       const float* weight, const float* bias) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = c0 + i;
      const float2 st = stats[group_of(g, c0, i) - first_group];
      sc[i] = st.y * (weight ? weight[c] : 1.f);
      sh[i] = fmaf(-st.x, sc[i], bias ? bias[c] : 0.f);
    }
  }
  __device__ __forceinline__ void z(const float* x, float* out) const {
    fma_all<V>(x, sc, sh, out);
  }
};
// xh = x rs + mr of the same channels, for the gradient. Vectors of 8 lie in one group (the
// gradient takes narrower ones where groups are not multiples of 8 wide), so one value each.
template <int V>
struct Hats {
  static constexpr int kN = V == 8 ? 1 : V;
  float rs[kN], mr[kN];
  __device__ __forceinline__ void load(const NormGeom& g, const float2* stats, int first_group, int c0) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const float2 st = stats[group_of(g, c0, i) - first_group];
      rs[i] = st.y;
      mr[i] = -st.x * st.y;
    }
  }
  __device__ __forceinline__ void of(const float* x, float* out) const { fma_all<V, kN, kN>(x, rs, mr, out); }
};

// A block's sums of two values per channel over its row lanes. Every thread leaves its V
// channels' sums; (segment, channel) threads add some lanes each; `at` adds the segments.
// Memory: [lanes][channels] of each value, then [segments][channels] of each.
template <int V, int T>
struct BlockSums {
  __host__ __device__ static int floats(int tc) { return 2 * V * T + 2 * (tc * V > T ? tc * V : T); }
  float *a, *b, *sa, *sb;
  int channels, segs;
  __device__ __forceinline__ void add(float* mem, const NormGeom& g, const float* va, const float* vb, int lane) {
    channels = g.tc * V;
    segs = min(g.rp, T / channels);
    segs = segs < 1 ? 1 : segs;
    a = mem;
    b = mem + V * T;
    sa = mem + 2 * V * T;
    sb = sa + max(T, channels);
    const int t = threadIdx.x - lane * g.tc;
    if (lane < g.rp) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        a[lane * channels + t * V + i] = va[i];
        b[lane * channels + t * V + i] = vb[i];
      }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < segs * channels; k += T) {
      const int seg = k / channels, ch = k - seg * channels;
      float xa = 0.f, xb = 0.f;
      for (int r = seg; r < g.rp; r += segs) {
        xa += a[r * channels + ch];
        xb += b[r * channels + ch];
      }
      sa[k] = xa;
      sb[k] = xb;
    }
    __syncthreads();
  }
  __device__ __forceinline__ float2 at(int ch) const {
    float xa = 0.f, xb = 0.f;
    for (int k = 0; k < segs; ++k) {
      xa += sa[k * channels + ch];
      xb += sb[k * channels + ch];
    }
    return make_float2(xa, xb);
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d >= 1; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Mean and M2 of channels [lo, hi) of a chunk over `rows` rows, by one warp: the channels'
// means average to the group's, M2 = sum (M2_c + rows (mean_c - mean)^2). `far` is set where
// the sums about `first` lose too much of M2.
template <int V, int T>
__device__ __forceinline__ float2 group_moments(const BlockSums<V, T>& s, const float* first, int lo, int hi,
                                                float rows, bool& far) {
  const int lane = threadIdx.x & 31;
  const float inv = rows > 0.f ? 1.f / rows : 0.f;
  float mean = 0.f;
  for (int ch = lo + lane; ch < hi; ch += 32) mean += first[ch] + s.at(ch).x * inv;
  mean = warp_sum(mean) / (float)(hi - lo);
  float m2 = 0.f, sq = 0.f;
  for (int ch = lo + lane; ch < hi; ch += 32) {
    const float2 v = s.at(ch);
    const float d = first[ch] + v.x * inv - mean, own = v.y - v.x * v.x * inv;
    m2 += (own < 0.f ? 0.f : own) + rows * d * d;  // (a NaN stays)
    sq += v.y;
  }
  m2 = warp_sum(m2);
  sq = warp_sum(sq);
  far |= sq > NORM_FAR * m2;
  return make_float2(mean, m2);
}

// Whether any thread of the block found a group's sums too far off; then K of the chunk's
// channels becomes their mean.
template <int V, int T>
__device__ __forceinline__ bool recentre(const BlockSums<V, T>& s, float* first, float rows, bool far) {
  if (!__syncthreads_or(far)) return false;
  for (int ch = threadIdx.x; ch < s.channels; ch += T) first[ch] += s.at(ch).x / rows;
  __syncthreads();
  return true;
}

// The channels' K from `many` rows, `stride` elements apart.
template <typename T, int V>
__device__ __forceinline__ void middle_of_rows(const T* src, long stride, long many, float* k) {
  Pack<T, V> a, b, c;
  a.load(src);
  b.load(src + many / 2 * stride);
  c.load(src + (many - 1) * stride);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float x = to_f32(a.v[i]), y = to_f32(b.v[i]), z = to_f32(c.v[i]);
    k[i] = fmaxf(fminf(x, y), fminf(fmaxf(x, y), z));
  }
}

// s += v - k, q += (v - k)^2; two channels an instruction where there are two
template <int V>
__device__ __forceinline__ void add_moments(const float* v, const float* k, float* s, float* q) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 d = __fadd2_rn(make_float2(v[i], v[i + 1]), make_float2(-k[i], -k[i + 1]));
      add2_f32x2(s + i, d.x, d.y);
      const float2 e = __ffma2_rn(d, d, make_float2(q[i], q[i + 1]));
      q[i] = e.x;
      q[i + 1] = e.y;
    }
  } else {
    const float d = v[0] - k[0];
    s[0] += d;
    q[0] = fmaf(d, d, q[0]);
  }
}

// A thread's vectors of successive rows, copied ahead into its own places of a ring in shared
// memory (cp.async: no registers wait for them, no barrier since nobody else reads them).
// Plain loads, two rows a thread in flight, left the pass waiting for memory at 2/3 of its
// rate. `Tensors` streams of the same rows run together. Vectors under 4 bytes are loaded
// when they are used.
template <typename T, int V, int Tensors, int Threads>
struct RowStream {
  static constexpr int kBytes = V * (int)sizeof(T), kRows = 2;          // rows of a group
  static constexpr int kGroups = kBytes * Tensors > 16 ? 2 : 4;         // groups in flight: 64 KB a block at most
  static constexpr bool kAsync = kBytes >= 4;
  static constexpr int kSmem = kAsync ? kGroups * kRows * Tensors * Threads * kBytes : 0;
  unsigned char* mine;
  const T* src[Tensors];  // of the thread's next row to copy
  long step[Tensors];
  long left;              // rows still to copy
  int put, get;
  __device__ __forceinline__ void place(long k, int t, unsigned char*& at, int group) {
    at = mine + ((group * kRows + (int)k) * Tensors + t) * (Threads * kBytes);
  }
  __device__ __forceinline__ void fetch() {
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (left > 0) {
#pragma unroll
        for (int t = 0; t < Tensors; ++t) {
          unsigned char* at;
          place(k, t, at, put);
          if constexpr (kBytes == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(at)), "l"(src[t]) : "memory");
          else
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(at)), "l"(src[t]), "n"(kBytes)
                         : "memory");
          src[t] += step[t];
        }
        --left;
      }
    }
    cp_async_commit();
    put = put + 1 == kGroups ? 0 : put + 1;
  }
  // `n` rows from `first` on, `step` elements apart
  __device__ __forceinline__ void start(void* ring, long n) {
    mine = static_cast<unsigned char*>(ring) + threadIdx.x * kBytes;
    left = n;
    put = get = 0;
    if constexpr (kAsync) {
#pragma unroll
      for (int k = 0; k + 1 < kGroups; ++k) fetch();
    }
  }
  // The next group's rows, `n` of them wanted (the rest of `a` is not touched).
  __device__ __forceinline__ void next(int n, Pack<T, V> (*a)[Tensors]) {
    if constexpr (kAsync) {
      fetch();
      asm volatile("cp.async.wait_group %0;" ::"n"(kGroups - 1) : "memory");
#pragma unroll
      for (int k = 0; k < kRows; ++k)
        if (k < n) {
#pragma unroll
          for (int t = 0; t < Tensors; ++t) {
            unsigned char* at;
            place(k, t, at, get);
            a[k][t] = *reinterpret_cast<const Pack<T, V>*>(at);
          }
        }
      get = get + 1 == kGroups ? 0 : get + 1;
    } else {
#pragma unroll
      for (int k = 0; k < kRows; ++k)
        if (k < n) {
#pragma unroll
          for (int t = 0; t < Tensors; ++t) {
            a[k][t].load(src[t]);
            src[t] += step[t];
          }
        }
    }
  }
};

// Split s of a picture takes rp rows of every rp * splits: all blocks together walk through
// memory side by side (a range of rows for each block was 10 % slower on maps past L2).
// How many rows that is.
__device__ __forceinline__ float norm_rows(const NormGeom& g, int s) {
  const long rest = g.l - g.cycles * g.rp * g.splits - (long)s * g.rp;
  return (float)(g.cycles * g.rp + (rest <= 0 ? 0 : rest < g.rp ? rest : g.rp));
}

// A block's place: picture, split, chunk, its thread's vector and row lane.
struct NormPlace {
  long pic, first, step;  // the thread's first row, from one of its rows to the next
  int split, chunk, col, lane;
  bool on;
  int c0, c1;  // the chunk's channels
  __device__ __forceinline__ NormPlace(const NormGeom& g, int vec) {
    pic = blockIdx.x / g.splits;
    split = (int)(blockIdx.x % g.splits);
    chunk = blockIdx.y;
    lane = threadIdx.x / g.tc;
    col = chunk * g.tc + threadIdx.x - lane * g.tc;
    on = lane < g.rp && col < g.cols;
    first = split * g.rp + lane;
    step = (long)g.rp * g.splits;
    c0 = chunk * g.tc * vec;
    c1 = min(c0 + g.tc * vec, g.c);
  }
  // the thread's rows
  __device__ __forceinline__ long mine(const NormGeom& g) const {
    const long most = g.cycles + (first + g.cycles * step < g.l);
    return on ? most : 0;
  }
};

// A block's sums about `first` joined to the mean and M2 of its part of every group of its chunk;
// whether `first` is too far from the means (in some thread).
template <int V>
__device__ __forceinline__ bool norm_partials(const NormGeom& g, const NormPlace& p,
                                              const BlockSums<V, NORM_THREADS>& sums, const float* first,
                                              float2* part) {
  bool far = false;
  float2* out = part + (p.pic * g.splits + p.split) * g.slots + p.chunk;
  for (int grp = p.c0 / g.cpg + (threadIdx.x >> 5); grp * g.cpg < p.c1; grp += NORM_THREADS / 32) {
    const float2 m = group_moments(sums, first, max(grp * g.cpg, p.c0) - p.c0, min((grp + 1) * g.cpg, p.c1) - p.c0,
                                   norm_rows(g, p.split), far);
    if ((threadIdx.x & 31) == 0) out[grp] = m;
  }
  return far;
}

// The block's sums once more, about `first`, for which it has moved. (Rare, and a function of its
// own, so that it takes no registers from the first time, which would spill.)
template <typename T, int V>
__device__ __noinline__ void norm_stats_again(const T* x, float2* part, const NormGeom& g, float* mem) {
  const NormPlace p(g, V);
  const float* first = mem + g.keep;
  float k[V], sum[V], sq[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    k[i] = first[(threadIdx.x - p.lane * g.tc) * V + i];
    sum[i] = sq[i] = 0.f;
  }
  const T* src = x + p.pic * g.x_sn + p.first * g.x_sl + (long)p.col * V;
  for (long n = p.mine(g); n > 0; --n, src += p.step * g.x_sl) {
    Pack<T, V> a;
    float v[V];
    a.load(src);
    unpack(a, v);
    add_moments<V>(v, k, sum, sq);
  }
  BlockSums<V, NORM_THREADS> sums;
  sums.add(mem, g, sum, sq, p.lane);
  norm_partials<V>(g, p, sums, first, part);
}

// First pass: per (picture, split, chunk's part of a group) mean and M2.
template <typename T, int V>
__global__ void __launch_bounds__(NORM_THREADS, 2)
norm_stats_kernel(const T* __restrict__ x, float2* __restrict__ part, const __grid_constant__ NormGeom g) {
  extern __shared__ __align__(16) float norm_sm[];
  let_next_start();
  const NormPlace p(g, V);
  float k[V], sum[V], sq[V];
#pragma unroll
  for (int i = 0; i < V; ++i) k[i] = sum[i] = sq[i] = 0.f;
  float* first = norm_sm + g.keep;  // K of the chunk's channels, behind the ring and, later, the sums
  if (p.on && p.first - p.lane < g.l) {
    const T* src = x + p.pic * g.x_sn + (long)p.col * V;
    using Stream = RowStream<T, V, 1, NORM_THREADS>;
    Stream rows;
    long n = p.mine(g);
    rows.src[0] = src + p.first * g.x_sl;
    rows.step[0] = p.step * g.x_sl;
    rows.start(norm_sm, n);
    // of the block's rows of lane 0: the same K for every lane
    const long top = p.first - p.lane, many = g.cycles + (top + g.cycles * p.step < g.l);
    middle_of_rows<T, V>(src + top * g.x_sl, p.step * g.x_sl, many, k);
    for (; n > 0; n -= Stream::kRows) {
      Pack<T, V> a[Stream::kRows][1];
      const int now = n < Stream::kRows ? (int)n : Stream::kRows;
      rows.next(now, a);
#pragma unroll
      for (int r = 0; r < Stream::kRows; ++r) {
        if (r >= now) break;
        float v[V];
        unpack(a[r][0], v);
        add_moments<V>(v, k, sum, sq);
      }
    }
  }
  if (p.lane == 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) first[threadIdx.x * V + i] = k[i];
  }
  __syncthreads();  // the sums lie over the ring
  BlockSums<V, NORM_THREADS> sums;
  sums.add(norm_sm, g, sum, sq, p.lane);
  const bool far = norm_partials<V>(g, p, sums, first, part);
  if (recentre(sums, first, norm_rows(g, p.split), far)) norm_stats_again<T, V>(x, part, g, norm_sm);
}

// Partials s0, s0 + 32, ... of a picture's slot, all on their way at once.
constexpr int kJoinBatch = 10;
__device__ __forceinline__ void load_partials(const NormGeom& g, const float2* part, long pic, int slot, int s0,
                                              float2* v) {
#pragma unroll
  for (int b = 0; b < kJoinBatch; ++b)
    if (s0 + 32 * b < g.splits) v[b] = __ldcg(part + (pic * g.splits + s0 + 32 * b) * g.slots + slot);
}

// A picture's group, joined over splits (and chunks) by one warp: (mean, rstd).
__device__ __forceinline__ float2 norm_join(const NormGeom& g, const float2* part, long pic, int grp, int vec) {
  const int per = g.tc * vec;  // channels of a chunk
  const int k0 = grp * g.cpg / per, k1 = ((grp + 1) * g.cpg - 1) / per;
  Moments m{0.f, 0.f, 0.f};
  for (int k = k0; k <= k1; ++k) {
    const float width = (float)(min((grp + 1) * g.cpg, (k + 1) * per) - max(grp * g.cpg, k * per));
    for (int s0 = threadIdx.x & 31; s0 < g.splits; s0 += 32 * kJoinBatch) {
      float2 v[kJoinBatch];
      load_partials(g, part, pic, grp + k, s0, v);
#pragma unroll
      for (int b = 0; b < kJoinBatch; ++b)
        if (s0 + 32 * b < g.splits) m = join(m, Moments{norm_rows(g, s0 + 32 * b) * width, v[b].x, v[b].y});
    }
  }
  m = warp_join(m);
  return make_float2(m.mean, 1.f / sqrtf((m.n > 0.f ? m.m2 / m.n : 0.f) + g.eps));
}

// Second pass: y = act((x - mean) rstd w + b).
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(NORM_THREADS, 2)
norm_apply_kernel(const T* x, T* y, const float2* __restrict__ part,
                  float* __restrict__ mean, float* __restrict__ rstd, const float* __restrict__ weight,
                  const float* __restrict__ bias, const __grid_constant__ NormGeom g) {
  extern __shared__ __align__(16) float2 norm_stat[];  // of the chunk's groups
  const NormPlace p(g, V);
  const int g0 = p.c0 / g.cpg;
  // x does not come from the pass before: its first rows are on their way while the partials
  // are waited for and joined
  using Stream = RowStream<T, V, 1, NORM_THREADS>;
  Stream rows;
  long n = p.mine(g);
  rows.src[0] = x + p.pic * g.x_sn + p.first * g.x_sl + (long)p.col * V;
  rows.step[0] = p.step * g.x_sl;
  rows.start(reinterpret_cast<float*>(norm_stat) + g.keep, n);
  wait_for_previous();
  for (int grp = g0 + (threadIdx.x >> 5); grp * g.cpg < p.c1; grp += NORM_THREADS / 32) {
    const float2 s = norm_join(g, part, p.pic, grp, V);
    if ((threadIdx.x & 31) == 0) {
      norm_stat[grp - g0] = s;
      if (p.split == 0 && grp * g.cpg >= p.c0) {  // the chunk that holds the group's start
        if (mean) mean[p.pic * g.groups + grp] = s.x;
        if (rstd) rstd[p.pic * g.groups + grp] = s.y;
      }
    }
  }
  __syncthreads();
  if (!n) return;
  Channels<V> ch;
  ch.load(g, norm_stat, g0, p.col * V, weight, bias);
  T* dst = y + p.pic * g.y_sn + p.first * g.y_sl + (long)p.col * V;
  for (; n > 0; n -= Stream::kRows) {
    Pack<T, V> a[Stream::kRows][1];
    const int now = n < Stream::kRows ? (int)n : Stream::kRows;
    rows.next(now, a);
#pragma unroll
    for (int r = 0; r < Stream::kRows; ++r) {
      if (r >= now) break;
      float v[V];
      unpack(a[r][0], v);
      ch.z(v, v);
      act_all<ACT, V>(g, v);
      repack<T, V>(v).store(dst);
      dst += p.step * g.y_sl;
    }
  }
}

// gz = dy act'(z) of V values.
template <int ACT, int V>
__device__ __forceinline__ void grad_z(const NormGeom& g, const Channels<V>& ch, const float* x, const float* dy,
                                       float* gz) {
  ch.z(x, gz);
  slope_all<ACT, V>(g, gz);
  mul_all<V>(gz, dy, gz);
}

// (mean, rstd) of the chunk's groups into shared memory.
__device__ __forceinline__ void grad_stats(const NormGeom& g, float2* stats, int g0, int c1, const float* mean,
                                           const float* rstd, long pic) {
  for (int grp = g0 + threadIdx.x; grp * g.cpg < c1; grp += blockDim.x)
    stats[grp - g0] = make_float2(mean[pic * g.groups + grp], rstd[pic * g.groups + grp]);
}

template <typename T, int V, int ACT>
__device__ __forceinline__ void add_grad(const NormGeom& g, const Channels<V>& ch, const Hats<V>& hat,
                                         const Pack<T, V>& a, const Pack<T, V>& e, float* sa, float* sb) {
  float v[V], d[V], gz[V];
  unpack(a, v);
  unpack(e, d);
  grad_z<ACT, V>(g, ch, v, d, gz);
  hat.of(v, v);
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) add2_f32x2(sa + i, gz[i], gz[i + 1]);
  } else {
    sa[0] += gz[0];
  }
  fma_all<V>(gz, v, sb, sb);
}

// First pass of the gradient: per (picture, split) the channels' sums of gz and gz xh for dw
// and db, and the parts of the groups' sums of h and h xh.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(NORM_THREADS, norm_grad_blocks(V))
norm_grad_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean,
                      const float* __restrict__ rstd, const float* __restrict__ weight,
                      const float* __restrict__ bias, float2* __restrict__ part, float2* __restrict__ cpart,
                      const __grid_constant__ NormGeom g) {
  extern __shared__ __align__(16) float norm_sm[];  // the ring, then the block's sums; the groups' statistics
  let_next_start();
  const NormPlace p(g, V);
  const int g0 = p.c0 / g.cpg;
  float2* stats = reinterpret_cast<float2*>(norm_sm + g.keep);
  grad_stats(g, stats, g0, p.c1, mean, rstd, p.pic);
  __syncthreads();
  float sa[V], sb[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sa[i] = sb[i] = 0.f;
  if (p.on) {
    Channels<V> ch;
    Hats<V> hat;
    ch.load(g, stats, g0, p.col * V, weight, bias);
    hat.load(g, stats, g0, p.col * V);
    using Stream = RowStream<T, V, 2, NORM_THREADS>;
    Stream rows;
    long n = p.mine(g);
    rows.src[0] = x + p.pic * g.x_sn + p.first * g.x_sl + (long)p.col * V;
    rows.src[1] = dy + p.pic * g.d_sn + p.first * g.d_sl + (long)p.col * V;
    rows.step[0] = p.step * g.x_sl;
    rows.step[1] = p.step * g.d_sl;
    rows.start(norm_sm, n);
    for (; n > 0; n -= Stream::kRows) {
      Pack<T, V> a[Stream::kRows][2];
      const int now = n < Stream::kRows ? (int)n : Stream::kRows;
      rows.next(now, a);
#pragma unroll
      for (int r = 0; r < Stream::kRows; ++r) {
        if (r >= now) break;
        add_grad<T, V, ACT>(g, ch, hat, a[r][0], a[r][1], sa, sb);
      }
    }
  }
  __syncthreads();  // the sums lie over the ring
  BlockSums<V, NORM_THREADS> sums;
  sums.add(norm_sm, g, sa, sb, p.lane);
  float2* out = part + (p.pic * g.splits + p.split) * g.slots + p.chunk;
  float2* cout = cpart + (p.pic * g.splits + p.split) * g.c;
  for (int grp = g0 + (threadIdx.x >> 5); grp * g.cpg < p.c1; grp += NORM_THREADS / 32) {
    float2 m = make_float2(0.f, 0.f);
    for (int c = max(grp * g.cpg, p.c0) + (threadIdx.x & 31); c < min((grp + 1) * g.cpg, p.c1); c += 32) {
      const float2 s = sums.at(c - p.c0);
      cout[c] = s;
      const float w = weight ? weight[c] : 1.f;
      m = join(m, make_float2(w * s.x, w * s.y));
    }
    m = warp_join(m);
    if ((threadIdx.x & 31) == 0) out[grp] = m;
  }
}

// (E[h], E[h xh]) of a picture's group, joined by one warp.
__device__ __forceinline__ float2 norm_grad_join(const NormGeom& g, const float2* part, long pic, int grp, int vec) {
  const int per = g.tc * vec, k0 = grp * g.cpg / per, k1 = ((grp + 1) * g.cpg - 1) / per;
  float2 m = make_float2(0.f, 0.f);
  for (int k = k0; k <= k1; ++k)
    for (int s0 = threadIdx.x & 31; s0 < g.splits; s0 += 32 * kJoinBatch) {
      float2 v[kJoinBatch];
      load_partials(g, part, pic, grp + k, s0, v);
#pragma unroll
      for (int b = 0; b < kJoinBatch; ++b)
        if (s0 + 32 * b < g.splits) m = join(m, v[b]);
    }
  m = warp_join(m);
  const float inv = 1.f / ((float)g.l * (float)g.cpg);
  return make_float2(m.x * inv, m.y * inv);
}

// dx = gz sc - rs E[h] - xh rs E[h xh] of one vector (sc = rs w).
template <int V>
struct GradMeans {
  static constexpr int kN = Hats<V>::kN;
  float m1[kN], m2[kN];  // - rs E[h], - rs E[h xh]
  __device__ __forceinline__ void load(const NormGeom& g, const Hats<V>& hat, const float2* means, int first_group,
                                       int c0) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const float2 m = means[group_of(g, c0, i) - first_group];
      m1[i] = -hat.rs[i] * m.x;
      m2[i] = -hat.rs[i] * m.y;
    }
  }
};
template <typename T, int V, int ACT>
__device__ __forceinline__ Pack<T, V> grad_x(const NormGeom& g, const Channels<V>& ch, const Hats<V>& hat,
                                             const GradMeans<V>& m, const Pack<T, V>& a, const Pack<T, V>& e) {
  float v[V], d[V], gz[V];
  unpack(a, v);
  unpack(e, d);
  grad_z<ACT, V>(g, ch, v, d, gz);
  hat.of(v, v);
  fma_all<V, V, Hats<V>::kN>(gz, ch.sc, m.m1, gz);
  fma_all<V, Hats<V>::kN, V>(v, m.m2, gz, v);
  return repack<T, V>(v);
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(NORM_THREADS, norm_grad_blocks(V))
norm_grad_apply_kernel(const T* dy, const T* x, T* dx,
                       const float* __restrict__ mean, const float* __restrict__ rstd,
                       const float* __restrict__ weight, const float* __restrict__ bias,
                       const float2* __restrict__ part, const __grid_constant__ NormGeom g) {
  extern __shared__ __align__(16) float2 norm_stat[];  // (mean, rstd), then (E[h], E[h xh]) of the chunk's groups
  const NormPlace p(g, V);
  const int g0 = p.c0 / g.cpg, ng = (p.c1 - 1) / g.cpg - g0 + 1;
  using Stream = RowStream<T, V, 2, NORM_THREADS>;
  Stream rows;
  long n = p.mine(g);
  rows.src[0] = x + p.pic * g.x_sn + p.first * g.x_sl + (long)p.col * V;
  rows.src[1] = dy + p.pic * g.d_sn + p.first * g.d_sl + (long)p.col * V;
  rows.step[0] = p.step * g.x_sl;
  rows.step[1] = p.step * g.d_sl;
  rows.start(reinterpret_cast<float*>(norm_stat) + g.keep, n);
  grad_stats(g, norm_stat, g0, p.c1, mean, rstd, p.pic);
  wait_for_previous();
  for (int grp = g0 + (threadIdx.x >> 5); grp * g.cpg < p.c1; grp += NORM_THREADS / 32) {
    const float2 m = norm_grad_join(g, part, p.pic, grp, V);
    if ((threadIdx.x & 31) == 0) norm_stat[ng + grp - g0] = m;
  }
  __syncthreads();
  if (!n) return;
  Channels<V> ch;
  ch.load(g, norm_stat, g0, p.col * V, weight, bias);
  Hats<V> hat;
  GradMeans<V> m;
  hat.load(g, norm_stat, g0, p.col * V);
  m.load(g, hat, norm_stat + ng, g0, p.col * V);
  T* dst = dx + p.pic * g.y_sn + p.first * g.y_sl + (long)p.col * V;
  for (; n > 0; n -= Stream::kRows) {
    Pack<T, V> a[Stream::kRows][2];
    const int now = n < Stream::kRows ? (int)n : Stream::kRows;
    rows.next(now, a);
#pragma unroll
    for (int r = 0; r < Stream::kRows; ++r) {
      if (r >= now) break;
      grad_x<T, V, ACT>(g, ch, hat, m, a[r][0], a[r][1]).store(dst);
      dst += p.step * g.y_sl;
    }
  }
}

// dw and db from `parts` partials (pictures x splits): 32 neighbouring channels a block, 32
// threads each.
__global__ void __launch_bounds__(1024) norm_grad_params_kernel(const float2* __restrict__ cpart, long parts, int c,
                                                                float* __restrict__ dweight,
                                                                float* __restrict__ dbias) {
  __shared__ float2 sums[32][33];
  const int ch = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;
  float2 m = make_float2(0.f, 0.f);
  if (ch < c) {
#pragma unroll 4
    for (long k = lane; k < parts; k += 32) m = join(m, cpart[k * c + ch]);
  }
  sums[threadIdx.x & 31][lane] = m;
  __syncthreads();
  m = warp_join(sums[lane][threadIdx.x & 31]);
  const int mine = blockIdx.x * 32 + lane;
  if ((threadIdx.x & 31) == 0 && mine < c) {
    if (dbias) dbias[mine] = m.x;
    if (dweight) dweight[mine] = m.y;
  }
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The float2 at `p` of this block's shared memory, in the cluster's block `rank`.
__device__ __forceinline__ float2 cluster_read(const float2* p, int rank) {
  uint32_t a;
  float2 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}

// The small form: cluster (picture, chunk of whole groups), of `splits` blocks that take a
// range of the rows each; the chunk's values in shared memory; kT threads: 128 where the
// values are few, else 512. GRAD: x and dy, dx out; the channels' sums go to dw and db when
// there is one block of them, else to cpart.
template <typename T, int V, bool GRAD, int kT>
__global__ void __launch_bounds__(kT)
norm_small_kernel(const T* dy, const T* x, T* y, float* __restrict__ mean,
                  float* __restrict__ rstd, const float* __restrict__ weight, const float* __restrict__ bias,
                  float* __restrict__ dweight, float* __restrict__ dbias, float2* __restrict__ cpart,
                  const __grid_constant__ NormGeom g) {
  extern __shared__ __align__(16) float norm_sm[];
  // the block's sums; K; (mean, rstd), (E[h], E[h xh]), shared sums of the groups; the values
  float* first = norm_sm + BlockSums<V, kT>::floats(g.tc);
  float2* stats = reinterpret_cast<float2*>(first + (g.tc * V + 1) / 2 * 2);
  const NormPlace p(g, V);
  const int g0 = p.c0 / g.cpg, ng = (p.c1 - p.c0) / g.cpg;
  float2* share = stats + 2 * ng;  // what the cluster's blocks read of one another, by group
  Pack<T, V>* keep = reinterpret_cast<Pack<T, V>*>(norm_sm + g.keep);
  Pack<T, V>* keep_d = keep + (GRAD ? g.range * g.tc : 0);
  const int t = threadIdx.x - p.lane * g.tc;
  const long r0 = min(p.split * g.range, g.l), rows = min(g.range, g.l - r0);  // the block's
  const T* src = x + p.pic * g.x_sn + r0 * g.x_sl + (long)p.col * V;
  T* dst = y + p.pic * g.y_sn + r0 * g.y_sl + (long)p.col * V;
  const float inv = 1.f / ((float)g.l * (float)g.cpg);
  if constexpr (!GRAD) {
    float k[V], sum[V], sq[V];
#pragma unroll
    for (int i = 0; i < V; ++i) k[i] = sum[i] = sq[i] = 0.f;
    if (p.on && rows > 0) {
      Pack<T, V> a;
      float v[V];
      middle_of_rows<T, V>(src, g.x_sl, rows, k);
#pragma unroll 4
      for (long row = p.lane; row < rows; row += g.rp) {
        a.load(src + row * g.x_sl);
        keep[row * g.tc + t] = a;
        unpack(a, v);
        add_moments<V>(v, k, sum, sq);
      }
    }
    if (p.lane == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) first[t * V + i] = k[i];
    }
    BlockSums<V, kT> sums;
    for (bool again = false;; again = true) {  // twice where K turns out to be far from the mean
      sums.add(norm_sm, g, sum, sq, p.lane);
      bool far = false;
      for (int n = threadIdx.x >> 5; n < ng; n += kT / 32) {
        const float2 m = group_moments(sums, first, n * g.cpg, (n + 1) * g.cpg, (float)rows, far);
        if ((threadIdx.x & 31) == 0) share[n] = m;
      }
      if (again || !recentre(sums, first, (float)rows, far)) break;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        k[i] = first[t * V + i];
        sum[i] = sq[i] = 0.f;
      }
      for (long row = p.on ? p.lane : rows; row < rows; row += g.rp) {
        float v[V];
        unpack(keep[row * g.tc + t], v);
        add_moments<V>(v, k, sum, sq);
      }
    }
    g.splits > 1 ? cluster_sync() : __syncthreads();
    for (int n = threadIdx.x; n < ng; n += kT) {
      Moments m{0.f, 0.f, 0.f};
      for (int r = 0; r < g.splits; ++r) {
        const float2 v = g.splits > 1 ? cluster_read(share + n, r) : share[n];
        const long from = min(r * g.range, g.l);
        m = join(m, Moments{(float)min(g.range, g.l - from) * (float)g.cpg, v.x, v.y});
      }
      const float rs = 1.f / sqrtf((g.l > 0 ? m.m2 * inv : 0.f) + g.eps);
      stats[n] = make_float2(m.mean, rs);
      if (p.split == 0) {
        if (mean) mean[p.pic * g.groups + g0 + n] = m.mean;
        if (rstd) rstd[p.pic * g.groups + g0 + n] = rs;
      }
    }
    __syncthreads();
    if (p.on) {
      Channels<V> ch;
      ch.load(g, stats, g0, p.col * V, weight, bias);
      for (long row = p.lane; row < rows; row += g.rp) {
        float v[V];
        unpack(keep[row * g.tc + t], v);
        ch.z(v, v);
        act_all<ACT_ANY, V>(g, v);
        repack<T, V>(v).store(dst + row * g.y_sl);
      }
    }
  } else {
    const T* del = dy + p.pic * g.d_sn + r0 * g.d_sl + (long)p.col * V;
    grad_stats(g, stats, g0, p.c1, mean, rstd, p.pic);
    __syncthreads();
    Channels<V> ch;
    Hats<V> hat;
    float sa[V], sb[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sa[i] = sb[i] = 0.f;
    if (p.on) {
      ch.load(g, stats, g0, p.col * V, weight, bias);
      hat.load(g, stats, g0, p.col * V);
#pragma unroll 2
      for (long row = p.lane; row < rows; row += g.rp) {
        Pack<T, V> a, e;
        a.load(src + row * g.x_sl);
        e.load(del + row * g.d_sl);
        keep[row * g.tc + t] = a;
        keep_d[row * g.tc + t] = e;
        add_grad<T, V, ACT_ANY>(g, ch, hat, a, e, sa, sb);
      }
    }
    BlockSums<V, kT> sums;
    sums.add(norm_sm, g, sa, sb, p.lane);
    float2* means = stats + ng;
    for (int k = threadIdx.x >> 5; k < ng; k += kT / 32) {
      float2 m = make_float2(0.f, 0.f);
      for (int e = k * g.cpg + (threadIdx.x & 31); e < (k + 1) * g.cpg; e += 32) {
        const int c = p.c0 + e;
        const float2 s = sums.at(e);
        const float w = weight ? weight[c] : 1.f;
        m = join(m, make_float2(w * s.x, w * s.y));
        if (cpart) {
          cpart[(long)blockIdx.x * g.c + c] = s;
        } else {
          if (dbias) dbias[c] = s.x;
          if (dweight) dweight[c] = s.y;
        }
      }
      m = warp_join(m);
      if ((threadIdx.x & 31) == 0) share[k] = m;
    }
    g.splits > 1 ? cluster_sync() : __syncthreads();
    for (int k = threadIdx.x; k < ng; k += kT) {
      float2 m = make_float2(0.f, 0.f);
      for (int r = 0; r < g.splits; ++r) m = join(m, g.splits > 1 ? cluster_read(share + k, r) : share[k]);
      means[k] = make_float2(m.x * inv, m.y * inv);
    }
    __syncthreads();
    if (p.on) {
      GradMeans<V> m;
      m.load(g, hat, means, g0, p.col * V);
      for (long row = p.lane; row < rows; row += g.rp)
        grad_x<T, V, ACT_ANY>(g, ch, hat, m, keep[row * g.tc + t], keep_d[row * g.tc + t]).store(dst + row * g.y_sl);
    }
  }
  if (g.splits > 1) cluster_sync();  // the others may still be reading this block's sums
}

}  // namespace scb
