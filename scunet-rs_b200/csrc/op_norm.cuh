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
//  * norm_small_kernel: a picture's rows of a few whole groups fit in one block's shared
//    memory; the values are read once, one launch.
//  * norm_stats_kernel, then norm_apply_kernel (norm_grad_sums_kernel, then
//    norm_grad_apply_kernel): blocks take row ranges of all pictures and leave one partial
//    per group; the second launch starts while the first one ends, every block joins its
//    picture's partials itself, and walks its rows backwards, so that what the first pass
//    read last is still in L2.
// A thread keeps its channels (a vector of up to 16 bytes) and steps over rows.
//
// Statistics are fp32: a block sums x - K and (x - K)^2 with K the median of the channel's
// values in its first, middle and last row, so that the sum of squares loses nothing to a
// large mean or to one value far from the rest, and (count, mean, M2) triples are joined,
//   M2 = M2a + M2b + (mb - ma)^2 na nb / (na + nb).
// No atomics: the order of every sum is fixed by the sizes.
#pragma once
#include "ops_common.cuh"

namespace scb {

struct NormGeom {
  long n, l;          // pictures, rows of each
  long first;         // first picture of the launch
  int c, groups, cpg; // channels, groups, channels per group
  int cols;           // vectors of a row
  int tc, rp;         // vectors of a row that one block takes (a chunk), rows it takes at once
  int chunks, slots;  // chunks of a row; groups + chunks - 1 partials of a split: a chunk's
                      // part of a group is slot group + chunk (a group may span chunks)
  int splits;         // row ranges of a picture
  int whole;          // a vector never spans two groups
  long x_sn, x_sl;    // element strides of pictures and rows
  long y_sn, y_sl;
  long d_sn, d_sl;    // dy
  float eps;
  int act;            // read by the kernels compiled for ACT_ANY
  int keep;           // small form: where the values start in shared memory, in floats
};

constexpr int NORM_THREADS = 512;  // two blocks an SM: every block reads its picture's partials

struct Moments {
  float n, mean, m2;
};
__device__ __forceinline__ Moments join(const Moments& a, const Moments& b) {
  const float n = a.n + b.n;
  if (n == 0.f) return a;
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

// Activations of V values. SiLU takes one reciprocal for two values (1/a = b / (ab)): the
// special function unit, at two operations a value, would bound the pass; e^-z is capped at
// 2^60, where the product stays finite and z sigmoid(z) is 0 to 1e-17.
template <int ACT, int V>
__device__ __forceinline__ void sigmoids(const float* z, float* s) {
#pragma unroll
  for (int i = 0; i < V; i += 2) {
    const float a = 1.f + ex2_approx(fminf(z[i] * -1.4426950408889634f, 60.f));
    if (i + 1 < V) {
      const float b = 1.f + ex2_approx(fminf(z[i + 1] * -1.4426950408889634f, 60.f));
      const float r = rcp_approx(a * b);
      s[i] = b * r;
      s[i + 1] = a * r;
    } else {
      s[i] = rcp_approx(a);
    }
  }
}
template <int ACT, int V>
__device__ __forceinline__ void act_all(const NormGeom& g, float* z) {
  if (ACT == ACT_SILU) {
    float s[V];
    sigmoids<ACT, V>(z, s);
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] *= s[i];
  } else if (ACT == ACT_ANY) {
    if (g.act == ACT_SILU) return act_all<ACT_SILU, V>(g, z);
    if (g.act == ACT_GELU) return act_all<ACT_GELU, V>(g, z);
    if (g.act == ACT_RELU) return act_all<ACT_RELU, V>(g, z);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = act_fwd<ACT>(z[i]);
  }
}
// z -> act'(z)
template <int ACT, int V>
__device__ __forceinline__ void slope_all(const NormGeom& g, float* z) {
  if (ACT == ACT_SILU) {
    float s[V];
    sigmoids<ACT, V>(z, s);
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = s[i] * (1.f + z[i] * (1.f - s[i]));
  } else if (ACT == ACT_ANY) {
    if (g.act == ACT_SILU) return slope_all<ACT_SILU, V>(g, z);
    if (g.act == ACT_GELU) return slope_all<ACT_GELU, V>(g, z);
    if (g.act == ACT_RELU) return slope_all<ACT_RELU, V>(g, z);
    return slope_all<ACT_NONE, V>(g, z);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = act_slope<ACT>(z[i]);
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
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = fmaf(x[i], sc[i], sh[i]);
  }
};
// xh = x rs + mr of the same channels, for the gradient.
template <int V>
struct Hats {
  float rs[V], mr[V];
  __device__ __forceinline__ void load(const NormGeom& g, const float2* stats, int first_group, int c0) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 st = stats[group_of(g, c0, i) - first_group];
      rs[i] = st.y;
      mr[i] = -st.x * st.y;
    }
  }
  __device__ __forceinline__ float at(int i, float x) const { return fmaf(x, rs[i], mr[i]); }
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
// means average to the group's, M2 = sum (M2_c + rows (mean_c - mean)^2).
template <int V, int T>
__device__ __forceinline__ float2 group_moments(const BlockSums<V, T>& s, const float* first, int lo, int hi,
                                                float rows) {
  const int lane = threadIdx.x & 31;
  const float inv = rows > 0.f ? 1.f / rows : 0.f;
  float mean = 0.f;
  for (int ch = lo + lane; ch < hi; ch += 32) mean += first[ch] + s.at(ch).x * inv;
  mean = warp_sum(mean) / (float)(hi - lo);
  float m2 = 0.f;
  for (int ch = lo + lane; ch < hi; ch += 32) {
    const float2 v = s.at(ch);
    const float d = first[ch] + v.x * inv - mean, own = v.y - v.x * v.x * inv;
    m2 += (own < 0.f ? 0.f : own) + rows * d * d;  // (a NaN stays)
  }
  return make_float2(mean, warp_sum(m2));
}

// The channels' K for rows [r0, r1) of a block.
template <typename T, int V>
__device__ __forceinline__ void middle_of_rows(const T* src, long stride, long r0, long r1, float* k) {
  Pack<T, V> a, b, c;
  a.load(src + r0 * stride);
  b.load(src + (r0 + (r1 - r0) / 2) * stride);
  c.load(src + (r1 - 1) * stride);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float x = to_f32(a.v[i]), y = to_f32(b.v[i]), z = to_f32(c.v[i]);
    k[i] = fmaxf(fminf(x, y), fminf(fmaxf(x, y), z));
  }
}

// s += v - k, q += (v - k)^2
template <int V>
__device__ __forceinline__ void add_moments(const float* v, const float* k, float* s, float* q) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float d = v[i] - k[i];
    s[i] += d;
    q[i] = fmaf(d, d, q[i]);
  }
}

// The row range of split s.
__device__ __forceinline__ void norm_rows(const NormGeom& g, int s, long& r0, long& r1) {
  r0 = g.l * s / g.splits;
  r1 = g.l * (s + 1) / g.splits;
}

// A block's place: picture, split, chunk, its thread's vector and row lane.
struct NormPlace {
  long pic, r0, r1;
  int split, chunk, col, lane;
  bool on;
  int c0, c1;  // the chunk's channels
  __device__ __forceinline__ NormPlace(const NormGeom& g, int vec) {
    pic = g.first + blockIdx.x / g.splits;
    split = (int)(blockIdx.x % g.splits);
    chunk = blockIdx.y;
    col = chunk * g.tc + threadIdx.x % g.tc;
    lane = threadIdx.x / g.tc;
    on = lane < g.rp && col < g.cols;
    norm_rows(g, split, r0, r1);
    c0 = chunk * g.tc * vec;
    c1 = min(c0 + g.tc * vec, g.c);
  }
};

// Launch order of the two passes (programmatic dependent launch): the first lets the second
// start early, the second waits for the first's results before it reads or writes anything.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

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
  float* first = norm_sm + BlockSums<V, NORM_THREADS>::floats(g.tc);  // K of the chunk's channels
  if (p.on && p.r0 < p.r1) {
    const T* src = x + p.pic * g.x_sn + (long)p.col * V;
    Pack<T, V> a;
    float v[V];
    middle_of_rows<T, V>(src, g.x_sl, p.r0, p.r1, k);
#pragma unroll 4
    for (long row = p.r0 + p.lane; row < p.r1; row += g.rp) {
      a.load(src + row * g.x_sl);
      unpack(a, v);
      add_moments<V>(v, k, sum, sq);
    }
  }
  if (p.lane == 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) first[threadIdx.x * V + i] = k[i];
  }
  BlockSums<V, NORM_THREADS> sums;
  sums.add(norm_sm, g, sum, sq, p.lane);
  float2* out = part + (p.pic * g.splits + p.split) * g.slots + p.chunk;
  for (int grp = p.c0 / g.cpg + (threadIdx.x >> 5); grp * g.cpg < p.c1; grp += NORM_THREADS / 32) {
    const float2 m = group_moments(sums, first, max(grp * g.cpg, p.c0) - p.c0, min((grp + 1) * g.cpg, p.c1) - p.c0,
                                   (float)(p.r1 - p.r0));
    if ((threadIdx.x & 31) == 0) out[grp] = m;
  }
}

// A picture's group, joined over splits (and chunks) by one warp: (mean, rstd).
__device__ __forceinline__ float2 norm_join(const NormGeom& g, const float2* part, long pic, int grp, int vec) {
  const int per = g.tc * vec;  // channels of a chunk
  const int k0 = grp * g.cpg / per, k1 = ((grp + 1) * g.cpg - 1) / per;
  Moments m{0.f, 0.f, 0.f};
  for (int s = threadIdx.x & 31; s < g.splits; s += 32) {
    long r0, r1;
    norm_rows(g, s, r0, r1);
    for (int k = k0; k <= k1; ++k) {
      const int width = min((grp + 1) * g.cpg, (k + 1) * per) - max(grp * g.cpg, k * per);
      const float2 v = __ldcg(part + (pic * g.splits + s) * g.slots + grp + k);
      m = join(m, Moments{(float)(r1 - r0) * (float)width, v.x, v.y});
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
  if (!p.on || p.r0 + p.lane >= p.r1) return;
  Channels<V> ch;
  ch.load(g, norm_stat, g0, p.col * V, weight, bias);
  const T* src = x + p.pic * g.x_sn + (long)p.col * V;
  T* dst = y + p.pic * g.y_sn + (long)p.col * V;
  // batches of loads before their stores: y may be x, so the compiler must not reorder them
  constexpr int kBatch = sizeof(Pack<T, V>) == 16 ? 2 : 4;
  const long steps = (p.r1 - p.r0 - p.lane - 1) / g.rp;
  for (long row = p.r0 + p.lane + steps * g.rp; row >= p.r0; row -= kBatch * g.rp) {
    Pack<T, V> a[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (row - b * g.rp >= p.r0) a[b].load(src + (row - b * g.rp) * g.x_sl);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (row - b * g.rp < p.r0) break;
      float v[V];
      unpack(a[b], v);
      ch.z(v, v);
      act_all<ACT, V>(g, v);
      repack<T, V>(v).store(dst + (row - b * g.rp) * g.y_sl);
    }
  }
}

// gz = dy act'(z) of V values.
template <int ACT, int V>
__device__ __forceinline__ void grad_z(const NormGeom& g, const Channels<V>& ch, const float* x, const float* dy,
                                       float* gz) {
  ch.z(x, gz);
  slope_all<ACT, V>(g, gz);
#pragma unroll
  for (int i = 0; i < V; ++i) gz[i] *= dy[i];
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
#pragma unroll
  for (int i = 0; i < V; ++i) {
    sa[i] += gz[i];
    sb[i] = fmaf(gz[i], hat.at(i, v[i]), sb[i]);
  }
}

// First pass of the gradient: per (picture, split) the channels' sums of gz and gz xh for dw
// and db, and the parts of the groups' sums of h and h xh.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(NORM_THREADS, 2)
norm_grad_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean,
                      const float* __restrict__ rstd, const float* __restrict__ weight,
                      const float* __restrict__ bias, float2* __restrict__ part, float2* __restrict__ cpart,
                      const __grid_constant__ NormGeom g) {
  extern __shared__ __align__(16) float norm_sm[];  // the block's sums, then the chunk's groups' statistics
  let_next_start();
  const NormPlace p(g, V);
  const int g0 = p.c0 / g.cpg;
  float2* stats = reinterpret_cast<float2*>(norm_sm + BlockSums<V, NORM_THREADS>::floats(g.tc));
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
    const T* src = x + p.pic * g.x_sn + (long)p.col * V;
    const T* del = dy + p.pic * g.d_sn + (long)p.col * V;
#pragma unroll 4
    for (long row = p.r0 + p.lane; row < p.r1; row += g.rp) {
      Pack<T, V> a, e;
      a.load(src + row * g.x_sl);
      e.load(del + row * g.d_sl);
      add_grad<T, V, ACT>(g, ch, hat, a, e, sa, sb);
    }
  }
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
  for (int s = threadIdx.x & 31; s < g.splits; s += 32)
    for (int k = k0; k <= k1; ++k) m = join(m, __ldcg(part + (pic * g.splits + s) * g.slots + grp + k));
  m = warp_join(m);
  const float inv = 1.f / ((float)g.l * (float)g.cpg);
  return make_float2(m.x * inv, m.y * inv);
}

// dx = gz sc - rs E[h] - xh rs E[h xh] of one vector (sc = rs w).
template <int V>
struct GradMeans {
  float m1[V], m2[V];  // rs E[h], rs E[h xh]
  __device__ __forceinline__ void load(const NormGeom& g, const Hats<V>& hat, const float2* means, int first_group,
                                       int c0) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 m = means[group_of(g, c0, i) - first_group];
      m1[i] = hat.rs[i] * m.x;
      m2[i] = hat.rs[i] * m.y;
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
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = fmaf(gz[i], ch.sc[i], -m.m1[i]) - hat.at(i, v[i]) * m.m2[i];
  return repack<T, V>(v);
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(NORM_THREADS, 2)
norm_grad_apply_kernel(const T* dy, const T* x, T* dx,
                       const float* __restrict__ mean, const float* __restrict__ rstd,
                       const float* __restrict__ weight, const float* __restrict__ bias,
                       const float2* __restrict__ part, const __grid_constant__ NormGeom g) {
  extern __shared__ __align__(16) float2 norm_stat[];  // (mean, rstd), then (E[h], E[h xh]) of the chunk's groups
  const NormPlace p(g, V);
  const int g0 = p.c0 / g.cpg, ng = (p.c1 - 1) / g.cpg - g0 + 1;
  grad_stats(g, norm_stat, g0, p.c1, mean, rstd, p.pic);
  wait_for_previous();
  for (int grp = g0 + (threadIdx.x >> 5); grp * g.cpg < p.c1; grp += NORM_THREADS / 32) {
    const float2 m = norm_grad_join(g, part, p.pic, grp, V);
    if ((threadIdx.x & 31) == 0) norm_stat[ng + grp - g0] = m;
  }
  __syncthreads();
  if (!p.on || p.r0 + p.lane >= p.r1) return;
  Channels<V> ch;
  ch.load(g, norm_stat, g0, p.col * V, weight, bias);
  Hats<V> hat;
  GradMeans<V> m;
  hat.load(g, norm_stat, g0, p.col * V);
  m.load(g, hat, norm_stat + ng, g0, p.col * V);
  const T* src = x + p.pic * g.x_sn + (long)p.col * V;
  const T* del = dy + p.pic * g.d_sn + (long)p.col * V;
  T* dst = dx + p.pic * g.y_sn + (long)p.col * V;
  const long steps = (p.r1 - p.r0 - p.lane - 1) / g.rp;
  constexpr int kBatch = 2;
  for (long row = p.r0 + p.lane + steps * g.rp; row >= p.r0; row -= kBatch * g.rp) {
    Pack<T, V> a[kBatch], e[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (row - k * g.rp >= p.r0) {
        a[k].load(src + (row - k * g.rp) * g.x_sl);
        e[k].load(del + (row - k * g.rp) * g.d_sl);
      }
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (row - k * g.rp >= p.r0)
        grad_x<T, V, ACT>(g, ch, hat, m, a[k], e[k]).store(dst + (row - k * g.rp) * g.y_sl);
  }
}

// dw and db: one warp a channel joins `parts` partials (pictures x splits).
__global__ void __launch_bounds__(256) norm_grad_params_kernel(const float2* __restrict__ cpart, long parts,
                                                                        int c, float* __restrict__ dweight,
                                                                        float* __restrict__ dbias) {
  // 32 neighbouring channels a block, eight threads each
  __shared__ float2 sums[8][33];
  const int ch = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;
  float2 m = make_float2(0.f, 0.f);
  if (ch < c)
    for (long k = lane; k < parts; k += 8) m = join(m, cpart[k * c + ch]);
  sums[lane][threadIdx.x & 31] = m;
  __syncthreads();
  if (lane == 0 && ch < c) {
    for (int k = 1; k < 8; ++k) m = join(m, sums[k][threadIdx.x]);
    if (dbias) dbias[ch] = m.x;
    if (dweight) dweight[ch] = m.y;
  }
}

// The small form: block (picture, chunk of whole groups), the chunk's values in shared
// memory; kT threads: 128 where the values are few and blocks many, else 512. GRAD: x and dy, dx out; the channels' sums go to dw and db when there is one
// picture, else to cpart.
template <typename T, int V, bool GRAD, int kT>
__global__ void __launch_bounds__(kT)
norm_small_kernel(const T* dy, const T* x, T* y, float* __restrict__ mean,
                  float* __restrict__ rstd, const float* __restrict__ weight, const float* __restrict__ bias,
                  float* __restrict__ dweight, float* __restrict__ dbias, float2* __restrict__ cpart,
                  const __grid_constant__ NormGeom g) {
  extern __shared__ __align__(16) float norm_sm[];
  // the block's sums; K; (mean, rstd), (E[h], E[h xh]) of the groups; the values
  float* first = norm_sm + BlockSums<V, kT>::floats(g.tc);
  float2* stats = reinterpret_cast<float2*>(first + (g.tc * V + 1) / 2 * 2);
  const NormPlace p(g, V);
  const int g0 = p.c0 / g.cpg, ng = (p.c1 - p.c0) / g.cpg;
  Pack<T, V>* keep = reinterpret_cast<Pack<T, V>*>(norm_sm + g.keep);
  Pack<T, V>* keep_d = keep + (GRAD ? g.l * g.tc : 0);
  const int t = threadIdx.x % g.tc;
  const T* src = x + p.pic * g.x_sn + (long)p.col * V;
  const T* del = GRAD ? dy + p.pic * g.d_sn + (long)p.col * V : nullptr;
  if (!GRAD) {
    float k[V], sum[V], sq[V];
#pragma unroll
    for (int i = 0; i < V; ++i) k[i] = sum[i] = sq[i] = 0.f;
    if (p.on && g.l > 0) {
      Pack<T, V> a;
      float v[V];
      middle_of_rows<T, V>(src, g.x_sl, 0, g.l, k);
#pragma unroll 4
      for (long row = p.lane; row < g.l; row += g.rp) {
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
    sums.add(norm_sm, g, sum, sq, p.lane);
    for (int n = threadIdx.x >> 5; n < ng; n += kT / 32) {
      const float2 m = group_moments(sums, first, n * g.cpg, (n + 1) * g.cpg, (float)g.l);
      if ((threadIdx.x & 31) == 0) {
        const float rs = 1.f / sqrtf((g.l > 0 ? m.y / ((float)g.l * (float)g.cpg) : 0.f) + g.eps);
        stats[n] = make_float2(m.x, rs);
        if (mean) mean[p.pic * g.groups + g0 + n] = m.x;
        if (rstd) rstd[p.pic * g.groups + g0 + n] = rs;
      }
    }
  } else {
    grad_stats(g, stats, g0, p.c1, mean, rstd, p.pic);
  }
  __syncthreads();
  Channels<V> ch;
  Hats<V> hat;
  if (p.on) {
    ch.load(g, stats, g0, p.col * V, weight, bias);
    if (GRAD) hat.load(g, stats, g0, p.col * V);
  }
  T* dst = y + p.pic * g.y_sn + (long)p.col * V;
  if constexpr (!GRAD) {
    if (p.on)
      for (long row = p.lane; row < g.l; row += g.rp) {
        float v[V];
        unpack(keep[row * g.tc + t], v);
        ch.z(v, v);
        act_all<ACT_ANY, V>(g, v);
        repack<T, V>(v).store(dst + row * g.y_sl);
      }
  } else {
    float sa[V], sb[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sa[i] = sb[i] = 0.f;
    if (p.on) {
#pragma unroll 2
      for (long row = p.lane; row < g.l; row += g.rp) {
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
          cpart[p.pic * g.c + c] = s;
        } else {
          if (dbias) dbias[c] = s.x;
          if (dweight) dweight[c] = s.y;
        }
      }
      m = warp_join(m);
      const float inv = 1.f / ((float)g.l * (float)g.cpg);
      if ((threadIdx.x & 31) == 0) means[k] = make_float2(m.x * inv, m.y * inv);
    }
    __syncthreads();
    if (!p.on) return;
    GradMeans<V> m;
    m.load(g, hat, means, g0, p.col * V);
    for (long row = p.lane; row < g.l; row += g.rp)
      grad_x<T, V, ACT_ANY>(g, ch, hat, m, keep[row * g.tc + t], keep_d[row * g.tc + t]).store(dst + row * g.y_sl);
  }
}

}  // namespace scb
