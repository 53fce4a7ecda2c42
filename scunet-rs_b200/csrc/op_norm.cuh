// Group norm with an activation over channels-last maps, and its gradient.
//
//   x [N][L][C], G groups of C / G neighbouring channels; per picture n and group g
//   mean = E[x], var = E[(x - mean)^2] over the L rows and the group's channels,
//   xh = (x - mean) / sqrt(var + eps),  z = w_c xh + b_c,  y = act(z).
// Gradient, with gz = dy act'(z) and h = gz w_c:
//   db_c = sum gz,  dw_c = sum gz xh  (over n and L),
//   dx = rstd (h - E_g[h] - xh E_g[h xh]).
//
// Three launches: per-channel partials of row ranges, their join per group, and the
// elementwise pass. Statistics are fp32: a thread sums x - K and (x - K)^2 with K its
// first value of the channel, so that the sum of squares loses nothing to a large mean
// (K is one of the values, so a K far from the rest is itself part of the spread it
// stands against), and (count, mean, M2) triples are joined pairwise,
//   M2 = M2a + M2b + (mb - ma)^2 na nb / (na + nb).
// No atomics: the order of every sum is fixed by the sizes.
#pragma once
#include "ops_common.cuh"

namespace scb {

struct NormGeom {
  long n, l;          // pictures, rows of each
  int c, groups, cpg; // channels, groups, channels per group
  int cols;           // vectors of a row
  int tc, rp;         // vectors of a row that one block takes, rows it takes at once
  int splits;         // row ranges of a picture
  long x_sn, x_sl;    // element strides of pictures and rows
  long y_sn, y_sl;
  long d_sn, d_sl;    // dy
  float eps;
  int act;            // read by the kernels compiled for ACT_ANY
};

constexpr int NORM_THREADS = 256;

// The narrow vectors take the activation at run time (ACT_ANY).
template <int ACT>
__device__ __forceinline__ float act_of(const NormGeom& g, float z) {
  if (ACT != ACT_ANY) return act_fwd<ACT>(z);
  return g.act == ACT_RELU ? act_fwd<ACT_RELU>(z) : g.act == ACT_SILU ? act_fwd<ACT_SILU>(z)
         : g.act == ACT_GELU ? act_fwd<ACT_GELU>(z) : z;
}
template <int ACT>
__device__ __forceinline__ float slope_of(const NormGeom& g, float z) {
  if (ACT != ACT_ANY) return act_slope<ACT>(z);
  return g.act == ACT_RELU ? act_slope<ACT_RELU>(z) : g.act == ACT_SILU ? act_slope<ACT_SILU>(z)
         : g.act == ACT_GELU ? act_slope<ACT_GELU>(z) : 1.f;
}

struct Moments {
  float n, mean, m2;
};
__device__ __forceinline__ Moments join(const Moments& a, const Moments& b) {
  const float n = a.n + b.n;
  if (n == 0.f) return a;
  const float d = b.mean - a.mean, f = b.n / n;
  return {n, a.mean + d * f, a.m2 + b.m2 + d * d * a.n * f};
}

// The row range of split s.
__device__ __forceinline__ void norm_rows(const NormGeom& g, int s, long& r0, long& r1) {
  r0 = g.l * s / g.splits;
  r1 = g.l * (s + 1) / g.splits;
}

// Per (picture, split, channel): mean and M2 of the split's rows -> part[n][split][c].
template <typename T, int V>
__global__ void __launch_bounds__(NORM_THREADS) norm_stats_kernel(const T* __restrict__ x, float2* __restrict__ part,
                                                                  const NormGeom g) {
  extern __shared__ float norm_sm[];
  const int tid = threadIdx.x, col = blockIdx.y * g.tc + tid % g.tc, lane = tid / g.tc;
  const bool on = lane < g.rp && col < g.cols;
  long r0, r1;
  const long pic = blockIdx.x / g.splits;
  const int split = (int)(blockIdx.x % g.splits);
  norm_rows(g, split, r0, r1);
  float k[V], s[V], q[V];
  float cnt = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) k[i] = s[i] = q[i] = 0.f;
  if (on) {
    const T* p = x + pic * g.x_sn + (long)col * V;
    long r = r0 + lane;
    if (r < r1) {
      Pack<T, V> a;
      a.load(p + r * g.x_sl);
#pragma unroll
      for (int i = 0; i < V; ++i) k[i] = to_f32(a.v[i]);
      cnt = (float)((r1 - r + g.rp - 1) / g.rp);
    }
#pragma unroll 4
    for (; r < r1; r += g.rp) {
      Pack<T, V> a;
      a.load(p + r * g.x_sl);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = to_f32(a.v[i]) - k[i];
        s[i] += d;
        q[i] += d * d;
      }
    }
  }
  // join the block's row lanes, channel by channel, as a tree over lanes
  float* sn = norm_sm;                    // [256]
  float* sm = norm_sm + NORM_THREADS;     // [V][256]
  float* sq = sm + V * NORM_THREADS;      // [V][256]
  const float inv = cnt > 0.f ? 1.f / cnt : 0.f;
  sn[tid] = cnt;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    sm[i * NORM_THREADS + tid] = k[i] + s[i] * inv;
    sq[i * NORM_THREADS + tid] = fmaxf(q[i] - s[i] * s[i] * inv, 0.f);
  }
  int top = 1;
  while (top < g.rp) top *= 2;
  for (int h = top / 2; h >= 1; h /= 2) {
    __syncthreads();
    if (lane < h && lane + h < g.rp) {
      const int o = tid + h * g.tc;
      const float na = sn[tid], nb = sn[o];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int a = i * NORM_THREADS;
        const Moments m = join({na, sm[a + tid], sq[a + tid]}, {nb, sm[a + o], sq[a + o]});
        sm[a + tid] = m.mean;
        sq[a + tid] = m.m2;
      }
      sn[tid] = na + nb;
    }
  }
  if (lane == 0 && on) {
    float2* o = part + (long)blockIdx.x * g.c + (long)col * V;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = make_float2(sm[i * NORM_THREADS + tid], sq[i * NORM_THREADS + tid]);
  }
}

__device__ __forceinline__ Moments shfl_down(const Moments& m, int d) {
  return {__shfl_down_sync(0xffffffffu, m.n, d), __shfl_down_sync(0xffffffffu, m.mean, d),
          __shfl_down_sync(0xffffffffu, m.m2, d)};
}

// One block per (group, picture): joins the partials of all splits and channels.
__global__ void __launch_bounds__(NORM_THREADS) norm_join_kernel(const float2* __restrict__ part,
                                                                 float* __restrict__ mean, float* __restrict__ rstd,
                                                                 const NormGeom g) {
  __shared__ Moments sw[NORM_THREADS / 32];
  Moments m{0.f, 0.f, 0.f};
  const long pic = blockIdx.x / g.groups, grp = blockIdx.x % g.groups;
  for (int i = threadIdx.x; i < g.splits * g.cpg; i += NORM_THREADS) {
    const int s = i / g.cpg, c = i - s * g.cpg;
    long r0, r1;
    norm_rows(g, s, r0, r1);
    const float2 v = part[(pic * g.splits + s) * g.c + grp * g.cpg + c];
    m = join(m, {(float)(r1 - r0), v.x, v.y});
  }
  for (int d = 16; d >= 1; d /= 2) m = join(m, shfl_down(m, d));
  if ((threadIdx.x & 31) == 0) sw[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x < 32) {
    m = threadIdx.x < NORM_THREADS / 32 ? sw[threadIdx.x] : Moments{0.f, 0.f, 0.f};
    for (int d = NORM_THREADS / 64; d >= 1; d /= 2) m = join(m, shfl_down(m, d));
    if (threadIdx.x == 0) {
      mean[pic * g.groups + grp] = m.mean;
      rstd[pic * g.groups + grp] = 1.f / sqrtf((m.n > 0.f ? m.m2 / m.n : 0.f) + g.eps);
    }
  }
}

// y = act(x scale_c + shift_c), the pass over the values.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(NORM_THREADS)
norm_apply_kernel(const T* __restrict__ x, T* __restrict__ y, const float* __restrict__ mean,
                  const float* __restrict__ rstd, const float* __restrict__ weight, const float* __restrict__ bias,
                  const NormGeom g) {
  const int tid = threadIdx.x, col = blockIdx.y * g.tc + tid % g.tc, lane = tid / g.tc;
  if (lane >= g.rp || col >= g.cols) return;
  const long pic = blockIdx.x / g.splits;
  const int split = (int)(blockIdx.x % g.splits);
  float mu[V], sc[V], sh[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = col * V + i;
    const long k = pic * g.groups + c / g.cpg;
    mu[i] = mean[k];
    sc[i] = rstd[k] * (weight ? weight[c] : 1.f);
    sh[i] = bias ? bias[c] : 0.f;
  }
  long r0, r1;
  norm_rows(g, split, r0, r1);
  const T* p = x + pic * g.x_sn + (long)col * V;
  T* o = y + pic * g.y_sn + (long)col * V;
#pragma unroll 4
  for (long r = r0 + lane; r < r1; r += g.rp) {
    Pack<T, V> a;
    a.load(p + r * g.x_sl);
#pragma unroll
    for (int i = 0; i < V; ++i) a.v[i] = from_f32<T>(act_of<ACT>(g, (to_f32(a.v[i]) - mu[i]) * sc[i] + sh[i]));
    a.store(o + r * g.y_sl);
  }
}

// Per (picture, split, channel): sums of gz and gz xh over the split's rows.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(NORM_THREADS)
norm_grad_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean,
                      const float* __restrict__ rstd, const float* __restrict__ weight,
                      const float* __restrict__ bias, float2* __restrict__ part, const NormGeom g) {
  extern __shared__ float norm_sm[];
  const int tid = threadIdx.x, col = blockIdx.y * g.tc + tid % g.tc, lane = tid / g.tc;
  const bool on = lane < g.rp && col < g.cols;
  const long pic = blockIdx.x / g.splits;
  const int split = (int)(blockIdx.x % g.splits);
  float sa[V], sb[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sa[i] = sb[i] = 0.f;
  if (on) {
    float mu[V], rs[V], w[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = col * V + i;
      const long k = pic * g.groups + c / g.cpg;
      mu[i] = mean[k];
      rs[i] = rstd[k];
      w[i] = weight ? weight[c] : 1.f;
      b[i] = bias ? bias[c] : 0.f;
    }
    long r0, r1;
    norm_rows(g, split, r0, r1);
    const T* p = x + pic * g.x_sn + (long)col * V;
    const T* d = dy + pic * g.d_sn + (long)col * V;
#pragma unroll 2
    for (long r = r0 + lane; r < r1; r += g.rp) {
      Pack<T, V> a, e;
      a.load(p + r * g.x_sl);
      e.load(d + r * g.d_sl);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = (to_f32(a.v[i]) - mu[i]) * rs[i];
        const float gz = to_f32(e.v[i]) * slope_of<ACT>(g, xh * w[i] + b[i]);
        sa[i] += gz;
        sb[i] += gz * xh;
      }
    }
  }
  float* ra = norm_sm;                     // [V][256]
  float* rb = norm_sm + V * NORM_THREADS;  // [V][256]
#pragma unroll
  for (int i = 0; i < V; ++i) {
    ra[i * NORM_THREADS + tid] = sa[i];
    rb[i * NORM_THREADS + tid] = sb[i];
  }
  int top = 1;
  while (top < g.rp) top *= 2;
  for (int h = top / 2; h >= 1; h /= 2) {
    __syncthreads();
    if (lane < h && lane + h < g.rp) {
      const int o = tid + h * g.tc;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        ra[i * NORM_THREADS + tid] += ra[i * NORM_THREADS + o];
        rb[i * NORM_THREADS + tid] += rb[i * NORM_THREADS + o];
      }
    }
  }
  if (lane == 0 && on) {
    float2* o = part + (long)blockIdx.x * g.c + (long)col * V;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = make_float2(ra[i * NORM_THREADS + tid], rb[i * NORM_THREADS + tid]);
  }
}

// One block per channel: joins the splits. sums[n][c] = the picture's (sum gz, sum gz xh);
// dw and db add the pictures.
__global__ void __launch_bounds__(32) norm_grad_join_kernel(const float2* __restrict__ part, float2* __restrict__ sums,
                                                            float* __restrict__ dweight, float* __restrict__ dbias,
                                                            const NormGeom g) {
  const int c = blockIdx.x;
  float ta = 0.f, tb = 0.f;
  for (long pic = 0; pic < g.n; ++pic) {
    float a = 0.f, b = 0.f;
    for (int s = threadIdx.x; s < g.splits; s += 32) {
      const float2 v = part[(pic * g.splits + s) * g.c + c];
      a += v.x;
      b += v.y;
    }
    for (int d = 16; d >= 1; d /= 2) {
      a += __shfl_down_sync(0xffffffffu, a, d);
      b += __shfl_down_sync(0xffffffffu, b, d);
    }
    if (threadIdx.x == 0) sums[pic * g.c + c] = make_float2(a, b);
    ta += a;
    tb += b;
  }
  if (threadIdx.x == 0) {
    if (dbias) dbias[c] = ta;
    if (dweight) dweight[c] = tb;
  }
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(NORM_THREADS)
norm_grad_apply_kernel(const T* __restrict__ dy, const T* __restrict__ x, T* __restrict__ dx,
                       const float* __restrict__ mean, const float* __restrict__ rstd,
                       const float* __restrict__ weight, const float* __restrict__ bias,
                       const float2* __restrict__ sums, const NormGeom g) {
  const int tid = threadIdx.x, col = blockIdx.y * g.tc + tid % g.tc, lane = tid / g.tc;
  if (lane >= g.rp || col >= g.cols) return;
  const long pic = blockIdx.x / g.splits;
  const int split = (int)(blockIdx.x % g.splits);
  float mu[V], rs[V], w[V], b[V], m1[V], m2[V];
  int last = -1;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = col * V + i, grp = c / g.cpg;
    const long k = pic * g.groups + grp;
    mu[i] = mean[k];
    rs[i] = rstd[k];
    w[i] = weight ? weight[c] : 1.f;
    b[i] = bias ? bias[c] : 0.f;
    if (i > 0 && grp == last) {
      m1[i] = m1[i - 1];
      m2[i] = m2[i - 1];
    } else {
      float a1 = 0.f, a2 = 0.f;
      for (int j = 0; j < g.cpg; ++j) {
        const float2 v = sums[pic * g.c + grp * g.cpg + j];
        const float wj = weight ? weight[grp * g.cpg + j] : 1.f;
        a1 += wj * v.x;
        a2 += wj * v.y;
      }
      const float inv = 1.f / ((float)g.l * (float)g.cpg);
      m1[i] = a1 * inv;
      m2[i] = a2 * inv;
      last = grp;
    }
  }
  long r0, r1;
  norm_rows(g, split, r0, r1);
  const T* p = x + pic * g.x_sn + (long)col * V;
  const T* d = dy + pic * g.d_sn + (long)col * V;
  T* o = dx + pic * g.y_sn + (long)col * V;
#pragma unroll 2
  for (long r = r0 + lane; r < r1; r += g.rp) {
    Pack<T, V> a, e;
    a.load(p + r * g.x_sl);
    e.load(d + r * g.d_sl);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float xh = (to_f32(a.v[i]) - mu[i]) * rs[i];
      const float h = to_f32(e.v[i]) * slope_of<ACT>(g, xh * w[i] + b[i]) * w[i];
      a.v[i] = from_f32<T>(rs[i] * (h - m1[i] - xh * m2[i]));
    }
    a.store(o + r * g.y_sl);
  }
}

}  // namespace scb
