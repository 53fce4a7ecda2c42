// Rotation of queries and keys by several position axes (time, row, column of a cell).
//
//   x [B][L][H][D], pos [L or B x L][A]; pair p of a head turns with axis a(p):
//   t = pos[l][a(p)] * freq[p] (one fp32 product),  (u, v) -> (u cos t - v sin t,
//   u sin t + v cos t). The gradient of the rotation is the rotation by -t (`inverse`).
// Pairs 0 .. P-1 are split over the axes in order, `sections` pairs each; channels past
// 2 P are copied. Channels (u, v) of pair p:
//   half:        p, p + P
//   interleaved: 2 p, 2 p + 1
//   axial:       every axis has its own 2 m channels, in halves: 2 f + j, 2 f + j + m for
//                pair j of an axis whose pairs start at f
//
// The angles are shared by all heads of q and k: a block takes some tokens, computes their
// P cosines and sines once into shared memory, then streams the heads through, neighbouring
// lanes on neighbouring vectors of a token's heads. An item is V pairs in two vectors of V
// channels (interleaved: neighbouring ones), or V copied channels past the last pair.
// Bound by memory, x read once and written once: 33 us for q and k of a packed 136 x 240 map
// with 16 heads of 32 fp16 (4.1 TB/s), 126 us for 16 heads of 128 over 2 x 31995 tokens bf16
// (4.2 TB/s); one token is one launch, 3.3 us. Scalar pairs took 129 and 437 us.
#pragma once
#include "ops_common.cuh"

namespace scb {

constexpr int ROT_AXES = 4;
constexpr int ROT_THREADS = 256;
enum : int { ROT_HALF = 0, ROT_INTERLEAVED = 1, ROT_AXIAL = 2 };
enum : int { POS_I32 = 0, POS_I64 = 1, POS_F32 = 2 };

// n / d for 32-bit n: (n * m) >> 32 >> s with m = ceil(2^(32 + s) / d), s = ceil(log2 d), where
// m has 33 bits; the top one is added by hand (Granlund and Montgomery, division by
// invariant integers using multiplication).
struct Divide {
  unsigned d, m, s1, s2;
  __host__ static Divide by(unsigned d) {
    unsigned l = 0;
    while (l < 32 && (1ull << l) < d) ++l;
    const unsigned m = (unsigned)(((1ull << 32) * ((1ull << l) - d)) / d + 1);
    return {d, m, l < 1 ? l : 1, l > 1 ? l - 1 : 0};
  }
  __device__ __forceinline__ unsigned div(unsigned n) const {
    const unsigned t = __umulhi(m, n);
    return (t + ((n - t) >> s1)) >> s2;
  }
};

struct RotTensor {
  const void* x;
  void* y;
  int heads;
  long x_sb, x_sl, x_sh, y_sb, y_sl, y_sh;  // element strides: batch, token, head
};

struct RotGeom {
  RotTensor t[2];       // q and k (heads 0: absent)
  long b, l, tokens;    // tokens = b * l
  int d, pairs, axes;
  int first[ROT_AXES + 1];  // first pair of each axis, then the number of pairs
  const void* pos;
  int pos_type;
  long pos_sb, pos_sl, pos_sa;
  const float* freq;
  float sign;           // -1: the inverse rotation
  int per_block;        // tokens of a block
  int vecs;             // items of a head
  unsigned items;       // items of a token: vecs * (heads of q and k)
  Divide by_items, by_vecs, by_l, by_pairs;
};

__device__ __forceinline__ float rot_position(const RotGeom& g, long i) {
  if (g.pos_type == POS_I32) return (float)static_cast<const int*>(g.pos)[i];
  if (g.pos_type == POS_I64) return (float)static_cast<const long long*>(g.pos)[i];
  return static_cast<const float*>(g.pos)[i];
}

// Where an item's channels lie: V at `lo` and V at `hi` (hi < 0: copied channels only); its
// first pair is `p`. Interleaved items of V > 1 are 2 V neighbouring channels, of which
// those past the last pair are left as they are.
struct RotItem {
  int lo, hi, p;
};
template <int LAYOUT, int V>
__device__ __forceinline__ RotItem rot_item(const RotGeom& g, int v) {
  const int p = V * v;
  if (LAYOUT == ROT_INTERLEAVED && V > 1) return {2 * p, 2 * p + V, p};
  if (p >= g.pairs) return {p + g.pairs, -1, p};
  if (LAYOUT == ROT_INTERLEAVED) return {2 * p, 2 * p + 1, p};
  if (LAYOUT == ROT_HALF) return {p, p + g.pairs, p};
  int a = 0;
  while (a + 1 < g.axes && p >= g.first[a + 1]) ++a;
  return {p + g.first[a], p + g.first[a + 1], p};
}

template <typename T, int LAYOUT, int V>
__device__ __forceinline__ void rotate(const RotGeom& g, const float2* cs, const RotItem& it,
                                       Pack<T, V>& a, Pack<T, V>& b) {
  if (LAYOUT == ROT_INTERLEAVED && V > 1) {
    // a and b are the two halves of 2 V neighbouring channels
    T* e[2] = {a.v, b.v};
#pragma unroll
    for (int i = 0; i < V; ++i) {
      T &x = e[2 * i / V][2 * i % V], &y = e[(2 * i + 1) / V][(2 * i + 1) % V];
      if (it.p + i < g.pairs) {
        const float2 c = cs[it.p + i];
        const float u = to_f32(x), v = to_f32(y);
        x = from_f32<T>(u * c.x - v * c.y);
        y = from_f32<T>(u * c.y + v * c.x);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 c = cs[it.p + i];
      const float u = to_f32(a.v[i]), v = to_f32(b.v[i]);
      a.v[i] = from_f32<T>(u * c.x - v * c.y);
      b.v[i] = from_f32<T>(u * c.y + v * c.x);
    }
  }
}

template <typename T, int LAYOUT, int V>
__global__ void __launch_bounds__(ROT_THREADS) rotary_kernel(const __grid_constant__ RotGeom g) {
  extern __shared__ __align__(16) float2 rot_cs[];  // [tokens of the block][pairs]: cos, sin
  const long t0 = (long)blockIdx.x * g.per_block;
  const int nt = (int)min((long)g.per_block, g.tokens - t0);
  const long b0 = t0 / g.l;
  const unsigned l0 = (unsigned)(t0 - b0 * g.l);  // l0 + per_block < 2^32: l is below 2^31
  for (unsigned i = threadIdx.x; i < (unsigned)nt * g.pairs; i += ROT_THREADS) {
    const unsigned tk = g.by_pairs.div(i), p = i - tk * g.pairs;
    const unsigned over = g.by_l.div(l0 + tk), l = l0 + tk - over * (unsigned)g.l;
    int a = 0;
    while (a + 1 < g.axes && (int)p >= g.first[a + 1]) ++a;
    float s, c;
    sincosf(rot_position(g, (b0 + over) * g.pos_sb + l * g.pos_sl + a * g.pos_sa) * g.freq[p], &s, &c);
    rot_cs[i] = make_float2(c, s * g.sign);
  }
  __syncthreads();
  // two items at a time, both loaded before either is stored: y may be x
  constexpr int kBatch = 2;
  const unsigned all = (unsigned)nt * g.items;
  for (unsigned i0 = threadIdx.x; i0 < all; i0 += kBatch * ROT_THREADS) {
    Pack<T, V> a[kBatch], b[kBatch];
    T* y[kBatch];
    RotItem it[kBatch];
    unsigned tk[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const unsigned i = i0 + k * ROT_THREADS;
      if (i >= all) continue;
      tk[k] = g.by_items.div(i);
      unsigned r = i - tk[k] * g.items;
      const unsigned q_items = g.t[0].heads * g.vecs;
      const int w = r >= q_items;
      r -= w ? q_items : 0;
      const unsigned h = g.by_vecs.div(r);
      it[k] = rot_item<LAYOUT, V>(g, (int)(r - h * g.vecs));
      const unsigned over = g.by_l.div(l0 + tk[k]), l = l0 + tk[k] - over * (unsigned)g.l;
      const RotTensor& t = g.t[w];
      const T* x = static_cast<const T*>(t.x) + (b0 + over) * t.x_sb + l * t.x_sl + h * t.x_sh + it[k].lo;
      y[k] = static_cast<T*>(t.y) + (b0 + over) * t.y_sb + l * t.y_sl + h * t.y_sh + it[k].lo;
      a[k].load(x);
      if (it[k].hi >= 0) b[k].load(x + (it[k].hi - it[k].lo));
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (i0 + k * ROT_THREADS >= all) continue;
      if (it[k].hi >= 0) {
        rotate<T, LAYOUT, V>(g, rot_cs + tk[k] * g.pairs, it[k], a[k], b[k]);
        b[k].store(y[k] + (it[k].hi - it[k].lo));
      }
      a[k].store(y[k]);
    }
  }
}

}  // namespace scb
