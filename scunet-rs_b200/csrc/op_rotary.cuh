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
// P sines and cosines once into shared memory and then streams the heads through.
#pragma once
#include "ops_common.cuh"

namespace scb {

constexpr int ROT_AXES = 4;
constexpr int ROT_THREADS = 256;
enum : int { ROT_HALF = 0, ROT_INTERLEAVED = 1, ROT_AXIAL = 2 };
enum : int { POS_I32 = 0, POS_I64 = 1, POS_F32 = 2 };

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
};

__device__ __forceinline__ float rot_position(const RotGeom& g, long i) {
  if (g.pos_type == POS_I32) return (float)static_cast<const int*>(g.pos)[i];
  if (g.pos_type == POS_I64) return (float)static_cast<const long long*>(g.pos)[i];
  return static_cast<const float*>(g.pos)[i];
}

template <typename T, int LAYOUT>
__global__ void __launch_bounds__(ROT_THREADS) rotary_kernel(const RotGeom g) {
  extern __shared__ float2 rot_cs[];  // [tokens of the block][pairs]: cos, sin
  const long t0 = (long)blockIdx.x * g.per_block;
  const int nt = (int)min((long)g.per_block, g.tokens - t0);
  for (int i = threadIdx.x; i < nt * g.pairs; i += ROT_THREADS) {
    const int tk = i / g.pairs, p = i - tk * g.pairs;
    const long tok = t0 + tk, b = tok / g.l, l = tok - b * g.l;
    int a = 0;
    while (a + 1 < g.axes && p >= g.first[a + 1]) ++a;
    float s, c;
    sincosf(rot_position(g, b * g.pos_sb + l * g.pos_sl + a * g.pos_sa) * g.freq[p], &s, &c);
    rot_cs[i] = make_float2(c, s * g.sign);
  }
  __syncthreads();
  const int rest = g.d - 2 * g.pairs, items = g.pairs + rest;  // one pair or one copied channel each
  for (int w = 0; w < 2; ++w) {
    const RotTensor& q = g.t[w];
    const int per_tok = q.heads * items;
    for (int i = threadIdx.x; i < nt * per_tok; i += ROT_THREADS) {
      const int tk = i / per_tok, r = i - tk * per_tok, h = r / items, p = r - h * items;
      const long tok = t0 + tk, b = tok / g.l, l = tok - b * g.l;
      const T* x = static_cast<const T*>(q.x) + b * q.x_sb + l * q.x_sl + h * q.x_sh;
      T* y = static_cast<T*>(q.y) + b * q.y_sb + l * q.y_sl + h * q.y_sh;
      if (p >= g.pairs) {
        y[p + g.pairs] = x[p + g.pairs];
        continue;
      }
      int lo, hi;
      if (LAYOUT == ROT_HALF) {
        lo = p;
        hi = p + g.pairs;
      } else if (LAYOUT == ROT_INTERLEAVED) {
        lo = 2 * p;
        hi = lo + 1;
      } else {
        int a = 0;
        while (a + 1 < g.axes && p >= g.first[a + 1]) ++a;
        lo = p + g.first[a];
        hi = lo + g.first[a + 1] - g.first[a];
      }
      const float2 cs = rot_cs[tk * g.pairs + p];
      const float u = to_f32(x[lo]), v = to_f32(x[hi]);
      y[lo] = from_f32<T>(u * cs.x - v * cs.y);
      y[hi] = from_f32<T>(u * cs.y + v * cs.x);
    }
  }
}

}  // namespace scb
