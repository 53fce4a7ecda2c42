// Attention of every query over all visible keys of its picture:
//   o_i = sum_j p_ij v_j,  p_i = softmax over the visible j of scale q_i . k_j
// with key heads shared by runs of query heads (head h reads key head h / (H / Hk)) and a
// key mask per picture. A picture with no visible key gives zeros.
//
// One pass over the keys with the running maximum m and sum l of the softmax (in units of
// log2): when a tile raises m to m', the accumulated o and l are scaled by 2^(m - m').
#pragma once
#include <cfloat>

#include "ops_common.cuh"

namespace scb {

struct AttnArgs {
  const void *q, *k, *v;
  void* o;
  const unsigned char* mask;  // [b][lk], 0 = hidden; may be null
  int b, h, hk, d;
  long lq, lk;
  long q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh, o_sb, o_sl, o_sh, m_sb;
  float scale_log2;  // scale * log2 e
};

constexpr int ATTN_ANY_D = 256;  // widest head of the general kernel
constexpr int ATTN_ANY_WARPS = 4;

// General form, any strides and head widths up to 256, for operands that TMA cannot read
// and for no keys at all: one warp per query, 32 keys a step; a lane holds one key's score,
// then the channels lane, lane + 32, ... Bound by its scattered reads of K: 42 ms where the
// tensor-core form takes 0.12 ms (4 x 2040 x 2040, 16 heads of 32).
template <typename T>
__global__ void __launch_bounds__(32 * ATTN_ANY_WARPS) attn_any_kernel(const AttnArgs a) {
  __shared__ float sq[ATTN_ANY_WARPS][ATTN_ANY_D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long tiles = (a.lq + ATTN_ANY_WARPS - 1) / ATTN_ANY_WARPS, bh = blockIdx.x / tiles;
  const long i = (blockIdx.x - bh * tiles) * ATTN_ANY_WARPS + warp;
  if (i >= a.lq) return;
  const int b = (int)(bh / a.h), h = (int)(bh - (long)b * a.h), hk = h / (a.h / a.hk);
  const T* q = static_cast<const T*>(a.q) + b * a.q_sb + i * a.q_sl + h * a.q_sh;
  const T* k = static_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh;
  const T* v = static_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh;
  const unsigned char* mask = a.mask ? a.mask + b * a.m_sb : nullptr;
  for (int c = lane; c < a.d; c += 32) sq[warp][c] = to_f32(q[c]) * a.scale_log2;
  __syncwarp();
  float m = -INFINITY, l = 0.f, o[ATTN_ANY_D / 32];
#pragma unroll
  for (int c = 0; c < ATTN_ANY_D / 32; ++c) o[c] = 0.f;
  for (long j0 = 0; j0 < a.lk; j0 += 32) {
    const long j = j0 + lane;
    const bool seen = j < a.lk && (!mask || mask[j]);
    const unsigned any = __ballot_sync(0xffffffffu, seen);
    if (!any) continue;
    float s = -INFINITY;
    if (seen) {
      s = 0.f;
      const T* kj = k + j * a.k_sl;
      for (int c = 0; c < a.d; ++c) s += sq[warp][c] * to_f32(kj[c]);
    }
    float top = s;
    for (int x = 16; x >= 1; x /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    // (a step whose visible scores are all -inf gets the lowest finite maximum, so that they weigh
    // nothing beside a finite score of another step; alone they leave l at 0, and 0 / 0 is NaN)
    const float m2 = fmaxf(fmaxf(m, top), -FLT_MAX);
    const float keep = m == -INFINITY ? 0.f : exp2f(m - m2);
    const float p = seen ? exp2f(s - m2) : 0.f;
    float sum = p;
    for (int x = 16; x >= 1; x /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    l = l * keep + sum;
    m = m2;
#pragma unroll
    for (int c = 0; c < ATTN_ANY_D / 32; ++c) o[c] *= keep;
    for (int t = 0; t < 32; ++t) {
      if (!(any >> t & 1)) continue;
      const float pt = __shfl_sync(0xffffffffu, p, t);
      const T* vj = v + (j0 + t) * a.v_sl;
#pragma unroll
      for (int c = 0; c < ATTN_ANY_D / 32; ++c)
        if (lane + 32 * c < a.d) o[c] += pt * to_f32(vj[lane + 32 * c]);
    }
  }
  T* out = static_cast<T*>(a.o) + b * a.o_sb + i * a.o_sl + h * a.o_sh;
  const bool none = m == -INFINITY;  // no visible key
#pragma unroll
  for (int c = 0; c < ATTN_ANY_D / 32; ++c)
    if (lane + 32 * c < a.d) out[lane + 32 * c] = from_f32<T>(none ? 0.f : o[c] / l);
}

}  // namespace scb
