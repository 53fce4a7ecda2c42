// Attention on the tensor cores (heads up to 128 channels wide, K and V in TMA's alignment).
//
// Rows: the R = H / Hk query heads that share a key head are packed with their queries into
// one list of Lq R rows (row = query * R + head), so K and V are read once for all of them.
// A unit is a picture's key head and 256 rows (two tiles of 128, sharing every K and V
// tile), or 128 rows when there are no more: then both tiles hold the same rows and take
// the even and the odd key tiles (`twin`), which keeps two score tiles in flight.
//
// Work: all units' key tiles in one line, cut into equal ranges, one per CTA. A CTA walks
// the units its range touches. A unit that lies in one range is written to the output at
// once; of a unit that is cut, every piece goes to the workspace as float32 sums with its
// maximum and total, and attn_join_kernel adds them in order (no atomics).
//
// CTA: warps 0-3 and 4-7 are the softmax of tile 0 and 1, one thread a row; warp 8 issues
// the matrix products, warp 9 the TMA loads of K and V into a ring of 128-key slots (warps
// 10 and 11 fill their warpgroup up, which gives registers to the softmax).
//   S_t = Q_t K^T    M 128, N 128, K d        TMEM columns [128 t, +128)
//   P_t = 2^(c S - c m), 16-bit               columns [128 t, +64), over S
//   O_t += P_t V     M 128, N d, K 128        columns [256 + 128 t, +d), A from TMEM
// While one tile's softmax runs, the tensor cores compute the other tile's products. The
// maximum m that a row subtracts is raised only when a tile exceeds it by 2^8 (in P): sums
// are float32 and P at most 256, so a stale m changes no result, and O, which lives in
// TMEM, is rescaled only then.
#pragma once
#include "op_attn.cuh"

namespace scb {

constexpr int AT_KEYS = 128;               // keys of a tile
constexpr int AT_THREADS = 384;            // launched with 168 registers a thread
constexpr float AT_STALE = 8.f;            // log2 by which a tile may exceed m
constexpr int AT_BOX = AT_KEYS * 128;      // bytes of 128 rows x 64 channels

struct AttnTcArgs {
  AttnArgs a;
  int share;          // R
  long rows;          // Lq R
  int twin;           // both tiles on the same rows
  int unit_rows;      // 256, or 128 with twin
  long row_units;     // units of one (picture, key head)
  long units, tiles;  // all units; key tiles of each
  long total;         // units * tiles
  int kv_b, kv_h;     // 1 where K / V differ by picture / head (0: broadcast), bit 0 K, bit 1 V
  int qneg;           // the scale is negative (Q is negated) or, 2, zero (Q is cleared)
  float* part;        // pieces: [grid][2][256][d] sums, then [grid][2][256] (m c, l)
  float2* part_ml;
  int q_wide, o_wide; // 16-byte accesses to Q and the output allowed
};

__device__ __forceinline__ long at_start(const AttnTcArgs& g, long cta, long grid) { return cta * g.total / grid; }
// The CTA whose range holds tile x.
__device__ __forceinline__ long at_owner(const AttnTcArgs& g, long x, long grid) { return ((x + 1) * grid - 1) / g.total; }

template <typename T>
__device__ __forceinline__ uint32_t at_pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t at_pack<__half>(float a, float b) {
  return pack_half2(a, b);
}
template <>
__device__ __forceinline__ uint32_t at_pack<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Boxes: 64-channel halves of a head (1 or 2); Slots: K and V tiles in the ring.
template <int Boxes>
struct AtLayout {
  static constexpr int kTile = Boxes * AT_BOX;            // one Q, K or V tile
  static constexpr int kSlots = Boxes == 1 ? 10 : 5;
  static constexpr int kQ = 0;
  static constexpr int kRing = 2 * kTile;
  static constexpr int kBars = kRing + kSlots * kTile;
  static constexpr int kSmem = kBars + 256 + 1024;        // + alignment to 1 KB
};

// A bounded wait that gives up at once when another wait of the CTA has given up.
__device__ __forceinline__ void at_wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
  if (mbar_try_wait(bar, parity)) return;
  if (*dead) return;
  if (!mbar_wait(bar, parity, SCB_ERR_WAIT_ATTN)) *dead = 1;
}

template <typename T, int Boxes>
__global__ void __launch_bounds__(AT_THREADS, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
               const __grid_constant__ AttnTcArgs g) {
  using L = AtLayout<Boxes>;
  extern __shared__ uint8_t at_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(at_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::kBars);
  uint64_t* empty = full + L::kSlots;
  uint64_t* q_ready = empty + L::kSlots;
  uint64_t* s_full = q_ready + 2;
  uint64_t* p_ready = s_full + 2;
  uint64_t* o_done = p_ready + 2;
  uint64_t* drain = o_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < L::kSlots; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(q_ready + t, 128);
      mbar_init(s_full + t, 1);
      mbar_init(p_ready + t, 128);
      mbar_init(o_done + t, 1);
    }
    mbar_init(drain, 1);
    *dead = 0;
    mbar_fence_init();
  }
  if (warp == 8) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const long x0 = at_start(g, blockIdx.x, gridDim.x), x1 = at_start(g, blockIdx.x + 1, gridDim.x);
  const int d = g.a.d, ksteps = (d + 15) / 16;

  // 384 x 168 = 64512 registers at launch; 256 x 208 + 128 x 80 = 63488 after the two splits
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 9 && lane == 0) {
      // ---- TMA: K and V tiles into the ring, in the order of their use
      uint32_t seq = 0;
      for (long x = x0; x < x1;) {
        const long unit = x / g.tiles, j0 = x - unit * g.tiles, n = min(x1 - x, g.tiles - j0);
        const long bh = unit / g.row_units;
        const int b = (int)(bh / g.a.hk), h = (int)(bh - (long)b * g.a.hk);
        for (long j = j0; j < j0 + n; ++j)
          for (int w = 0; w < 2; ++w, ++seq) {  // K, V
            const uint32_t slot = seq % L::kSlots, turn = seq / L::kSlots;
            if (turn) at_wait(empty + slot, (turn - 1) & 1, dead);
            if (*dead) break;
            mbar_arrive_expect_tx(full + slot, L::kTile);
            for (int c = 0; c < Boxes; ++c)
              tma_load_4d(sm + L::kRing + slot * L::kTile + c * AT_BOX, w ? &tv : &tk, full + slot, 64 * c,
                          (int)(j * AT_KEYS), (g.kv_h >> w & 1) * h, (g.kv_b >> w & 1) * b);
          }
        x += n;
      }
      // after a wait gave up, loads may still be on their way: none may outlive the CTA
      if (*dead)
        for (uint32_t back = 1; back <= L::kSlots && back <= seq; ++back) {
          const uint32_t s = seq - back;
          mbar_wait(full + s % L::kSlots, (s / L::kSlots) & 1, SCB_ERR_WAIT_ATTN);
        }
    } else if (warp == 8 && lane == 0) {
      // ---- matrix products
      const uint32_t sb = smem_u32(sm);
      constexpr bool kBf = sizeof(T) == 2 && !__is_same(T, __half);
      constexpr uint32_t fmt = kBf ? (1u << 7) | (1u << 10) : 0u;
      const uint32_t id_s = make_idesc_f16(128, 128) | fmt;
      const uint32_t id_o = make_idesc_f16_bmn(128, 16 * ksteps) | fmt;
      uint32_t cnt[2] = {0, 0}, segs[2] = {0, 0}, base = 0;
      auto scores = [&](int t, uint32_t jj, bool release) {
        const uint32_t seq = 2 * jj, slot = seq % L::kSlots;
        at_wait(full + slot, (seq / L::kSlots) & 1, dead);
        tc_fence_after();
        const uint32_t q = sb + L::kQ + t * L::kTile, k = sb + L::kRing + slot * L::kTile;
        for (int s = 0; s < ksteps; ++s) {
          const uint32_t o = (s >> 2) * AT_BOX + (s & 3) * 32;
          umma_f16(tmem + 128 * t, make_sdesc(q + o, 128, SW_128B), make_sdesc(k + o, 128, SW_128B), id_s, s > 0);
        }
        umma_commit(s_full + t);
        if (release) umma_commit(empty + slot);
      };
      for (long x = x0; x < x1;) {
        const long unit = x / g.tiles, j0 = x - unit * g.tiles;
        const uint32_t n = (uint32_t)min(x1 - x, g.tiles - j0);
        const uint32_t nt[2] = {g.twin ? (n + 1) / 2 : n, g.twin ? n / 2 : n};
        for (int t = 0; t < 2; ++t) {
          if (!nt[t]) continue;
          at_wait(q_ready + t, segs[t]++ & 1, dead);
          tc_fence_after();
          scores(t, base + (g.twin ? t : 0), g.twin || t == 1);
        }
        for (uint32_t i = 0; i < nt[0]; ++i)
          for (int t = 0; t < 2; ++t) {
            if (i >= nt[t]) continue;
            const uint32_t jj = base + (g.twin ? 2 * i + t : i);
            at_wait(p_ready + t, cnt[t] & 1, dead);
            const uint32_t seq = 2 * jj + 1, slot = seq % L::kSlots;
            at_wait(full + slot, (seq / L::kSlots) & 1, dead);
            tc_fence_after();
            const uint32_t v = sb + L::kRing + slot * L::kTile;
#pragma unroll
            for (int s = 0; s < AT_KEYS / 16; ++s)
              umma_f16_ts(tmem + 256 + 128 * t, tmem + 128 * t + 8 * s,
                          make_sdesc_lbo_sbo(v + 2048 * s, AT_BOX, 1024, SW_128B), id_o, i > 0 || s > 0);
            umma_commit(o_done + t);
            if (g.twin || t == 1) umma_commit(empty + slot);
            if (i + 1 < nt[t]) {
              // S_t overwrites P_t, so P_t V must have read it; the other tile's softmax
              // runs meanwhile
              at_wait(o_done + t, cnt[t] & 1, dead);
              scores(t, base + (g.twin ? 2 * (i + 1) + t : i + 1), g.twin || t == 1);
            }
            ++cnt[t];
            if (*dead) break;
          }
        base += n;
        x += n;
      }
      if (*dead) {  // products may still be running on TMEM and shared memory
        umma_commit(drain);
        mbar_wait(drain, 0, SCB_ERR_WAIT_ATTN);
      }
    }
  } else {
    // ---- softmax: tile t, one thread a row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = warp >> 2, row = tid & 127;
    const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t ts = trow + 128 * t, to = trow + 256 + 128 * t;
    uint8_t* sq = sm + L::kQ + t * L::kTile;
    const float c = g.a.scale_log2, stale = fminf(AT_STALE / c, 1e30f);
    uint32_t cnt = 0, base = 0;
    for (long x = x0; x < x1;) {
      const long unit = x / g.tiles, j0 = x - unit * g.tiles, n = min(x1 - x, g.tiles - j0);
      const long bh = unit / g.row_units;
      const int b = (int)(bh / g.a.hk), hk = (int)(bh - (long)b * g.a.hk);
      const long r = (unit - bh * g.row_units) * g.unit_rows + (g.twin ? 0 : 128 * t) + row;
      const bool on = r < g.rows;
      const long ql = on ? r / g.share : 0;
      const int qh = hk * g.share + (int)(on ? r - ql * g.share : 0);
      const long step = g.twin ? 2 : 1, jt = j0 + (g.twin ? t : 0);
      const bool any = jt < j0 + n;
      if (any) {
        // this row of Q, zeros past the last row and channel; K-major, 128-byte swizzle
        const T* q = static_cast<const T*>(g.a.q) + b * g.a.q_sb + ql * g.a.q_sl + qh * g.a.q_sh;
        const uint32_t flip = g.qneg == 1 ? 0x80008000u : 0u;
        for (int k = 0; k < 2 * ksteps; ++k) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (on && g.qneg < 2) {
            if (g.q_wide && 8 * k + 8 <= d) {
              v = *reinterpret_cast<const uint4*>(q + 8 * k);
            } else {
              const unsigned short* e = reinterpret_cast<const unsigned short*>(q);
              unsigned w[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) w[i] = 8 * k + i < d ? e[8 * k + i] : 0;
              v = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
            }
            v.x ^= flip;
            v.y ^= flip;
            v.z ^= flip;
            v.w ^= flip;
          }
          *reinterpret_cast<uint4*>(sq + (k >> 3) * AT_BOX + swz_off(row, k & 7, 128)) = v;
        }
        fence_proxy_async_smem();
        mbar_arrive(q_ready + t);
      }
      const unsigned char* mask = g.a.mask ? g.a.mask + b * g.a.m_sb : nullptr;
      float m = -INFINITY, l = 0.f;
      for (long j = jt; j < j0 + n; j += step) {
        // which keys of the tile are visible, one bit each
        uint32_t seen[4];
        {
          const long key = j * AT_KEYS + lane;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const long k = key + 32 * i;
            seen[i] = __ballot_sync(0xffffffffu, k < g.a.lk && (!mask || mask[k]));
          }
        }
        at_wait(s_full + t, cnt & 1, dead);
        tc_fence_after();
        float s[128];
        {
          uint32_t u[128];
#pragma unroll
          for (int i = 0; i < 8; ++i) tmem_ld16_issue(ts + 16 * i, u + 16 * i);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            tmem_fence16(u + 16 * i);
            u32_to_f32_16(u + 16 * i, s + 16 * i);
          }
        }
        const bool part = (seen[0] & seen[1] & seen[2] & seen[3]) != 0xffffffffu;
        if (part) {
#pragma unroll
          for (int i = 0; i < 128; ++i) s[i] = seen[i >> 5] >> (i & 31) & 1 ? s[i] : -INFINITY;
          if (mask) {
            // hidden values may be NaN or infinite, and 0 times those is NaN: clear them
            const uint32_t seq = 2 * (base + (uint32_t)(j - j0)) + 1, slot = seq % L::kSlots;
            at_wait(full + slot, (seq / L::kSlots) & 1, dead);
            const uint32_t word = (row >> 5) == 0 ? seen[0] : (row >> 5) == 1 ? seen[1] : (row >> 5) == 2 ? seen[2] : seen[3];
            if (!(word >> (row & 31) & 1)) {
              uint4* v = reinterpret_cast<uint4*>(sm + L::kRing + slot * L::kTile + row * 128);
              for (int k = 0; k < 8; ++k) {
                v[k] = make_uint4(0, 0, 0, 0);
                if (Boxes == 2) v[AT_BOX / 16 + k] = make_uint4(0, 0, 0, 0);
              }
            }
            fence_proxy_async_smem();
          }
        }
        const float top = row_max<128>(s);
        if (j == jt) {
          m = top;
        } else {
          const bool raise = top > m + stale;
          if (__any_sync(0xffffffffu, raise)) {
            // P_t V of the tile before is complete (S_t was issued after it)
            const float f = raise ? ex2_approx((m - top) * c) : 1.f;
            m = raise ? top : m;
            l *= f;
            for (int i = 0; i < ksteps; ++i) {
              float o[16];
              tmem_ld16(to + 16 * i, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= f;
              tmem_st16(to + 16 * i, o);
            }
          }
        }
        const float mc = m == -INFINITY ? 0.f : -m * c;
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 y = __ffma2_rn(make_float2(s[32 * i + 2 * e], s[32 * i + 2 * e + 1]), make_float2(c, c),
                                        make_float2(mc, mc));
            const float2 v = make_float2(ex2_approx(y.x), ex2_approx(y.y));
            sum[e & 1] = __fadd2_rn(sum[e & 1], v);
            p[e] = at_pack<T>(v.x, v.y);
          }
          tmem_st16u(ts + 16 * i, p);
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(p_ready + t);
        ++cnt;
      }
      // ---- the unit's rows: to the output when the unit is whole, else to the workspace
      if (any) {
        at_wait(o_done + t, (cnt - 1) & 1, dead);
        tc_fence_after();
      }
      if (!g.twin && n == g.tiles) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T* o = static_cast<T*>(g.a.o) + b * g.a.o_sb + ql * g.a.o_sl + qh * g.a.o_sh;
        for (int i = 0; i < ksteps; ++i) {
          float v[16];
          tmem_ld16(to + 16 * i, v);
          if (!on) continue;
          if (g.o_wide && 16 * i + 16 <= d) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = at_pack<T>(v[2 * e] * inv, v[2 * e + 1] * inv);
            *reinterpret_cast<uint4*>(o + 16 * i) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(o + 16 * i + 8) = make_uint4(w[4], w[5], w[6], w[7]);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (16 * i + e < d) o[16 * i + e] = from_f32<T>(v[e] * inv);
          }
        }
      } else {
        const long at = (2L * blockIdx.x + (x == x0 ? 0 : 1)) * 256 + 128 * t + row;
        if (on) g.part_ml[at] = make_float2(m == -INFINITY ? m : m * c, l);
        float* o = g.part + at * d;
        for (int i = 0; i < ksteps; ++i) {
          float v[16];
          if (any) tmem_ld16(to + 16 * i, v);
          if (!on) continue;
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (16 * i + e < d) o[16 * i + e] = any ? v[e] : 0.f;
        }
      }
      tc_fence_before();
      base += (uint32_t)n;
      x += n;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

// Adds the pieces of the units that were cut: one warp a row.
//   o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i, M the largest m_i
template <typename T>
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ AttnTcArgs g, int grid) {
  const int lane = threadIdx.x & 31, d = g.a.d;
  const long w = (long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const long unit = w / g.unit_rows;
  const int row = (int)(w - unit * g.unit_rows);
  if (unit >= g.units) return;
  const long bh = unit / g.row_units, r = (unit - bh * g.row_units) * g.unit_rows + row;
  if (r >= g.rows) return;
  const long t0 = unit * g.tiles, c0 = at_owner(g, t0, grid), c1 = at_owner(g, t0 + g.tiles - 1, grid);
  if (c0 == c1 && !g.twin) return;  // written by its CTA
  const int subs = g.twin ? 2 : 1;
  const int pieces = (int)(c1 - c0 + 1) * subs;
  auto place = [&](int i) {
    const long cta = c0 + i / subs;
    return (2 * cta + (at_start(g, cta, grid) >= t0 ? 0 : 1)) * 256 + row + 128 * (i % subs);
  };
  float top = -INFINITY;
  for (int i = lane; i < pieces; i += 32) top = fmaxf(top, g.part_ml[place(i)].x);
  for (int k = 16; k >= 1; k /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
  float o[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
  for (int i = 0; i < pieces; ++i) {
    const long at = place(i);
    const float2 ml = g.part_ml[at];
    const float f = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - top);
    l += f * ml.y;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (lane + 32 * k < d && f != 0.f) o[k] += f * g.part[at * d + lane + 32 * k];
  }
  const int b = (int)(bh / g.a.hk), hk = (int)(bh - (long)b * g.a.hk);
  const long ql = r / g.share;
  const int qh = hk * g.share + (int)(r - ql * g.share);
  T* out = static_cast<T*>(g.a.o) + b * g.a.o_sb + ql * g.a.o_sl + qh * g.a.o_sh;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (lane + 32 * k < d) out[lane + 32 * k] = from_f32<T>(l == 0.f ? 0.f : o[k] / l);
}

}  // namespace scb
