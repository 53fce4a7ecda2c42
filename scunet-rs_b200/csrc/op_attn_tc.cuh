// Attention on the tensor cores (heads up to 128 channels wide, K and V in TMA's alignment).
//
// Rows: the R = H / Hk query heads that share a key head are packed with their queries into
// one list of Lq R rows (row = query * R + head), so K and V are read once for all of them.
// A unit is a picture's key head and 256 rows (two tiles of 128, sharing every K and V
// tile), or 128 rows when there are no more: then both tiles hold the same rows and take
// the even and the odd key tiles (`twin`), which keeps two score tiles in flight.
//
// Work: all units' key tiles in one line, cut into equal ranges, one per CTA (at_start). A CTA walks
// the units its range touches. A unit that lies in one range is written to the output at
// once; of a unit that is cut, every piece goes to the workspace as float32 sums with its
// maximum and total, and attn_join_kernel adds them in order (no atomics).
//
// CTA: warps 0-7 and 8-15 are the softmax of tile 0 and 1, two threads a row with 64 keys
// each; warps 16 and 17 issue the matrix products of tile 0 and 1, warp 18 the TMA loads of
// K and V into a ring of 128-key slots (warp 19 fills the warpgroup up, which gives
// registers to the softmax).
//   S_t = Q_t K^T    M 128, N 128, K d        TMEM columns [128 t, +128)
//   P_t = 2^(c S - c m + AT_LIFT), 16-bit     64 columns
//   O_t += P_t V     M 128, N d, K 128        columns [256 + 64 or 128 t, +d), A from TMEM
// Heads up to 64 wide leave columns for P_t beside S_t, and wider ones keep P_t in shared
// memory, so the next S_t is computed as soon as this one is in registers (Twin with wide
// heads: P_t lies over S_t, and the next S_t waits for P_t V). While one tile's softmax
// runs, the tensor cores compute the other tile's products. The maximum m that a row
// subtracts is raised only when a tile exceeds it by 2^8 (in P): sums are float32 and P at
// most 256 (2^15 with AT_LIFT), so a stale m changes no result, and O, which lives in TMEM, is rescaled only
// then. m is -inf while no key was visible and at least AT_LOWEST after that, so the end can
// tell rows that see nothing (zeros) from rows whose visible scores are all -inf (0 / 0, NaN):
// the weights of any other row sum up to 1 or more.
//
// Precision: scores, maxima, sums and O are float32, exponentials those of the special function
// unit (2 ulp); the weights are rounded to the operands' type for P V, which the tensor cores
// want alike, and which makes the result's error 1.4 times that of its own rounding.
//
// Bound: the softmax. A pair of 128 x 128 tiles takes 2048 cycles of the special function
// units (the softmax alone, without products or waits, measured 2190 with 16 warps and 2712
// with 8) and 2830 here with heads up to 64; 3270 with heads of 128 whose keys come from L2,
// 4060 from DRAM (2048 of them products). Between two units of a CTA 5000 to 6000 cycles pass
// without either (heads of 32), 15000 with heads of 128, and the join of cut units adds 11 to 28
// us. 4 x 2040 x 2040, 16 heads of 32 fp16: 121 us. 8160 queries and keys, 8 heads of 128 bf16:
// 267 us at 1.9 GHz, 297 us where the power limit holds the clock at 1.7 (918 TFLOP/s). One query
// over 32640 keys, 2 x 16 heads of 64 fp16: 66 us (4.1 TB/s), 12 of them the join.
#pragma once
#include <cfloat>

#include "op_attn.cuh"

namespace scb {

constexpr int AT_KEYS = 128;               // keys of a tile
constexpr int AT_THREADS = 640;
constexpr int AT_REGS = 96;                // registers a thread at launch (checked there)
constexpr float AT_STALE = 8.f;            // log2 by which a tile may exceed m
// log2 by which weights (and so their sums and O) are kept larger than 2^(c S - c m): 2^15 at
// most with AT_STALE. fp16 loses what is below 2^-25, which a long faint tail would show: this
// way that is 2^-32 of the row's largest weight, 2^-32 times the keys in all.
template <typename T>
constexpr float AT_LIFT = __is_same(T, __half) ? 7.f : 0.f;
constexpr float AT_LOWEST = -FLT_MAX;      // m of visible scores that are all -inf
constexpr int AT_BOX = AT_KEYS * 128;      // bytes of 128 rows x 64 channels

constexpr uint32_t AT_NONE = 0xffffffffu;

struct AttnTcArgs {
  AttnArgs a;
  int share;          // R
  long rows;          // Lq R
  int twin;           // both tiles on the same rows
  int unit_rows;      // 256, or 128 with twin
  int cuts;           // pieces of a twin unit
  int turns;          // twin: the tiles' exponentials take turns
  long row_units;     // units of one (picture, key head)
  long units, tiles;  // all units; key tiles of each
  long total;         // units * tiles
  int kv_b, kv_h;     // 1 where K / V differ by picture / head (0: broadcast), bit 0 K, bit 1 V
  int qneg;           // the scale is negative (Q is negated) or, 2, zero (Q is cleared)
  float* part;        // pieces, two of a CTA (its first and last unit), one with twin:
                      // [pieces][d][256] sums, then [pieces][256] (m c, l)
  float2* part_ml;
  int q_wide, o_wide; // 16-byte accesses to Q and the output allowed
  uint32_t lose;      // the load that CTA 0 leaves out (scb_probe_attention_lost), else AT_NONE
};

// Tiles [at_start(cta), at_start(cta + 1)) of the line. Twin units are cut into `cuts` equal
// pieces instead, one a CTA, pieces of one place next to each other in the grid: all heads
// then walk the same keys at the same time, and a token's heads lie in the same DRAM page.
__device__ __forceinline__ long at_start(const AttnTcArgs& g, long cta, long grid) { return cta * g.total / grid; }
__device__ __forceinline__ void at_range(const AttnTcArgs& g, long cta, long grid, long& x0, long& x1) {
  if (g.twin) {
    const long cut = cta / g.units, unit = cta - cut * g.units;
    x0 = unit * g.tiles + g.tiles * cut / g.cuts;
    x1 = unit * g.tiles + g.tiles * (cut + 1) / g.cuts;
  } else {
    x0 = at_start(g, cta, grid);
    x1 = at_start(g, cta + 1, grid);
  }
}
// The CTA whose range holds tile x.
__device__ __forceinline__ long at_owner(const AttnTcArgs& g, long x, long grid) {
  return ((x + 1) * grid - 1) / g.total;
}

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

// 1 / l of a row's final sum: 0 when no key was visible, NaN when nothing was above -inf.
__device__ __forceinline__ float at_inverse(float m, float l) {
  return m == -INFINITY && l == l ? 0.f : l >= 0.5f ? 1.f / l : NAN;
}

// A sum of weights as it is, or NaN when a weight was (weights are at most 2^15, so a sum of
// them stays far below 1e30).
__device__ __forceinline__ float at_total(float l) { return l < 1e30f ? l : NAN; }

// Whether `p` holds for any of the 256 threads of barrier `id`, which all arrive.
__device__ __forceinline__ bool at_any(int id, bool p) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %2, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"((uint32_t)p)
      : "memory");
  return r != 0;
}
// The two tiles' exponentials take turns: a tile waits for its turn, and gives the other
// tile's half-way through its own (512 threads: 256 wait, 256 give).
__device__ __forceinline__ void at_turn_wait(int t) {
  asm volatile("barrier.cta.sync %0, 512;" ::"r"(3 + t) : "memory");
}
__device__ __forceinline__ void at_turn_give(int t) {
  asm volatile("barrier.cta.arrive %0, 512;" ::"r"(4 - t) : "memory");
}
__device__ __forceinline__ void at_sync(int id) { asm volatile("barrier.cta.sync %0, 256;" ::"r"(id) : "memory"); }

// Boxes: 64-channel halves of a head (1 or 2); Slots: K and V tiles in the ring.
template <int Boxes, bool Twin>
struct AtLayout {
  static constexpr int kTile = Boxes * AT_BOX;            // one Q, K or V tile
  // Where P_t lies: beside S_t in TMEM for heads up to 64 wide; in shared memory for wider
  // ones, where S and O fill TMEM, at the price of two ring slots (8160 x 8160 x 8 x 128 in
  // short runs: 293 us over S_t, 272 us so when it came in; where every key is read from DRAM for
  // 256 rows only, 159 and 179 us); over S_t with Twin, whose tiles need two slots each
  static constexpr bool kSharedP = Boxes == 2 && !Twin;
  static constexpr bool kOwnP = Boxes == 1 || kSharedP;
  static constexpr int kSlots = Boxes == 1 ? 10 : kSharedP ? 3 : 4;
  static_assert(!Twin || kSlots % 2 == 0, "each tile of Twin has half of the ring");
  static constexpr int kQ = 0;
  static constexpr int kPTile = 2 * AT_BOX;               // 128 rows x 128 keys
  static constexpr int kSharedPAt = 2 * kTile;
  static constexpr int kRing = kSharedPAt + (kSharedP ? 2 * kPTile : 0);
  static constexpr int kBars = kRing + kSlots * kTile;
  // full and empty of every slot, six pairs of barriers, the TMEM address, `dead`
  static constexpr int kRow = kBars + 8 * (2 * kSlots + 12) + 8;  // [2 tiles][2 halves][128] floats
  static constexpr int kSmem = kRow + 2048;
  // TMEM columns: S_t at 128 t; then O_t; P_t (no meaning with kSharedP)
  static constexpr int kO = 256, kOStep = 64 * Boxes;
  static constexpr int kP = Boxes == 1 ? 384 : 0, kPStep = Boxes == 1 ? 64 : 128;
};

// One lane of a converged warp. Selecting the issuing thread this way instead of by lane
// number lets the compiler keep descriptors in uniform registers: eight products were
// issued in 780 cycles before.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// The ring place of a K or V tile, and how often the place was filled before. The tiles of
// Twin have a half of the ring each: a wait tells a filling only from the one before it, and
// in a shared ring a tile could be two fillings ahead of loads that only the other waits for.
template <bool Twin, int Slots>
struct AtPlace {
  uint32_t slot, turn;
  __device__ __forceinline__ explicit AtPlace(uint32_t seq) {
    if (Twin) {
      constexpr uint32_t kHalf = Slots / 2;
      const uint32_t own = (seq >> 2) * 2 + (seq & 1);  // seq: K V of tile 0, K V of tile 1, ...
      slot = (seq >> 1 & 1) * kHalf + own % kHalf;
      turn = own / kHalf;
    } else {
      slot = seq % Slots;
      turn = seq / Slots;
    }
  }
};

// A bounded wait that gives up at once when another wait of the CTA has given up. The error
// word tells the place of the first one that did. `dead` is set before anything that depends on
// the lost handshake goes on, so whoever writes rows finds it set, and writes NaN.
enum : unsigned {
  AT_EMPTY = 0x100,
  AT_FULL = 0x200,
  AT_Q = 0x300,
  AT_S = 0x400,
  AT_FREE = 0x500,
  AT_P = 0x600,
  AT_O = 0x700,
};
__device__ __forceinline__ void at_wait(uint64_t* bar, uint32_t parity, volatile int* dead, unsigned place) {
  if (mbar_try_wait(bar, parity)) return;
  if (*dead) return;
  if (!mbar_wait(bar, parity, SCB_ERR_WAIT_ATTN | place)) *dead = 1;
}

template <typename T, int Boxes, bool Twin>
__global__ void __launch_bounds__(AT_THREADS, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
               const __grid_constant__ AttnTcArgs g) {
  using L = AtLayout<Boxes, Twin>;
  using Place = AtPlace<Twin, L::kSlots>;
  extern __shared__ __align__(1024) uint8_t sm[];  // the swizzled tiles' alignment
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::kBars);
  uint64_t* empty = full + L::kSlots;
  uint64_t* q_ready = empty + L::kSlots;
  uint64_t* s_full = q_ready + 2;
  uint64_t* p_ready = s_full + 2;
  uint64_t* o_done = p_ready + 2;
  uint64_t* s_free = o_done + 2;
  uint64_t* drain = s_free + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  let_next_start();
  if (tid == 0) {
    for (int i = 0; i < L::kSlots; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, Twin ? 1 : 2);  // the tiles that read the slot
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(q_ready + t, 256);
      mbar_init(s_full + t, 1);
      mbar_init(p_ready + t, 256);
      mbar_init(o_done + t, 1);
      mbar_init(s_free + t, 256);
      mbar_init(drain + t, 1);
    }
    *dead = 0;
    mbar_fence_init();
  }
  if (warp == 16) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  long x0, x1;
  at_range(g, blockIdx.x, gridDim.x, x0, x1);
  const int d = g.a.d, ksteps = (d + 15) / 16;

  // 640 x 96 = 61440 registers at launch, 512 x 104 + 128 x 64 = 61440 after the split
  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 18 && elect_one()) {
      // ---- TMA: K and V tiles into the ring, in the order of their use
      uint32_t seq = 0;
      for (long x = x0; x < x1;) {
        const long unit = x / g.tiles, j0 = x - unit * g.tiles, n = min(x1 - x, g.tiles - j0);
        const long bh = unit / g.row_units;
        const int b = (int)(bh / g.a.hk), h = (int)(bh - (long)b * g.a.hk);
        for (long j = j0; j < j0 + n; ++j)
          for (int w = 0; w < 2; ++w, ++seq) {  // K, V
            const Place at(seq);
            if (at.turn) at_wait(empty + at.slot, (at.turn - 1) & 1, dead, AT_EMPTY);
            if (*dead) break;
            mbar_arrive_expect_tx(full + at.slot, L::kTile);
            if (seq == g.lose && blockIdx.x == 0) continue;
            for (int c = 0; c < Boxes; ++c)
              tma_load_4d(sm + L::kRing + at.slot * L::kTile + c * AT_BOX, w ? &tv : &tk, full + at.slot, 64 * c,
                          (int)(j * AT_KEYS), (g.kv_h >> w & 1) * h, (g.kv_b >> w & 1) * b);
          }
        x += n;
      }
      // after a wait gave up, loads may still be on their way: none may outlive the CTA. Each
      // place's last filling is waited for (a wait for one before it, with the same parity as
      // the filling after, would run out)
      if (*dead) {
        uint32_t waited = 0;
        for (uint32_t back = 1; back <= 2 * L::kSlots && back <= seq; ++back) {
          const Place at(seq - back);
          if (waited >> at.slot & 1) continue;
          waited |= 1u << at.slot;
          mbar_wait(full + at.slot, at.turn & 1, SCB_ERR_WAIT_ATTN);
        }
      }
    } else if (warp < 18 && elect_one()) {
      // ---- matrix products of tile t
      const int t = warp - 16;
      const uint32_t sb = smem_u32(sm);
      constexpr uint32_t fmt = __is_same(T, __half) ? 0u : (1u << 7) | (1u << 10);  // bf16 operands
      constexpr uint32_t id_s = make_idesc_f16(128, 128) | fmt;
      const uint32_t id_o = make_idesc_f16_bmn(128, 16 * ksteps) | fmt;
      const uint64_t dq = make_sdesc(sb + L::kQ + t * L::kTile, 128, SW_128B);
      const uint64_t dp = make_sdesc(sb + L::kSharedPAt + t * L::kPTile, 128, SW_128B);
      const uint64_t dk = make_sdesc(sb + L::kRing, 128, SW_128B);
      const uint64_t dv = make_sdesc_lbo_sbo(sb + L::kRing, AT_BOX, 1024, SW_128B);
      const uint32_t ts = tmem + 128 * t, tp = tmem + L::kP + L::kPStep * t, to = tmem + L::kO + L::kOStep * t;
      const uint32_t step = Twin ? 4 : 2;  // ring places from one K to the tile's next
      uint32_t cnt = 0, segs = 0, base = 0;
      const auto scores = [&](uint32_t seq) {
        const Place at(seq);
        at_wait(full + at.slot, at.turn & 1, dead, AT_FULL);
        tc_fence_after();
        const uint64_t k = dk + at.slot * (uint32_t)(L::kTile >> 4);
#pragma unroll
        for (int s = 0; s < 4 * Boxes; ++s) {
          const uint32_t o = ((s >> 2) * AT_BOX + (s & 3) * 32) >> 4;
          if (s < ksteps) umma_f16(ts, dq + o, k + o, id_s, s > 0);
        }
        umma_commit(s_full + t);
        umma_commit(empty + at.slot);
      };
      for (long x = x0; x < x1;) {
        const long unit = x / g.tiles, j0 = x - unit * g.tiles;
        const uint32_t n = (uint32_t)min(x1 - x, g.tiles - j0);
        const uint32_t nt = Twin ? (n + 1 - t) / 2 : n;
        uint32_t seq = 2 * (base + (Twin ? t : 0));  // of K; V is the next
        if (nt) {
          at_wait(q_ready + t, segs++ & 1, dead, AT_Q);
          tc_fence_after();
          scores(seq);
        }
        for (uint32_t i = 0; i < nt && !*dead; ++i, ++cnt, seq += step) {
          if (L::kOwnP && i + 1 < nt) {  // the next scores, as soon as S_t is in registers
            at_wait(s_free + t, cnt & 1, dead, AT_FREE);
            scores(seq + step);
          }
          const Place at(seq + 1);
          at_wait(full + at.slot, at.turn & 1, dead, AT_FULL);
          const uint64_t v = dv + at.slot * (uint32_t)(L::kTile >> 4);
          at_wait(p_ready + t, cnt & 1, dead, AT_P);
          tc_fence_after();
#pragma unroll
          for (int s = 0; s < AT_KEYS / 16; ++s)
            if constexpr (L::kSharedP)
              umma_f16(to, dp + (uint32_t)(((s >> 2) * AT_BOX + (s & 3) * 32) >> 4), v + (uint32_t)(2048 * s >> 4),
                       id_o, i > 0 || s > 0);
            else
              umma_f16_ts(to, tp + 8 * s, v + (uint32_t)(2048 * s >> 4), id_o, i > 0 || s > 0);
          umma_commit(o_done + t);
          umma_commit(empty + at.slot);
          if (!L::kOwnP && i + 1 < nt) {
            // S_t overwrites P_t, so P_t V must have read it; the other tile's softmax runs
            // meanwhile
            at_wait(o_done + t, cnt & 1, dead, AT_O);
            scores(seq + step);
          }
        }
        base += n;
        x += n;
      }
      if (*dead) {  // products may still be running on TMEM and shared memory
        umma_commit(drain + t);
        mbar_wait(drain + t, 0, SCB_ERR_WAIT_ATTN);
      }
    }
  } else {
    // ---- softmax: tile t, two threads a row (warps 8 t + w and 8 t + 4 + w)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const int t = warp >> 3, half = warp >> 2 & 1, row = tid & 127, id = 1 + t;
    const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t ts = trow + 128 * t + 64 * half, to = trow + L::kO + L::kOStep * t;
    const uint32_t tp = trow + L::kP + L::kPStep * t + 32 * half;
    uint8_t* sq = sm + L::kQ + t * L::kTile;
    uint8_t* sp = sm + L::kSharedPAt + t * L::kPTile + half * AT_BOX;
    float* mine = reinterpret_cast<float*>(sm + L::kRow) + 256 * t + 128 * half + row;
    const float* other = reinterpret_cast<float*>(sm + L::kRow) + 256 * t + 128 * (half ^ 1) + row;
    const float c = g.a.scale_log2, stale = fminf(AT_STALE / c, 1e30f);
    // the last tile, and its keys from this half's first on
    const int last = (int)(g.tiles - 1), tail = (int)(g.a.lk - (long)last * AT_KEYS) - 64 * half;
    uint32_t cnt = 0, base = 0;
    if ((!Twin || g.turns) && t == 1) at_turn_give(t);
    for (long x = x0; x < x1;) {
      const long unit = x / g.tiles, j0 = x - unit * g.tiles, n = min(x1 - x, g.tiles - j0);
      const long bh = unit / g.row_units;
      const int b = (int)(bh / g.a.hk), hk = (int)(bh - (long)b * g.a.hk);
      // Twin: tile 1 holds the rows turned by 64, so that few rows are on another scheduler of
      // the SM than tile 0's
      const int unit_row = Twin ? (row + 64 * t) & 127 : 128 * t + row;
      const long r = (unit - bh * g.row_units) * g.unit_rows + unit_row;
      const int step = Twin ? 2 : 1, jt = (int)j0 + (Twin ? t : 0), jn = (int)(j0 + n);
      const bool any = jt < jn;
      // row rr of this warp's 32 (or -1 past the last): its query and head
      const int warp_row = (warp & 3) * 32;
      const long r0 = r - lane;
      // a warp with no row left only keeps the others company (with 256 rows of a unit that is
      // rare, and looking costs 10 %)
      const bool live = !Twin || r0 < g.rows;
      const auto locate = [&](int rr, int64_t sb, int64_t sl, int64_t sh) -> long {
        const long x = r0 + rr;
        if (x >= g.rows) return -1;
        const long at = g.share == 1 ? x : x / g.share;
        return b * sb + at * sl + (hk * g.share + (x - at * g.share)) * sh;
      };
      const int chunks = 2 * ksteps, wide = chunks > 8 ? 16 : chunks > 4 ? 8 : 4;  // 16-byte chunks of a row
      if (any) {
        // this warp's 16 rows of Q, `wide` lanes a row; zeros past the last row and channel.
        // K-major, 128-byte swizzle
        const uint32_t flip = g.qneg == 1 ? 0x80008000u : 0u;
        const int k = lane & (wide - 1);
        for (int rr = 16 * half + lane / wide; rr < 16 * half + 16; rr += 32 / wide) {
          uint4 v = make_uint4(0, 0, 0, 0);
          const long at = locate(rr, g.a.q_sb, g.a.q_sl, g.a.q_sh);
          if (at >= 0 && g.qneg < 2 && k < chunks) {
            const T* q = static_cast<const T*>(g.a.q) + at + 8 * k;
            if (g.q_wide && 8 * k + 8 <= d) {
              v = *reinterpret_cast<const uint4*>(q);
            } else {
              const unsigned short* e = reinterpret_cast<const unsigned short*>(q);
              unsigned w[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) w[i] = 8 * k + i < d ? e[i] : 0;
              v = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
            }
            v.x ^= flip;
            v.y ^= flip;
            v.z ^= flip;
            v.w ^= flip;
          }
          if (k < chunks) *reinterpret_cast<uint4*>(sq + (k >> 3) * AT_BOX + swz_off(warp_row + rr, k & 7, 128)) = v;
        }
        fence_proxy_async_smem();
        mbar_arrive(q_ready + t);
      }
      const unsigned char* mask = g.a.mask ? g.a.mask + b * g.a.m_sb : nullptr;
      float m = -INFINITY, l = 0.f;
      const uint32_t first = cnt;
      unsigned char ahead[2] = {1, 1};  // the next tile's mask bytes, 0 past the last key
      const auto look = [&](int j) {
        if (!mask || j > last) return;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          ahead[i] = j < last || 32 * i + lane < tail ? mask[(long)j * AT_KEYS + 64 * half + 32 * i + lane] : 0;
      };
      look(jt);
      for (int j = jt; j < jn; j += step) {
        // which of this half's keys are visible, one bit each
        bool part = !mask && j == last && tail < 64;
        uint32_t seen[2];
        if (mask) {
#pragma unroll
          for (int i = 0; i < 2; ++i) seen[i] = __ballot_sync(0xffffffffu, ahead[i] != 0);
          part = (seen[0] & seen[1]) != 0xffffffffu;
          look(j + step);
        } else if (part) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int k = tail - 32 * i;
            seen[i] = k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1u;
          }
        }
        at_wait(s_full + t, cnt & 1, dead, AT_S);
        tc_fence_after();
        float s[64];
        if (live) {
          uint32_t u[64];
#pragma unroll
          for (int i = 0; i < 4; ++i) tmem_ld16_issue(ts + 16 * i, u + 16 * i);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            tmem_fence16(u + 16 * i);
            u32_to_f32_16(u + 16 * i, s + 16 * i);
          }
        }
        if (L::kOwnP) {
          tc_fence_before();
          mbar_arrive(s_free + t);
        }
        if (part) {
          asm volatile("");  // keeps this a branch: 64 selects would cost every tile
          if (live) {
#pragma unroll
            for (int i = 0; i < 64; ++i) s[i] = seen[i >> 5] >> (i & 31) & 1 ? s[i] : -INFINITY;
          }
          if (mask && (Twin || t == 0)) {
            // hidden values may be NaN or infinite, and 0 times those is NaN: clear this
            // half's hidden rows of V. (Tile 1 reads the same V, without Twin, and comes after
            // tile 0 in their turns.) Two threads a row, each with a box or every other chunk;
            // neighbouring rows start at different chunks, that is, banks
            const Place at(2 * (base + (uint32_t)(j - (int)j0)) + 1);
            at_wait(full + at.slot, at.turn & 1, dead, AT_FULL);
            if (!((row & 32 ? seen[1] : seen[0]) >> (row & 31) & 1)) {
              uint4* v = reinterpret_cast<uint4*>(sm + L::kRing + at.slot * L::kTile + (64 * half + (row & 63)) * 128);
              const int part = row >> 6;
              for (int k = 0; k < 4 * Boxes; ++k)
                v[Boxes == 2 ? part * (AT_BOX / 16) + ((k + row) & 7) : (2 * k + part + row) & 7] =
                    make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
        }
        // (-inf only where this half's 64 keys are all hidden)
        float top = part && !(seen[0] | seen[1]) ? -INFINITY : live ? fmaxf(row_max<64>(s), AT_LOWEST) : AT_LOWEST;
        if (cnt > first) at_wait(o_done + t, (cnt - 1) & 1, dead, AT_O);  // O_t is complete, P_t read
        // (the barrier also keeps P_t, where it lies over S_t, behind both halves' loads)
        if (at_any(id, j == jt || top > m + stale)) {
          *mine = top;
          at_sync(id);
          top = fmaxf(top, *other);
          if (j == jt) {
            m = top;
          } else {
            tc_fence_after();
            const bool raise = top > m + stale;
            const float f = raise ? ex2_approx((m - top) * c) : 1.f;
            m = raise ? top : m;
            l = at_total(l) * f;
            for (int i = half; live && i < ksteps; i += 2) {
              float o[16];
              tmem_ld16(to + 16 * i, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= f;
              tmem_st16(to + 16 * i, o);
            }
          }
        }
        // (a score of +inf makes m infinite, its own weight inf - inf, and the row's total, NaN)
        const float mc = m <= AT_LOWEST ? 0.f : fmaf(-m, c, AT_LIFT<T>);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        if (!Twin || g.turns) at_turn_wait(t);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t p[16];
          if (!live) break;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 y = __ffma2_rn(make_float2(s[32 * i + 2 * e], s[32 * i + 2 * e + 1]), make_float2(c, c),
                                        make_float2(mc, mc));
            const float2 v = make_float2(ex2_approx(y.x), ex2_approx(y.y));
            sum[e & 1] = __fadd2_rn(sum[e & 1], v);
            p[e] = at_pack<T>(v.x, v.y);
          }
          if constexpr (L::kSharedP) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *reinterpret_cast<uint4*>(sp + swz_off(row, 4 * i + k, 128)) =
                  make_uint4(p[4 * k], p[4 * k + 1], p[4 * k + 2], p[4 * k + 3]);
          } else {
            tmem_st16u(tp + 16 * i, p);
          }
          if (i == 0 && (!Twin || g.turns)) at_turn_give(t);
        }
        if (Twin && !live && g.turns) at_turn_give(t);
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_wait_st();
        if (L::kSharedP) fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(p_ready + t);
        ++cnt;
      }
      if (Twin && g.turns && t == 1 && n % 2 == 1) {  // tile 0 had one key tile more
        at_turn_wait(t);
        at_turn_give(t);
      }
      // ---- the unit's rows: to the output when the unit is whole, else to the workspace
      if (any) {
        at_wait(o_done + t, (cnt - 1) & 1, dead, AT_O);
        tc_fence_after();
      }
      *mine = l;
      at_sync(id);
      l = *dead ? NAN : at_total(half ? *other + l : l + *other);
      if (!Twin && n == g.tiles) {
        // through the Q tile, whose products are complete: 16-byte chunks of whole rows,
        // `wide` lanes a row, as Q was read
        const float inv = at_inverse(m, l);
        for (int i = half; live && i < ksteps; i += 2) {
          float v[16];
          tmem_ld16(to + 16 * i, v);
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = at_pack<T>(v[2 * e] * inv, v[2 * e + 1] * inv);
          uint8_t* o = sq + (i >> 2) * AT_BOX;
          *reinterpret_cast<uint4*>(o + swz_off(row, (2 * i) & 7, 128)) = make_uint4(w[0], w[1], w[2], w[3]);
          *reinterpret_cast<uint4*>(o + swz_off(row, (2 * i + 1) & 7, 128)) = make_uint4(w[4], w[5], w[6], w[7]);
        }
        at_sync(id);
        const int k = lane & (wide - 1);
        for (int rr = 16 * half + lane / wide; rr < 16 * half + 16; rr += 32 / wide) {
          const long at = locate(rr, g.a.o_sb, g.a.o_sl, g.a.o_sh);
          if (at < 0 || k >= chunks) continue;
          const uint4 v = *reinterpret_cast<const uint4*>(sq + (k >> 3) * AT_BOX + swz_off(warp_row + rr, k & 7, 128));
          T* o = static_cast<T*>(g.a.o) + at + 8 * k;
          if (g.o_wide && 8 * k + 8 <= d) {
            *reinterpret_cast<uint4*>(o) = v;
          } else {
            const T* e = reinterpret_cast<const T*>(&v);
            for (int i = 0; i < 8; ++i)
              if (8 * k + i < d) o[i] = e[i];
          }
        }
      } else {
        // the piece is kept channel by channel, so that a warp stores 32 rows side by side
        const long piece = Twin ? (long)blockIdx.x : 2L * blockIdx.x + (x == x0 ? 0 : 1);
        const int col = Twin ? 128 * t + unit_row : unit_row;
        if (half == 0) g.part_ml[piece * 256 + col] = make_float2(m == -INFINITY ? m : fmaxf(m * c, AT_LOWEST), l);
        float* o = g.part + piece * 256 * d + col;
        for (int i = half; live && i < ksteps; i += 2) {
          float v[16];
          if (any) tmem_ld16(to + 16 * i, v);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (16 * i + e < d) o[(16 * i + e) * 256] = any ? v[e] : 0.f;
        }
      }
      tc_fence_before();
      at_sync(id);  // the Q tile and the rows' sums are written again
      base += (uint32_t)n;
      x += n;
    }
    if ((!Twin || g.turns) && t == 0) at_turn_wait(t);  // the other tile's last
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 16) tmem_dealloc(tmem, 512);
}

// Adds the pieces of the units that were cut, 32 rows a block:
//   o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i, M the largest m_i
// A piece without a visible key for a row (m_i = -inf) weighs nothing; a NaN in any piece's
// total makes the row NaN as it does in an uncut unit.
// A lane is a row (the pieces are stored channel by channel). All maxima and totals are
// fetched at once and turned into weights in shared memory, then every warp adds its
// channels, whose loads wait for nothing (piece by piece, each behind its maximum, took 15 to
// 20 us). The result goes through shared memory to be written row by row.
constexpr int AT_JOIN = 256;
template <typename T>
__global__ void __launch_bounds__(AT_JOIN) attn_join_kernel(const __grid_constant__ AttnTcArgs g, int grid) {
  extern __shared__ float join_sm[];  // [pieces][32] maxima, later weights; [pieces][32] totals
  __shared__ T out[32][130];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = g.a.d;
  constexpr int kWarps = AT_JOIN / 32;
  const int groups = g.unit_rows / 32;
  const long unit = blockIdx.x / groups;
  const int row0 = (int)(blockIdx.x - unit * groups) * 32;
  const long bh = unit / g.row_units, r0 = (unit - bh * g.row_units) * g.unit_rows + row0;
  const long t0 = unit * g.tiles, c0 = at_owner(g, t0, grid), c1 = at_owner(g, t0 + g.tiles - 1, grid);
  if (r0 >= g.rows || (c0 == c1 && !g.twin)) {  // no rows, or written by their CTA
    // every block waits: a grid that ended without it would let the stream's next kernel start
    // before the main kernel's rows are written
    wait_for_previous();
    return;
  }
  const int pieces = g.twin ? 2 * g.cuts : (int)(c1 - c0 + 1);
  // piece i: its place among all, in rows; only the first can be its CTA's second
  const long first = 2 * c0 + (at_start(g, c0, grid) >= t0 ? 0 : 1);
  const auto place = [&](int i) -> long {
    return g.twin ? unit + g.units * (i >> 1) : i == 0 ? first : 2 * (c0 + i);
  };
  const auto column = [&](int i) { return (g.twin ? 128 * (i & 1) : 0) + row0 + lane; };
  float *ms = join_sm, *ls = join_sm + 32 * pieces;
  wait_for_previous();
  for (int i = warp; i < pieces; i += kWarps) {
    const float2 ml = __ldcg(g.part_ml + place(i) * 256 + column(i));
    ms[32 * i + lane] = ml.x;
    ls[32 * i + lane] = ml.y;
  }
  __syncthreads();
  float top = -INFINITY, l = 0.f;
  for (int i = 0; i < pieces; ++i) top = fmaxf(top, ms[32 * i + lane]);
  for (int i = 0; i < pieces; ++i) {
    const float m = ms[32 * i + lane], li = ls[32 * i + lane];
    l += m != -INFINITY ? ex2_approx(m - top) * li : li == li ? 0.f : li;
  }
  __syncthreads();
  for (int i = warp; i < pieces; i += kWarps) {
    const float m = ms[32 * i + lane];
    ms[32 * i + lane] = m == -INFINITY ? 0.f : ex2_approx(m - top);
  }
  __syncthreads();
  constexpr int kMost = 128 / kWarps;  // channels of a warp
  float o[kMost];
#pragma unroll
  for (int k = 0; k < kMost; ++k) o[k] = 0.f;
#pragma unroll 2
  for (int i = 0; i < pieces; ++i) {
    const float f = ms[32 * i + lane];
    const float* part = g.part + place(i) * 256 * d + column(i);
#pragma unroll
    for (int k = 0; k < kMost; ++k)
      if (warp + k * kWarps < d) {
        const float v = __ldcg(part + (warp + k * kWarps) * 256);
        o[k] += f == 0.f ? 0.f : f * v;
      }
  }
  const float inv = at_inverse(top, l);
#pragma unroll
  for (int k = 0; k < kMost; ++k)
    if (warp + k * kWarps < d) out[lane][warp + k * kWarps] = from_f32<T>(o[k] * inv);
  __syncthreads();
  const int b = (int)(bh / g.a.hk), hk = (int)(bh - (long)b * g.a.hk);
  for (int rr = warp; rr < 32 && r0 + rr < g.rows; rr += kWarps) {
    const long ql = (r0 + rr) / g.share;
    const long qh = hk * g.share + (r0 + rr - ql * g.share);
    T* dst = static_cast<T*>(g.a.o) + b * g.a.o_sb + ql * g.a.o_sl + qh * g.a.o_sh;
    for (int c = lane; c < d; c += 32) dst[c] = out[rr][c];
  }
}

}  // namespace scb
