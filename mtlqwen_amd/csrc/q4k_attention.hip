// Attention of a packed batch's new tokens over a paged key/value cache.
//
// For a row and head, x_j = scale q.k_j (capped, biased) over the keys that the row
// sees and o = sum_j 2^(t_j - m) v_j / sum_j 2^(t_j - m), t = x log2(e), in one pass
// over the keys with the running maximum m: the sums of a part of the keys are
// rescaled by 2^(m - m') where the maximum rises, and parts of the keys that were
// summed apart join the same way.
//
// The query rows of a sequence and a cache head are its tokens' rows times the
// `group` heads that share the cache head: row u = token u / group, head u %
// group.  Both products run on the matrix units, transposed, so that a query row
// is a lane's column throughout and neither the maxima nor the rescaling move
// between lanes:
//   S^T [16 keys x 16 rows] = K [keys x d] Q^T,  O^T [16 d x 16 rows] = V^T P^T
// Lane 16 g + i of S^T holds keys 4 g + 0..3 of row i, which is what the second
// product wants of P^T for the key order (4 g + e, 16 + 4 g + e) of 32 keys; V is
// read from LDS in that order with the transposing read.
//
// Work is a line of key tiles: cache heads, their units (blocks of query rows of a
// sequence), their tiles.  Lengths are on the device, so a launch has a fixed
// number of workgroups and each takes an equal stretch of that line (locate());
// a unit that several share leaves its sums, one per stretch, in the workspace,
// and the workgroup that comes last adds them, in the order of the stretches.
#include <cfloat>

#include "q4k_device.h"

namespace q4k {
namespace {

typedef short s4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4_t lds_s4_t;

// Weights are 2^(t - m + kTop), so that fp16 holds those down to 2^-22 of the
// largest with all its bits; the maximum is raised where a score passes it by kSlack
// (2^(kTop + kSlack) is still finite), which is rare after the first tiles.
constexpr float kTop = 8.0f, kSlack = 7.0f;
constexpr float kLog2e = 1.4426950408889634f;
// Rows whose maximum passes this are summed apart (sum_again): the multiply-add that
// makes t - m + kTop keeps what the maximum's own rounding took off, half a step, and
// rounds kTop with it, from 2^27 on by 8 and more, which makes weights that pass fp16 or are nothing.
constexpr float kFar = 0x1p26f;

// tanh within 2^-21 of the value: the odd series below 1/4 (its next term is
// 2^-26 of the value there), 1 - 2 / (e^2x + 1) above, whose error is 2^-23.
__device__ __forceinline__ float tanh_score(float x) {
  const float y = x * x;
  const float small = x * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
  const float e = __builtin_amdgcn_exp2f(x * (2.0f * kLog2e));
  const float large = 1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f);
  return fabsf(x) < 0.25f ? small : large;
}

// Maximum over the four lanes of a query row (lane ^ 16, lane ^ 32).
__device__ __forceinline__ float row_max(float v) {
  const uint32_t a = __builtin_bit_cast(uint32_t, v);
  const auto h = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  const float w = fmaxf(__builtin_bit_cast(float, (uint32_t)h[0]), __builtin_bit_cast(float, (uint32_t)h[1]));
  const uint32_t b = __builtin_bit_cast(uint32_t, w);
  const auto q = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)q[0]), __builtin_bit_cast(float, (uint32_t)q[1]));
}

__device__ __forceinline__ float row_sum(float v) {
  const uint32_t a = __builtin_bit_cast(uint32_t, v);
  const auto h = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  const float w = __builtin_bit_cast(float, (uint32_t)h[0]) + __builtin_bit_cast(float, (uint32_t)h[1]);
  const uint32_t b = __builtin_bit_cast(uint32_t, w);
  const auto q = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  return __builtin_bit_cast(float, (uint32_t)q[0]) + __builtin_bit_cast(float, (uint32_t)q[1]);
}

__device__ __forceinline__ int lane_value(int v, int lane) {
  return __builtin_amdgcn_readlane(v, lane);
}

// ---- the line of work --------------------------------------------------------
// Whole numbers of 32 bits throughout (attention_plan bounds the line): what is
// computed once per launch or unit is a chain of dependent instructions with little
// beside it, and a call of one row is hardly more than that.

// x / y for any x, m = 2^32 / y rounded down (2^32 - 1 for y = 1): the product is
// one too small at most.
__device__ __forceinline__ uint32_t divided(uint32_t x, uint32_t y, uint32_t m) {
  const uint32_t q = __umulhi(x, m);
  return q + ((uint64_t)(q + 1) * y <= x ? 1u : 0u);
}

// The token of query row u of a sequence.
__device__ __forceinline__ int token_of(const AttentionArgs& a, int u) {
  return (int)divided((uint32_t)u, (uint32_t)a.group, a.group_inverse);
}

// One sequence per lane: the position of its first row, the keys that its table
// holds, its query rows per cache head, the units before it, its table, its first
// row in the batch.
struct Sequences {
  int first, cap, rows, unit, slot, start;
};
constexpr int kSequenceInts = 6 * 64;

__device__ __forceinline__ Sequences load_sequences(const AttentionArgs& a) {
  const CacheArgs& c = a.cache;
  const int s = threadIdx.x & 63;
  Sequences q{0, 0, 0, a.units, 0, 0};
  if (s < c.nq) {
    const int p = c.positions[s];
    q.slot = c.slots ? c.slots[s] : s;
    q.rows = c.count[s] * a.group;
    q.unit = a.unit[s];
    q.start = c.start[s];
    q.first = p < -(1 << 30) ? -(1 << 30) : p > (1 << 30) ? 1 << 30 : p;
    q.cap = (uint32_t)q.slot < (uint32_t)c.table_rows && c.pages ? c.width << c.page_log : 0;
  }
  return q;
}

__device__ __forceinline__ void keep_sequences(const Sequences& q, int* lds) {
  const int s = threadIdx.x & 63;
  lds[s] = q.first, lds[64 + s] = q.cap, lds[128 + s] = q.rows, lds[192 + s] = q.unit, lds[256 + s] = q.slot, lds[320 + s] = q.start;
}

__device__ __forceinline__ Sequences kept_sequences(const int* lds) {
  const int s = threadIdx.x & 63;
  return Sequences{lds[s], lds[64 + s], lds[128 + s], lds[192 + s], lds[256 + s], lds[320 + s]};
}

// A unit: its sequence, query rows [row, row_end), the first key tile's first key,
// the key past the last row's, its tiles (one at least, so that rows that see nothing
// are written too).
struct Unit {
  int seq, row, row_end, lo, hi, tiles;
};

template <int QB, int TK>
__device__ __forceinline__ Unit unit_of(const AttentionArgs& a, const Sequences& q, int u) {
  Unit x{0, 0, 0, 0, 0, 0};
  int first = 0, cap = 0, rows = 0;
  for (int s = 0; s < a.cache.nq; ++s) {
    const int from = lane_value(q.unit, s);
    if (u >= from) {
      x.seq = s;
      x.row = (u - from) * QB;
      first = lane_value(q.first, s);
      cap = lane_value(q.cap, s);
      rows = lane_value(q.rows, s);
    }
  }
  if (u >= a.units)
    return x;
  x.row_end = x.row + QB < rows ? x.row + QB : rows;
  const int t0 = token_of(a, x.row), t1 = token_of(a, x.row_end - 1);
  x.hi = first + t1 + 1 < cap ? first + t1 + 1 : cap;
  x.hi = x.hi < 0 ? 0 : x.hi;
  x.lo = a.window && first + t0 + 1 > a.window ? (first + t0 + 1 - a.window) & -TK : 0;
  x.tiles = x.hi > x.lo ? (x.hi - x.lo + TK - 1) / TK : 1;
  return x;
}

// Sum over this lane and those before it.
__device__ __forceinline__ int scan_lanes(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}

// A unit takes EXTRA places of the line before its tiles: what its beginning and
// end cost a workgroup, in tiles.
// 64 units from u0 on, one per lane, and the places up to each.
struct Units {
  Unit unit;
  int upto;
};

template <int QB, int TK, int EXTRA>
__device__ __forceinline__ Units units_from(const AttentionArgs& a, const Sequences& q, int u0) {
  Units x;
  x.unit = unit_of<QB, TK>(a, q, u0 + (threadIdx.x & 63));
  x.upto = scan_lanes(x.unit.tiles ? x.unit.tiles + EXTRA : 0);
  return x;
}

// The line: places of one cache head and in all, and those of a stretch: a
// multiple of LEAST, so that the line makes no more stretches than workgroups.
// Wave-uniform.
struct Line {
  int per_head, total, step;

  // x / y where the quotient is small beside 2^23: the rounded one is one off at most.
  static __device__ __forceinline__ int quotient(int x, int y) {
    const int q = __builtin_amdgcn_readfirstlane((int)((float)x * __builtin_amdgcn_rcpf((float)y)));
    const int rest = (int)((uint32_t)x - (uint32_t)q * (uint32_t)y);
    return q + (rest >= y ? 1 : 0) - (rest < 0 ? 1 : 0);
  }
  __device__ __forceinline__ int stretches() const { return quotient(total - 1, step) + 1; }
  __device__ __forceinline__ int start(int r) const { return r * step; }
  __device__ __forceinline__ int end(int r) const { return r * step < total - step ? r * step + step : total; }
  // The stretch that holds place x.
  __device__ __forceinline__ int of(int x) const { return quotient(x, step); }
};

// `near`: the first 64 units.
template <int QB, int TK, int EXTRA, int LEAST>
__device__ __forceinline__ Line make_line(const AttentionArgs& a, const Sequences& q, const Units& near) {
  Line x;
  x.per_head = lane_value(near.upto, 63);
  for (int u0 = 64; u0 < a.units; u0 += 64)
    x.per_head += lane_value(units_from<QB, TK, EXTRA>(a, q, u0).upto, 63);
  x.total = x.per_head * (int)a.cache.heads;
  const int each = (int)divided((uint32_t)(x.total + a.stretches - 1), (uint32_t)a.stretches, a.stretches_inverse);
  x.step = (each + LEAST - 1) & -LEAST;
  return x;
}

// The unit that holds place x of the line, and the place of its first tile, behind
// the extra ones (wave-uniform).
struct Place {
  Unit unit;
  int head, at, index;
};

template <int QB, int TK, int EXTRA>
__device__ __forceinline__ Place locate(const AttentionArgs& a, const Sequences& q, const Line& line, const Units& near, int x) {
  Place p;
  p.head = Line::quotient(x, line.per_head);
  const int y = x - p.head * line.per_head;
  Units here = near;
  int before = 0, start = 0;
  while (y >= before + lane_value(here.upto, 63)) {  // ends: y < per_head
    before += lane_value(here.upto, 63);
    start += 64;
    here = units_from<QB, TK, EXTRA>(a, q, start);
  }
  const int lane = __ffsll((unsigned long long)__ballot(here.upto > y - before)) - 1;
  p.unit.seq = lane_value(here.unit.seq, lane);
  p.unit.row = lane_value(here.unit.row, lane);
  p.unit.row_end = lane_value(here.unit.row_end, lane);
  p.unit.lo = lane_value(here.unit.lo, lane);
  p.unit.hi = lane_value(here.unit.hi, lane);
  p.unit.tiles = lane_value(here.unit.tiles, lane);
  p.at = p.head * line.per_head + before + lane_value(here.upto, lane) - p.unit.tiles;
  p.index = start + lane;
  return p;
}

// The unit behind p's on the line.
template <int QB, int TK, int EXTRA>
__device__ __forceinline__ Place behind(const AttentionArgs& a, const Sequences& q, Place p) {
  p.at += p.unit.tiles + EXTRA;
  const bool last = p.index + 1 == a.units;
  p.index = last ? 0 : p.index + 1;
  p.head += last ? 1 : 0;
  const Unit u = unit_of<QB, TK>(a, q, p.index);
  p.unit.seq = __builtin_amdgcn_readfirstlane(u.seq);
  p.unit.row = __builtin_amdgcn_readfirstlane(u.row);
  p.unit.row_end = __builtin_amdgcn_readfirstlane(u.row_end);
  p.unit.lo = __builtin_amdgcn_readfirstlane(u.lo);
  p.unit.hi = __builtin_amdgcn_readfirstlane(u.hi);
  p.unit.tiles = __builtin_amdgcn_readfirstlane(u.tiles);
  return p;
}

// ---- query rows ----------------------------------------------------------------

// The row at `pos` (-1: none) sees key j + x for low < x <= high.
__device__ __forceinline__ void seen_keys(const AttentionArgs& a, int pos, int cap, int j, int& low, int& high) {
  high = (pos < cap ? pos : cap - 1) - j;
  low = a.window && pos >= a.window ? pos - a.window - j : -j - 1;
}

// NQ column tiles of 16 query rows: their fragments (fp32 rows as two fp16 parts
// under a power of two, 22 bits), what turns a product into t, and where the rows
// stand (-1: no row; it sees nothing).
template <typename T, int DP, int NQ>
struct Rows {
  static constexpr bool kParts = sizeof(T) == 4;
  h8_t q[NQ][DP / 32], ql[kParts ? NQ : 1][DP / 32];
  float c[kParts ? NQ : 1], slope[NQ];
  int pos[NQ], cap;

  __device__ __forceinline__ float factor(int n) const { return c[kParts ? n : 0]; }

  __device__ __forceinline__ void seen(const AttentionArgs& a, int n, int j, int& low, int& high) const { seen_keys(a, pos[n], cap, j, low, high); }

  __device__ __forceinline__ void load(const AttentionArgs& a, const Sequences& s, const Unit& u, int head, int row) {
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int first = lane_value(s.first, u.seq), start = lane_value(s.start, u.seq);
    cap = lane_value(s.cap, u.seq);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int r = row + 16 * n + i;
      const bool live = r < u.row_end;
      const int t = token_of(a, r), h = head * a.group + (r - t * a.group);
      const T* x = static_cast<const T*>(a.q) + (int64_t)(start + t) * a.q_row + (int64_t)h * a.q_head + 8 * g;
      c[kParts ? n : 0] = a.scale * kLog2e;
      if constexpr (kParts) {
        float f[DP / 32][8], mx = 0.0f, up, down;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            f[d][e] = 0.0f;
          if (live && 32 * d + 8 * g < a.cache.dim)
            load8(x + 32 * d, f[d]);
        }
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            mx = fmaxf(mx, fabsf(f[d][e]));
        pow2_scale(row_max(mx), up, down);
        c[n] *= down;
        up *= a.sign;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = f[d][e] * up;
            q[n][d][e] = (_Float16)v;
            ql[n][d][e] = (_Float16)(v - (float)q[n][d][e]);
          }
      } else {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          h8_t v = {};
          if (live && 32 * d + 8 * g < a.cache.dim)
            v = *reinterpret_cast<const h8_any_t*>(x + 32 * d);
          q[n][d] = v * (_Float16)a.sign;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      // Neither 0 nor infinite, which would make NaN of what is not seen or of zeros.
      c[kParts ? n : 0] = __builtin_amdgcn_fmed3f(c[kParts ? n : 0], 0x1p-126f, 0x1p127f);
      slope[n] = live && a.slopes ? a.slopes[h] * kLog2e : 0.0f;
      pos[n] = live ? first + t : -1;
    }
  }
};

// ---- one tile of keys --------------------------------------------------------------
// K lies in LDS as the fragments of the first product: 16 keys x 32 d, 1 KB, lane
// 16 g + i at 16 (16 g + i): key i, d = 8 g + 0..7.  V lies row by row, 16-byte
// chunks swizzled so that the rows of a transposing read meet no bank twice.

template <int DP>
__device__ __forceinline__ int v_swizzle(int row) {
  // Rows that start in the same banks: every one (512 and 256 bytes), every second
  // (384 and 128), every fourth (192).
  return DP % 128 == 0 ? 2 * (row & 7) : DP % 64 == 0 ? 2 * ((row >> 1) & 3) : 2 * ((row >> 2) & 1);
}

// `between`: called with every d / 32 behind the products of 32 d.
template <typename T, int DP, int NQ, int NA, typename F>
__device__ __forceinline__ void scores(const uint8_t* k, const Rows<T, DP, NQ>& r, f4_t (&s)[NA][NQ], const F& between) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int a = 0; a < NA; ++a)
#pragma unroll
    for (int n = 0; n < NQ; ++n)
      s[a][n] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  // The fragments of the next 32 d are asked for under the products of these, and
  // no earlier: more of them would not fit the registers beside O.
  h8_t f[2][NA];
  const auto read = [&](int d) {
#pragma unroll
    for (int a = 0; a < NA; ++a)
      f[d & 1][a] = *reinterpret_cast<const h8_t*>(k + (a * (DP / 32) + d) * 1024 + lane * 16);
    asm volatile("" ::: "memory");
  };
  read(0);
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) {
    if (d + 1 < DP / 32)
      read(d + 1);
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        s[a][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[d & 1][a], r.q[n][d], s[a][n], 0, 0, 0);
        if constexpr (Rows<T, DP, NQ>::kParts)
          s[a][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[d & 1][a], r.ql[n][d], s[a][n], 0, 0, 0);
      }
    __builtin_amdgcn_sched_barrier(0);
    between(d);
  }
}

// Products become t: capped, biased and, in a tile that not every row sees whole,
// -inf for the keys that a row does not see.  `there`: a bit per 16 keys whose page
// is there.  With neither cap nor bias products stay as they are (c turns them into
// t where the weights are formed).  `some`: a bit per row that sees a key.
template <typename T, int DP, int NQ, int NA>
__device__ __forceinline__ void finish_scores(const AttentionArgs& a, const Rows<T, DP, NQ>& r, int key, bool whole, uint32_t there, bool formed,
                                              f4_t (&s)[NA][NQ], uint32_t (&some)[NQ]) {
  const int g = (threadIdx.x & 63) >> 4;
  if (formed) {
    const float in = a.softcap > 0.0f ? 1.0f / (a.softcap * kLog2e) : 0.0f, out = a.softcap * kLog2e;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const float away = (float)(key + 4 * g - r.pos[n]);
#pragma unroll
      for (int b = 0; b < NA; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float t = s[b][n][e] * r.factor(n);
          if (a.softcap > 0.0f)
            t = out * tanh_score(t * in);
          s[b][n][e] = fmaf(r.slope[n], away + (float)(16 * b + e), t);
        }
    }
  }
  if (!whole) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      int low, high;
      bool any = false;
      r.seen(a, n, key + 4 * g, low, high);
#pragma unroll
      for (int b = 0; b < NA; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool sees = ((there >> b) & 1) && 16 * b + e > low && 16 * b + e <= high;
          any = any || sees;
          if (!sees)
            s[b][n][e] = -INFINITY;
        }
      const uint64_t lanes = __ballot(any), half = lanes | lanes >> 32;
      some[n] |= (uint32_t)(half | half >> 16);
    }
  } else {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
      some[n] = ~0u;
  }
}

// What a row becomes.  One that sees nothing (its maximum is -inf) is zero; scores that are
// all -inf have a maximum (Sums::settle) and no weights: 0 / 0.
__device__ __forceinline__ f4_t row_values(f4_t o, float l, float m) {
  const float f = l == 0.0f ? __builtin_nanf("") : 1.0f / l;
  return m == -INFINITY ? f4_t{0.0f, 0.0f, 0.0f, 0.0f} : o * f;
}

// What a wave's or stretch's sums under the maximum m count for under `top`.  Never 0: an
// infinite sum stays infinite, and 2^-126 of a finite one is nothing beside weights of 2^kTop.
__device__ __forceinline__ float share(float m, float top) {
  return m == top ? 1.0f : fmaxf(__builtin_amdgcn_exp2f(m - top), 0x1p-126f);
}

// The running sums of NQ column tiles: O^T, the maximum that its weights refer to,
// this lane's part of their sum, and a bit per row that sees a key.
template <int DP, int NQ>
struct Sums {
  f4_t o[NQ][DP / 16];
  float m[NQ], l[NQ];
  bool far;  // a maximum of the wave's rows has passed kFar or -kFar
  uint32_t some[NQ];

  // A row that sees keys whose scores are all -inf gets the lowest maximum: other
  // stretches' weights leave nothing of its sums, and alone it is no row that sees nothing.
  __device__ __forceinline__ void settle() {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const bool sees = (some[n] >> (threadIdx.x & 15)) & 1;
      m[n] = m[n] == -INFINITY && sees ? -FLT_MAX : m[n];
    }
  }

  // Sums that infinities, -infinities or both (NaN) reach: bit 4 d + e of `up` and `down`.
  static constexpr int kWords = (DP + 127) / 128;
  __device__ __forceinline__ void put(const uint32_t (&up)[NQ][kWords], const uint32_t (&down)[NQ][kWords]) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool u = (up[n][d / 8] >> (4 * (d % 8) + e)) & 1, v = (down[n][d / 8] >> (4 * (d % 8) + e)) & 1;
          o[n][d][e] = u || v ? (u ? INFINITY : 0.0f) - (v ? INFINITY : 0.0f) : o[n][d][e];
        }
  }

  // Whether a sum of this lane is infinite or NaN (only those leave 0 * o other than 0)
  // in a row whose sum of weights is not.
  __device__ __forceinline__ bool odd(const float (&weights)[NQ]) const {
    bool any = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      f4_t z = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          z[e] = fmaf(o[n][d][e], 0.0f, z[e]);
      any = any || (!(z[0] + z[1] + z[2] + z[3] == 0.0f) && weights[n] == weights[n]);
    }
    return any;
  }

  __device__ __forceinline__ void clear() {
    far = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
        o[n][d] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
      m[n] = -INFINITY;
      l[n] = 0.0f;
      some[n] = 0;
    }
  }

  // Scores to weights (in place), the sums rescaled where a maximum rises.
  template <int NA, typename F>
  __device__ __forceinline__ void weigh(f4_t (&s)[NA][NQ], const F& c) {
    float top[NQ];
    bool rise = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float v = -INFINITY;
#pragma unroll
      for (int b = 0; b < NA; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v = fmaxf(v, s[b][n][e]);
      top[n] = row_max(v) * c(n);
      rise = rise || top[n] > m[n] + kSlack;
    }
    if (__builtin_expect(__any(rise), 0)) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const float now = fmaxf(m[n], top[n]);
        const float f = now == m[n] ? 1.0f : __builtin_amdgcn_exp2f(m[n] - now);
        m[n] = now;
        far = far || __any(fabsf(now) >= kFar && fabsf(now) < INFINITY);
        l[n] *= f;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d)
          o[n][d] *= f;
      }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      // No score yet: weights of -inf become 0, of a NaN NaN.
      const float ref = (m[n] == -INFINITY ? 0.0f : m[n]) - kTop;
#pragma unroll
      for (int b = 0; b < NA; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[b][n][e] = __builtin_amdgcn_exp2f(fmaf(s[b][n][e], c(n), -ref));
          l[n] += s[b][n][e];
        }
    }
  }
};

__device__ __forceinline__ h8_t pack_weights(f4_t a, f4_t b) {
  return h8_t{(_Float16)a[0], (_Float16)a[1], (_Float16)a[2], (_Float16)a[3], (_Float16)b[0], (_Float16)b[1], (_Float16)b[2], (_Float16)b[3]};
}

__device__ __forceinline__ h8_t pack_rest(f4_t a, f4_t b, h8_t p) {
  return h8_t{(_Float16)(a[0] - (float)p[0]), (_Float16)(a[1] - (float)p[1]), (_Float16)(a[2] - (float)p[2]), (_Float16)(a[3] - (float)p[3]),
              (_Float16)(b[0] - (float)p[4]), (_Float16)(b[1] - (float)p[5]), (_Float16)(b[2] - (float)p[6]), (_Float16)(b[3] - (float)p[7])};
}

// A V^T fragment of 16 d x 32 keys: lane 16 g + i, d = 16 dt + i, keys 4 g + e
// and 16 + 4 g + e.  The swizzle is an exclusive or with bits of the row, so the
// fragments of a row differ by one with bits of dt.
template <int DP>
__device__ __forceinline__ uint32_t v_base(const uint8_t* v) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int row = 4 * g + (i >> 2);
  return lds_addr(v) + row * (DP * 2) + (v_swizzle<DP>(row) + ((i & 3) >> 1)) * 16 + (i & 1) * 8;
}

template <int DP>
__device__ __forceinline__ h8_t v_fragment(uint32_t base, int dt) {
  constexpr int kBits = DP % 128 == 0 ? 3 : DP % 64 == 0 ? 2 : 1;
  const uint32_t at = (base ^ ((dt & ((1 << kBits) - 1)) << 5)) + (dt >> kBits) * (32 << kBits);
  const s4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)(uintptr_t)at);
  const s4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)(uintptr_t)(at + 16 * DP * 2));
  typedef short s8_t __attribute__((ext_vector_type(8)));
  return __builtin_bit_cast(h8_t, s8_t{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]});
}

// A weight of zero does not keep an infinity or NaN of V out of a product, so a
// tile that some row does not see whole is looked over first (odd_values, by
// THREADS threads together).  If it holds one, a product of the places of infinities and
// NaN with who sees them says which sums they reach, which become NaN (mark_values), and
// they become zero in LDS (clear_values).  Tiles that all rows see are not looked over (it
// would be an eighth of their reads of LDS, and a barrier more).  An infinity there
// makes a sum infinite, or NaN where its weight, or the second part of one, is zero or
// negative in fp16.  So a wave some of whose sums come out as either (Sums::odd) reads V
// once more for what they are to be (mark_again).
// A half's exponent plus one step reaches its sign bit for infinities and NaN alone.
__device__ __forceinline__ uint32_t odd_bits(u4_t f) {
  return (((f.x & 0x7fff7fffu) + 0x04000400u) | ((f.y & 0x7fff7fffu) + 0x04000400u) | ((f.z & 0x7fff7fffu) + 0x04000400u) |
          ((f.w & 0x7fff7fffu) + 0x04000400u)) & 0x80008000u;
}

template <int THREADS, int BYTES>
__device__ __forceinline__ bool odd_values(const uint8_t* v, int thread) {
  uint32_t bits = 0;
#pragma unroll 4
  for (int at = thread * 16; at < BYTES; at += THREADS * 16)
    bits |= odd_bits(*reinterpret_cast<const u4_t*>(v + at));
  return bits != 0;
}

template <int THREADS, int BYTES>
__device__ __forceinline__ void clear_values(uint8_t* v, int thread) {
#pragma unroll 1
  for (int at = thread * 16; at < BYTES; at += THREADS * 16) {
    h8_t f = *reinterpret_cast<const h8_t*>(v + at);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      f[e] = __builtin_fabsf16(f[e]) <= (_Float16)65504.0f ? f[e] : (_Float16)0.0f;
    *reinterpret_cast<h8_t*>(v + at) = f;
  }
}

template <typename T, int DP, int NQ>
__device__ __forceinline__ void mark_values(const AttentionArgs& a, const uint8_t* v, const Rows<T, DP, NQ>& r, int key, uint32_t there,
                                            Sums<DP, NQ>& sums) {
  constexpr int kWords = Sums<DP, NQ>::kWords;
  const int g = (threadIdx.x & 63) >> 4;
  const uint32_t base = v_base<DP>(v);
  uint32_t reached[NQ][kWords], any = 0;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    int low, high;
    r.seen(a, n, key + 4 * g, low, high);
    h8_t one;  // who sees which key
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = 16 * (e >> 2) + (e & 3);
      one[e] = ((there >> (e >> 2)) & 1) && k > low && k <= high ? (_Float16)1.0f : (_Float16)0.0f;
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      reached[n][i] = 0;
#pragma unroll 1
    for (int d = 0; d < DP / 16; ++d) {  // a fragment at a time in registers
      h8_t f = v_fragment<DP>(base, d);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        f[e] = __builtin_fabsf16(f[e]) <= (_Float16)65504.0f ? (_Float16)0.0f : (_Float16)1.0f;
      const f4_t many = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, one, f4_t{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
      uint32_t bits = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        bits |= many[e] > 0.0f ? 1u << e : 0u;
      any |= bits;
      bits <<= 4 * (d & 7);
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        reached[n][i] |= d >> 3 == i ? bits : 0u;
    }
  }
  if (__any(any != 0))
    sums.put(reached, reached);
}

// O^T += V^T P^T of 32 keys.  PARTS: weights as two fp16 parts, 22 bits, and not one, 11
// bits.  One is the output's own precision in fp16 and adds as much again to its
// error (2.9e-4 of the values in all, 2.1e-4 with two parts).  Few rows take two, which they hardly
// notice beside the reading of keys (8 rows 209.1 us with one, 210.8 with two; 5 of 8
// sequences 59.0, 60.0; one row 14.2, 14.5); chunks of fp16 rows take one: 8192 rows 586 us with
// one, 807 with two, 2048 of heads of 256 235 and 298.
template <typename T, int DP, int NQ, bool PARTS>
__device__ __forceinline__ void add_values(const uint8_t* v, const f4_t (&p0)[NQ], const f4_t (&p1)[NQ], Sums<DP, NQ>& sums) {
  constexpr int kAhead = PARTS && DP == 256 ? 1 : 4;
  uint32_t base = v_base<DP>(v);
  asm volatile("" : "+v"(base));  // one register, not one per fragment
  h8_t f[kAhead + 1];
#pragma unroll
  for (int d = 0; d < kAhead; ++d)
    f[d] = v_fragment<DP>(base, d);
  h8_t w[NQ], wl[PARTS ? NQ : 1];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    w[n] = pack_weights(p0[n], p1[n]);
    if constexpr (PARTS)
      wl[n] = pack_rest(p0[n], p1[n], w[n]);
  }
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) {
    if (d + kAhead < DP / 16)
      f[(d + kAhead) % (kAhead + 1)] = v_fragment<DP>(base, d + kAhead);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      sums.o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[d % (kAhead + 1)], w[n], sums.o[n][d], 0, 0, 0);
      if constexpr (PARTS)
        sums.o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[d % (kAhead + 1)], wl[n], sums.o[n][d], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// ---- keys and values into LDS --------------------------------------------------------

// The pages of a sequence: 64 table entries at a time, one per lane, from entry
// `base` on.
struct Pages {
  const int32_t* table;
  int width, base, mine;

  __device__ __forceinline__ void open(const AttentionArgs& a, const Sequences& s, int seq) {
    const int slot = lane_value(s.slot, seq);
    const bool there = (uint32_t)slot < (uint32_t)a.cache.table_rows;
    table = a.cache.tables + (there ? (int64_t)slot * a.cache.width : 0);
    width = there ? a.cache.width : 0;
    base = -64;
    mine = -1;
  }
  // Entries e .. e + 7 are at hand.
  __device__ __forceinline__ void reach(const AttentionArgs& a, int e) {
    if (e < base || e + 7 >= base + 64) {
      base = e;
      const int at = e + (int)(threadIdx.x & 63);
      const int p = at < width ? table[at] : -1;
      mine = (uint32_t)p < a.cache.pages ? p : -1;
    }
  }
  // The page of entry e (wave-uniform), -1 if it is not there.
  __device__ __forceinline__ int page(int e) const { return lane_value(mine, e - base); }

  // Bytes from a head's first page to key j in `page` (one that is not there: page 0,
  // whose tokens nothing sees).
  static __device__ __forceinline__ int64_t bytes(const CacheArgs& c, int page, int j) {
    return (int64_t)(page < 0 ? 0 : page) * (c.page_stride * 2) + (int64_t)(j & ((1 << c.page_log) - 1)) * (c.token_stride * 2);
  }
};

// Where this lane's 16 bytes of each 1 KB transfer come from, relative to the
// first of 16 tokens.  K: key i, d = 8 g + 0..7 of a fragment.  V: chunk 64 x +
// lane of the rows.  Heads shorter than DP: chunks past them are not loaded (their
// LDS is zero).
template <int DP>
struct Lanes {
  uint32_t k, v[DP / 32];

  __device__ __forceinline__ void set(const CacheArgs& c) {
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    k = (uint32_t)(i * (int)c.token_stride) * 2 + g * 16;
#pragma unroll
    for (int x = 0; x < DP / 32; ++x) {
      const int n = x * 64 + lane, row = n / (DP / 8), chunk = (n - row * (DP / 8)) ^ v_swizzle<DP>(row);
      v[x] = (uint32_t)(row * (int)c.token_stride) * 2 + chunk * 16;
    }
  }
  __device__ __forceinline__ bool k_in_head(const CacheArgs& c, int d) const { return 32 * d + 8 * (int)((threadIdx.x & 63) >> 4) < c.dim; }
  __device__ __forceinline__ bool v_in_head(const CacheArgs& c, int x) const {
    const int n = x * 64 + (int)(threadIdx.x & 63), row = n / (DP / 8);
    return 8 * ((n - row * (DP / 8)) ^ v_swizzle<DP>(row)) < c.dim;
  }
};

// Marks the infinities and NaN of V of keys `key` .. `end` - 1, whole groups of 16, out
// of memory, for the wave's rows from `row` on.  The lanes look over 16 tokens together; those
// that hold some are gone through one by one.  Neither LDS nor barriers, all found
// anew, and expected of no wave: laid out among the tiles' code it took 8192 fp16 rows of heads of 64
// from 391 to 420 us.  8192 rows of 128 take 2.1 ms in place of 0.58 where every
// page holds an infinity, 35 ms where every token does.
template <int DP, int NQ>
__device__ __forceinline__ void mark_again(const AttentionArgs& a, const Sequences& s, const Unit& u, int head, int row, int key, int end,
                                           Sums<DP, NQ>& sums) {
  typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
  const CacheArgs& c = a.cache;
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane), "+s"(head), "+s"(row));
  const int g = lane >> 4, first = lane_value(s.first, u.seq), cap = lane_value(s.cap, u.seq);
  const uint8_t* const v = static_cast<const uint8_t*>(c.v) + (int64_t)head * c.head_stride * 2;
  Pages pages;
  pages.open(a, s, u.seq);
  uint32_t all_up[NQ][Sums<DP, NQ>::kWords] = {}, all_down[NQ][Sums<DP, NQ>::kWords] = {};
#pragma unroll 1
  for (; key < end; key += 16) {
    pages.reach(a, key >> c.page_log);
    const int page = pages.page(key >> c.page_log);
    if (page < 0)
      continue;
    const uint8_t* const tokens = v + Pages::bytes(c, page, key);
    uint32_t bits = 0;
#pragma unroll 1
    for (int d = 8 * g; d < c.dim; d += 32)
      bits |= odd_bits(*reinterpret_cast<const u4_t*>(tokens + ((lane & 15) * c.token_stride + d) * 2));
    const uint64_t lanes = __ballot(bits != 0), half = lanes | lanes >> 32;
#pragma unroll 1
    for (uint32_t odd = (uint32_t)(half | half >> 16) & 0xffff; odd; odd &= odd - 1) {
      const int t = __builtin_ctz(odd);
#pragma unroll 1
      for (int d = 0; d < DP / 16; ++d) {
        if (16 * d + 4 * g >= c.dim)
          continue;
        const h4_t f = *reinterpret_cast<const h4_t*>(tokens + (t * c.token_stride + 16 * d + 4 * g) * 2);
        uint32_t up = 0, down = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          up |= f[e] <= (_Float16)65504.0f ? 0u : 1u << e;
          down |= f[e] >= (_Float16)-65504.0f ? 0u : 1u << e;
        }
        up <<= 4 * (d & 7);
        down <<= 4 * (d & 7);
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          int low, high;
          const int mine = row + 16 * n + (lane & 15);
          seen_keys(a, mine < u.row_end ? first + token_of(a, mine) : -1, cap, key, low, high);
          const bool sees = t > low && t <= high;
#pragma unroll
          for (int x = 0; x < Sums<DP, NQ>::kWords; ++x) {
            all_up[n][x] |= sees && d >> 3 == x ? up : 0u;
            all_down[n][x] |= sees && d >> 3 == x ? down : 0u;
          }
        }
      }
    }
  }
  sums.put(all_up, all_down);
}

// The sums of the wave's rows from `row` on over the keys of tiles of TK from `key` on,
// every `step` keys, before `end`, for scores too large for the tiles' way with weights
// (Sums::far): a key at a time, out of memory, t rounded once and its distance from the
// maximum exact.  The four lanes of a row share its products and hold its values as after the tiles.
// Expected of no wave, as mark_again: slow (8192 rows of 128 93 ms, 8 rows of up to 65536
// keys 6 ms), and found anew.
template <typename T, int DP, int NQ, int TK>
__device__ __forceinline__ void sum_again(const AttentionArgs& a, const Sequences& s, const Unit& u, int head, int row, int key, int end, int step,
                                          Sums<DP, NQ>& sums) {
#pragma clang fp contract(off)
  typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
  typedef T t4_t __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  const CacheArgs& c = a.cache;
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane), "+s"(head), "+s"(row));
  const int g = lane >> 4, first = lane_value(s.first, u.seq), start = lane_value(s.start, u.seq), cap = lane_value(s.cap, u.seq);
  const float scale = __builtin_amdgcn_fmed3f(a.scale * kLog2e, 0x1p-126f, 0x1p127f);
  Pages pages;
  pages.open(a, s, u.seq);
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = row + 16 * n + (lane & 15), token = token_of(a, r), h = head * a.group + (r - token * a.group);
    const bool live = r < u.row_end;
    const T* const q = static_cast<const T*>(a.q) + (int64_t)(start + token) * a.q_row + (int64_t)h * a.q_head + 4 * g;
    const int pos = live ? first + token : -1;
    const float slope = live && a.slopes ? a.slopes[h] * kLog2e : 0.0f;
    sums.m[n] = -INFINITY;
    sums.l[n] = 0.0f;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
      sums.o[n][d] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int tile = key; tile < end; tile += step)
#pragma unroll 1
      for (int j = tile; j < tile + TK; ++j) {
        int low, high;
        seen_keys(a, pos, cap, j, low, high);
        const bool sees = 0 > low && 0 <= high;
        pages.reach(a, j >> c.page_log);
        const int page = pages.page(j >> c.page_log);
        if (page < 0 || !__any(sees))
          continue;
        const int64_t at = (int64_t)head * c.head_stride * 2 + Pages::bytes(c, page, j) + 8 * g;
        const uint8_t* const k = static_cast<const uint8_t*>(c.k) + at;
        const uint8_t* const v = static_cast<const uint8_t*>(c.v) + at;
        float x = 0.0f;
#pragma unroll 1
        for (int d = 0; d < c.dim; d += 16)
          if (live && d + 4 * g < c.dim) {
            const t4_t left = *reinterpret_cast<const t4_t*>(q + d);
            const h4_t right = *reinterpret_cast<const h4_t*>(k + 2 * d);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x = fmaf((float)left[e], (float)right[e], x);
          }
        float t = row_sum(x) * a.sign * scale;
        if (a.softcap > 0.0f)
          t = a.softcap * kLog2e * tanh_score(t / (a.softcap * kLog2e));
        t = sees ? fmaf(slope, (float)(j - pos), t) : -INFINITY;
        const float now = fmaxf(sums.m[n], t), f = now == sums.m[n] ? 1.0f : __builtin_amdgcn_exp2f(sums.m[n] - now);
        const float w = t == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((t - now) + kTop);
        sums.m[n] = now;
        sums.l[n] = sums.l[n] * f + (g == 0 ? w : 0.0f);
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
          h4_t y = {};
          if (sees && 16 * d + 4 * g < c.dim)
            y = *reinterpret_cast<const h4_t*>(v + 32 * d);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sums.o[n][d][e] = fmaf(w, (float)y[e], sums.o[n][d][e] * f);
          asm volatile("" ::: "memory");  // one after another: no registers for more
        }
      }
  }
}

// Transfer X of K or V of 16 tokens.
template <int X>
__device__ __forceinline__ void dma_k_one(uint32_t lane, const uint8_t* from, uint32_t lds) {
  lds_dma16_at<64 * X, (1024 - 64) * X>(from, lane, lds);  // the instruction's offset moves both addresses
}

template <int DP, bool WHOLE, int X = 0>
__device__ __forceinline__ void dma_k_from(const CacheArgs& c, const Lanes<DP>& l, const uint8_t* from, uint32_t lds) {
  if constexpr (X < DP / 32) {
    if (WHOLE || l.k_in_head(c, X))
      dma_k_one<X>(l.k, from, lds);
    dma_k_from<DP, WHOLE, X + 1>(c, l, from, lds);
  }
}

template <int DP, bool WHOLE, int X = 0>
__device__ __forceinline__ void dma_v_from(const CacheArgs& c, const Lanes<DP>& l, const uint8_t* from, uint32_t lds) {
  if constexpr (X < DP / 32) {
    if (WHOLE || l.v_in_head(c, X))
      lds_dma16_at<0, 1024 * X>(from, l.v[X], lds);
    dma_v_from<DP, WHOLE, X + 1>(c, l, from, lds);
  }
}

// The transfer x of an unrolled loop.
template <int DP, int X = 0>
__device__ __forceinline__ void dma_at(int x, bool k, bool v, const Lanes<DP>& l, const uint8_t* from_k, const uint8_t* from_v, uint32_t lds, uint32_t lds_v) {
  if constexpr (X < DP / 32) {
    if (x == X) {
      if (k)
        dma_k_one<X>(l.k, from_k, lds);
      if (v)
        lds_dma16_at<0, 1024 * X>(from_v, l.v[X], lds_v);
      return;
    }
    dma_at<DP, X + 1>(x, k, v, l, from_k, from_v, lds, lds_v);
  }
}

// K and V of 16 tokens, `lds` and `from` wave-uniform.
template <int DP>
__device__ __forceinline__ void dma_k(const CacheArgs& c, const Lanes<DP>& l, const uint8_t* from, uint32_t lds) {
  if (c.dim == DP)
    dma_k_from<DP, true>(c, l, from, lds);
  else
    dma_k_from<DP, false>(c, l, from, lds);
}

template <int DP>
__device__ __forceinline__ void dma_v(const CacheArgs& c, const Lanes<DP>& l, const uint8_t* from, uint32_t lds) {
  if (c.dim == DP)
    dma_v_from<DP, true>(c, l, from, lds);
  else
    dma_v_from<DP, false>(c, l, from, lds);
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// Of a tile's transfers of K by dma_k, one after another, only those that have a lane in the
// head are made: where a head's last 32 elements are all padding, one less of each
// 16 tokens.  (Those of V have lanes in the head all.)
constexpr bool one_transfer_at_most() {
  for (int dim = 8; dim <= 256; dim += 8)
    if ((dim + 31) / 32 < AttentionShape::padded(dim) / 32 - 1)
      return false;
  return true;
}
static_assert(one_transfer_at_most(), "one transfer of 16 tokens may be left out, not two");

// All transfers are done but those of K of the 32 tokens asked for last.
template <int DP>
__device__ __forceinline__ void wait_loads_before_k(const CacheArgs& c) {
  if (c.dim + 32 <= DP)
    wait_loads<DP / 16 - 2>();
  else
    wait_loads<DP / 16>();
}

// Every read of LDS so far is done (a transfer may overwrite what it read).
__device__ __forceinline__ void wait_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <typename T>
__device__ __forceinline__ void store4(T* p, f4_t v) {
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  vec y;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    y[e] = (T)v[e];
  *reinterpret_cast<vec*>(p) = y;
}

template <typename T>
__device__ __forceinline__ T* out_row(const AttentionArgs& a, int start, int head, int u) {
  const int t = token_of(a, u), h = head * a.group + (u - t * a.group);
  return static_cast<T*>(a.out) + (int64_t)(start + t) * a.out_row + (int64_t)h * a.out_head;
}

// ---- units that stretches share ------------------------------------------------------
// The sums of stretch r's first unit are in slot 2 r of the workspace, those of its
// last one in slot 2 r + 1: QB rows of DP values (chunks: as their waves hold them),
// and behind all slots each row's maximum and sum of weights.  They are written and
// read past the caches, which workgroups on different XCDs do not share.

template <int DP, int QB>
__device__ __forceinline__ float* part_row(const AttentionArgs& a, int64_t slot, int row) {
  return a.part + (slot * QB + row) * DP;
}

template <int DP, int QB>
__device__ __forceinline__ float* part_weights(const AttentionArgs& a, int64_t slot, int row) {
  return a.part + 2 * (int64_t)a.stretches * QB * DP + (slot * QB + row) * 2;
}

__device__ __forceinline__ float2 load_part(const float* p) {
  return __builtin_bit_cast(float2, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM));
}

// Called by all threads once their sums are stored: whether this workgroup is the
// last of the unit's `parts` stretches from r0 on.
__device__ __forceinline__ bool last_of_unit(const AttentionArgs& a, int r0, int parts) {
  __shared__ int arrived;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    arrived = count_arrival(a.counters + r0);
  __syncthreads();
  if (arrived != parts - 1)
    return false;
  if (threadIdx.x == 0)
    reset_counter(a.counters + r0);
  return true;
}

// Few rows: the last workgroup joins the sums.  A lane holds 4 values of a row; what
// bounds it is the way to memory, so the loads of eight stretches are on their way at
// once.
template <typename T, int DP, int QB, int EXTRA, int NW>
__device__ __forceinline__ void join_unit(const AttentionArgs& a, const Line& line, const Place& p, int start, int wave) {
  constexpr int kLanes = DP <= 64 ? 16 : DP <= 128 ? 32 : 64, kRows = NW * (64 / kLanes);  // lanes of a row, rows at once
  constexpr int kAtOnce = 8;
  const int lane = threadIdx.x & 63, d = 4 * (lane & (kLanes - 1)), row = wave * (64 / kLanes) + lane / kLanes;
  const Unit& u = p.unit;
  const int r0 = line.of(p.at), parts = line.of(p.at + u.tiles - 1) - r0 + 1, rows = u.row_end - u.row;
  if (!last_of_unit(a, r0, parts))
    return;
  // Stretch r0 began before the unit, or with it; the others within it.
  const int late = line.start(r0) < p.at - EXTRA ? 1 : 0;
#pragma unroll 1
  for (int r = row; r < rows; r += kRows) {
    float m = -INFINITY, l = 0.0f;
    f4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int s0 = 0; s0 < parts; s0 += kAtOnce) {
      float2 w[kAtOnce], lo[kAtOnce], hi[kAtOnce];
#pragma unroll
      for (int s = 0; s < kAtOnce; ++s) {
        // Past the last stretch or value: the last one again, left out below.
        const int at = s0 + s < parts ? s0 + s : parts - 1;
        const int64_t slot = 2 * (int64_t)(r0 + at) + (at == 0 ? late : 0);
        const float* v = part_row<DP, QB>(a, slot, r) + (d < DP ? d : 0);
        w[s] = load_part(part_weights<DP, QB>(a, slot, r));
        lo[s] = load_part(v);
        hi[s] = load_part(v + 2);
      }
#pragma unroll
      for (int s = 0; s < kAtOnce; ++s)
        if (s0 + s < parts) {
          const float in = w[s].x, top = fmaxf(m, in), old = share(m, top), f = share(in, top);
          m = top;
          l = l * old + f * w[s].y;
          o = o * old + f * f4_t{lo[s].x, lo[s].y, hi[s].x, hi[s].y};
        }
    }
    if (d < a.cache.dim)
      store4(out_row<T>(a, start, p.head, u.row + r) + d, row_values(o, l, m));
  }
}

// Chunks: every wave stores the sums of its 16 NQ rows as its lanes hold them, 1 KB
// at a time, and the waves of the last workgroup add those of the other stretches to
// their own (at their place in the order), all of a stretch on their way at once.
// 821 fp32 rows take 66 us so, 76 with the values laid out by rows and the loads of 8
// rows and 2 stretches at once; 8192 rows 572 and 586.
template <int DP, int NQ, int NW>
__device__ __forceinline__ void store_sums(const AttentionArgs& a, int slot, int wave, const Sums<DP, NQ>& sums, const float (&l)[NQ]) {
  constexpr int QB = 16 * NW * NQ;
  const int lane = threadIdx.x & 63;
  float* o = part_row<DP, QB>(a, slot, wave * 16 * NQ) + lane * 4;
#pragma unroll
  for (int y = 0; y < NQ; ++y) {
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
      store_coherent4(o + (y * (DP / 16) + d) * 256, sums.o[y][d]);
    if (lane < 16) {
      float* ml = part_weights<DP, QB>(a, slot, wave * 16 * NQ + 16 * y + lane);
      store_coherent(ml, sums.m[y]);
      store_coherent(ml + 1, l[y]);
    }
  }
}

// `own`: this workgroup's stretch, whose sums become the unit's.
template <int DP, int NQ, int NW>
__device__ __forceinline__ void add_stretches(const AttentionArgs& a, int r0, int parts, int late, int own, int wave, Sums<DP, NQ>& sums, float (&l)[NQ]) {
  constexpr int QB = 16 * NW * NQ, ND = DP / 16;
  constexpr int kAtOnce = NQ * DP <= 256 ? NQ : 1;  // 16-row tiles beside the wave's own in registers
  constexpr int kPastCaches = 17;                   // sc0 sc1
  const int lane = threadIdx.x & 63;
  const uint32_t floats = 2 * (uint32_t)a.stretches * QB * DP;
  const auto from = __builtin_amdgcn_make_buffer_rsrc(a.part, 0, (int)((floats + 2 * (uint32_t)a.stretches * QB * 2) * 4), 0x00020000);
#pragma unroll
  for (int y0 = 0; y0 < NQ; y0 += kAtOnce) {
    f4_t o[kAtOnce][ND];
    float m[kAtOnce], w[kAtOnce];
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y) {
      m[y] = -INFINITY;
      w[y] = 0.0f;
#pragma unroll
      for (int d = 0; d < ND; ++d)
        o[y][d] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll 1
    for (int s = 0; s < parts; ++s) {
      const uint32_t row = (uint32_t)(2 * (r0 + s) + (s == 0 ? late : 0)) * QB + wave * 16 * NQ;  // wave-uniform
#pragma unroll
      for (int y = 0; y < kAtOnce; ++y) {
        f4_t f[ND];
        float in = sums.m[y0 + y], weights = l[y0 + y];
        if (r0 + s == own) {
#pragma unroll
          for (int d = 0; d < ND; ++d)
            f[d] = sums.o[y0 + y][d];
        } else {
          const auto ml = __builtin_amdgcn_raw_buffer_load_b64(from, (lane & 15) * 8, (int)((floats + (row + 16 * (y0 + y)) * 2) * 4), kPastCaches);
#pragma unroll
          for (int d = 0; d < ND; ++d)
            f[d] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(from, lane * 16, (int)((row * DP + ((y0 + y) * ND + d) * 256) * 4), kPastCaches));
          in = __builtin_bit_cast(float, (uint32_t)ml[0]);
          weights = __builtin_bit_cast(float, (uint32_t)ml[1]);
        }
        const float top = fmaxf(m[y], in);
        const float old = m[y] == top ? 1.0f : __builtin_amdgcn_exp2f(m[y] - top), now = in == top ? 1.0f : __builtin_amdgcn_exp2f(in - top);
        m[y] = top;
        w[y] = w[y] * old + now * weights;
#pragma unroll
        for (int d = 0; d < ND; ++d)
          o[y][d] = o[y][d] * old + now * f[d];
      }
    }
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y) {
      sums.m[y0 + y] = m[y];
      l[y0 + y] = w[y];
#pragma unroll
      for (int d = 0; d < ND; ++d)
        sums.o[y0 + y][d] = o[y][d];
    }
  }
}

// ----------------------------------------------------------------------------
// Chunks of tokens: NW waves of 16 NQ query rows each over the same key tiles,
// two buffers of K and V in LDS, the next tile's transfers under the present
// tile's products.  8192 fp16 rows of 32 / 8 heads of 128 take 579 us (950 TFLOP/s):
// of a tile's 4000 clocks, a wave spends 660 to 950 on K Q^T, 1100 to 1220 on the weights
// and 970 to 1020 on V P^T, and the other wave of its SIMD does not always have
// what would fill them.  2048 rows of 16 / 4 heads of 256 take 231 us (788 TFLOP/s),
// bound by LDS: a fragment feeds the products of 16 rows there, not 32.  Ragged
// prompts (821 fp32 rows, window 1024) take 65 us: 17 tiles a workgroup, 35 us of it at
// 8192 rows' pace, and the beginnings and ends of units, nearly all of them shared.
// ----------------------------------------------------------------------------
template <typename T, int DP, int NQ, int NW, int TK, bool FORM>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2))) void attention_chunk_kernel(AttentionArgs a) {
  constexpr int QB = 16 * NW * NQ, NA = TK / 16, kTile = TK * DP * 2, kExtra = AttentionShape::chunk_extra;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * kTile];  // K, V of two tiles
  const CacheArgs& c = a.cache;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
  __shared__ int kept[kSequenceInts];
  const Sequences loaded = load_sequences(a);
  const Units near = units_from<QB, TK, kExtra>(a, loaded, 0);
  const Line line = make_line<QB, TK, kExtra, AttentionShape::chunk_least>(a, loaded, near);
  const int stretches = line.stretches();
  if ((int)blockIdx.x >= stretches)
    return;
  if (wave == 0)
    keep_sequences(loaded, kept);
  __syncthreads();
  // Neighbouring stretches read the same keys: they go to one XCD (workgroup L runs
  // on XCD L % 8).
  const int xcd = (int)blockIdx.x & 7, more = stretches & 7;
  const int wg = xcd * (stretches >> 3) + (xcd < more ? xcd : more) + ((int)blockIdx.x >> 3);
  const int begin = line.start(wg), end = line.end(wg);
  if (c.dim != DP) {
    for (int i = tid; i < 4 * kTile / 16; i += 64 * NW)
      reinterpret_cast<u4_t*>(lds)[i] = u4_t{0, 0, 0, 0};
    __syncthreads();
  }
  Lanes<DP> from;
  from.set(c);
  Place p = locate<QB, TK, kExtra>(a, loaded, line, near, begin);
  int t0 = begin > p.at ? begin - p.at : 0;  // the unit's first tile in the stretch
  bool leading = true;  // the stretch's first unit
  while (true) {
    const Sequences seqs = kept_sequences(kept);  // anew for each unit: no registers under its products
    const Unit& u = p.unit;
    const int start = lane_value(seqs.start, u.seq);
    const int left = u.tiles - t0, room = end - p.at - t0, n = room < left ? room : left;
    if (n <= 0)
      return;  // the stretch ends before the unit's tiles
    const int row = u.row + wave * 16 * NQ;
    // What the wave's rows see, at most and at least.
    const int first = lane_value(seqs.first, u.seq), cap = lane_value(seqs.cap, u.seq);
    const int last = (row + 16 * NQ < u.row_end ? row + 16 * NQ : u.row_end) - 1;
    const bool active = row < u.row_end;
    const int ta = first + token_of(a, row) + 1, tb = first + token_of(a, active ? last : row) + 1;
    const int hi_least = ta < cap ? ta : cap, hi_most = tb < cap ? tb : cap;
    const int lo_least = a.window && ta > a.window ? ta - a.window : 0, lo_most = a.window && tb > a.window ? tb - a.window : 0;
    const bool none = u.hi <= u.lo;
    // What all rows of the unit see.
    const int ua = first + token_of(a, u.row) + 1, ub = first + token_of(a, u.row_end - 1) + 1;
    const int unit_hi = ua < cap ? ua : cap, unit_lo = a.window && ub > a.window ? ub - a.window : 0;
    Pages pages;
    pages.open(a, seqs, u.seq);
    uint32_t there = 0;
    // A wave transfers K, V or both of 16 of the tile's tokens.
    static_assert(NW == NA || NW == 2 * NA, "16 tokens to a wave");
    const int group = wave % NA;
    const uint8_t* const k_head = uniform_ptr(static_cast<const uint8_t*>(c.k) + (int64_t)p.head * c.head_stride * 2);
    const uint8_t* const v_head = uniform_ptr(static_cast<const uint8_t*>(c.v) + (int64_t)p.head * c.head_stride * 2);
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_addr(lds) + group * (DP / 32) * 1024);
    constexpr bool kBoth = NW == NA;
    const bool k_mine = kBoth || wave < NA, v_mine = kBoth || wave >= NA;
    const uint8_t *k_next = nullptr, *v_next = nullptr;  // where the next tile's transfers come from and go to
    uint32_t to_next = 0;
    const auto find = [&](int t, int buffer) {
      const int key = u.lo + t * TK, mine = key + 16 * group;
      pages.reach(a, key >> c.page_log);
      const int page = pages.page(mine >> c.page_log);
      if (c.page_log >= (TK == 64 ? 6 : 5)) {
        there = page >= 0 ? (1u << NA) - 1 : 0u;
      } else {
        there = 0;
#pragma unroll
        for (int b = 0; b < NA; ++b)
          there |= pages.page((key + 16 * b) >> c.page_log) >= 0 ? 1u << b : 0u;
      }
      const int64_t at = Pages::bytes(c, page, mine);
      k_next = k_head + at;
      v_next = v_head + at;
      to_next = to + buffer * 2 * kTile;
    };
    const auto fetch = [&]() {
      if (k_mine)
        dma_k<DP>(c, from, k_next, to_next);
      if (v_mine)
        dma_v<DP>(c, from, v_next, to_next + kTile);
    };
    if (!none) {
      find(t0, 0);
      __syncthreads();  // the buffers' last readers are done
      __builtin_amdgcn_sched_barrier(0);
      fetch();
    }
    Rows<T, DP, NQ> rows;  // on their way with the first tile
    rows.load(a, seqs, u, p.head, row);
    Sums<DP, NQ> sums;
    sums.clear();
    if (!none) {
      for (int t = 0; t < n; ++t) {
        const uint32_t here = there;
        wait_loads<0>();
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
        bool asks = t + 1 < n;
        if (asks)
          find(t0 + t + 1, (t + 1) & 1);
        const int key = u.lo + (t0 + t) * TK;
        uint8_t* const k = lds + (t & 1) * 2 * kTile;
        const bool most = active && key < hi_most && key + TK > lo_least;
        if (__builtin_expect(key + TK > unit_hi || key < unit_lo || here != (1u << NA) - 1, 0)) {
          if (__syncthreads_or(odd_values<64 * NW, kTile>(k + kTile, tid))) {
            if (most)
#pragma unroll 1
              for (int h = 0; h < NA / 2; ++h)
                mark_values<T, DP, NQ>(a, k + kTile + h * 32 * DP * 2, rows, key + 32 * h, here >> (2 * h), sums);
            __syncthreads();
            clear_values<64 * NW, kTile>(k + kTile, tid);
            __syncthreads();
          }
        }
        // The next tile's transfers go between the first products: all at once they
        // would wait for the way to the caches before the products begin (1130 to 2510
        // clocks of a tile of 5700).
        if (__builtin_expect(asks && (!most || c.dim != DP), 0)) {
          fetch();
          asks = false;
        }
        if (__builtin_expect(!most, 0))
          continue;
        const bool whole = key + TK <= hi_least && key >= lo_most && here == (1u << NA) - 1;
        f4_t s[NA][NQ];
        scores<T, DP, NQ, NA>(k, rows, s, [&](int d) {
          if (asks)
            dma_at<DP>(d, k_mine, v_mine, from, k_next, v_next, to_next, to_next + kTile);
        });
        finish_scores<T, DP, NQ, NA>(a, rows, key, whole, here, FORM, s, sums.some);
        sums.weigh(s, [&](int y) { return FORM ? 1.0f : rows.factor(y); });
#pragma unroll
        for (int h = 0; h < NA / 2; ++h) {
          add_values<T, DP, NQ, Rows<T, DP, NQ>::kParts>(k + kTile + h * 32 * DP * 2, s[2 * h], s[2 * h + 1], sums);
        }
      }
    }
    if (__builtin_expect(sums.far, 0))
      sum_again<T, DP, NQ, TK>(a, kept_sequences(kept), u, p.head, row, u.lo + t0 * TK, u.lo + (t0 + n) * TK, TK, sums);
    float l[NQ];
#pragma unroll
    for (int y = 0; y < NQ; ++y)
      l[y] = row_sum(sums.l[y]);
    sums.settle();
    // Whole units are done; the sums of others go to the workspace, and the last of
    // their workgroups goes on with all of them.
    bool done = n == u.tiles;
    if (!done) {
      if (active)
        store_sums<DP, NQ, NW>(a, 2 * wg + (leading ? 0 : 1), wave, sums, l);
      const int r0 = line.of(p.at), parts = line.of(p.at + u.tiles - 1) - r0 + 1;
      done = last_of_unit(a, r0, parts);
      // Stretch r0 began before the unit, or with it; the others within it.
      if (done && active)
        add_stretches<DP, NQ, NW>(a, r0, parts, line.start(r0) < p.at - kExtra ? 1 : 0, wg, wave, sums, l);
    }
    if (done) {
      if (__builtin_expect(__any(sums.odd(l)), 0))
        mark_again<DP, NQ>(a, kept_sequences(kept), u, p.head, row, u.lo, u.lo + u.tiles * TK, sums);
#pragma unroll
      for (int y = 0; y < NQ; ++y) {
        const int r = row + 16 * y + (lane & 15);
        if (r >= u.row_end)
          continue;
        T* o = out_row<T>(a, start, p.head, r);
#pragma unroll
        for (int d = 0; d < DP / 16; ++d)
          if (16 * d + 4 * g < c.dim)
            store4(o + 16 * d + 4 * g, row_values(sums.o[y][d], l[y], sums.m[y]));
      }
    }
    if (p.at + t0 + n >= end)
      return;
    leading = false;
    t0 = 0;
    p = behind<QB, TK, kExtra>(a, kept_sequences(kept), p);
  }
}

// ----------------------------------------------------------------------------
// Few query rows: every wave takes every NW-th tile of 32 keys of its workgroup's
// stretch, with a buffer for K and one for V of its own, refilled as soon as each
// has been read; the waves' sums join in LDS at the end of a unit.  Bound by the
// reading of K and V: 8 rows of 16 / 4 heads of 256 over 1.2 GB of them take 210 us
// (5.75 TB/s), 40 capped fp32 rows of 32 / 8 heads of 128 over 304 MB 70 us.  One
// row over 777 keys takes 15 us, the latency of its steps: units of the line, rows
// and keys, the waves' sums, the stretches' sums.  Four waves: with eight, heads of 128
// of 8 sequences take 20.1 us in place of 17.0 (fp32 rows, 1024 keys; fp16 16.6 and
// 15.3) and, over 16384 keys, 54.4 in place of 56.4 (fp16; fp32 57.7 and 57.1).
// ----------------------------------------------------------------------------
template <typename T, int DP, int NQ, int NW>
__global__ __launch_bounds__(64 * NW) void attention_rows_kernel(AttentionArgs a) {
  constexpr int QB = 16 * NQ, TK = 32, kTile = TK * DP * 2, kExtra = AttentionShape::rows_extra, kLoads = DP / 16;
  static_assert(NW * 16 * DP * 4 <= NW * 2 * kTile, "the waves' sums fit into the buffers");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[NW * 2 * kTile];
  __shared__ float sm[NW][QB], sl[NW][QB];
  const CacheArgs& c = a.cache;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
  __shared__ int kept[kSequenceInts];
  const Sequences loaded = load_sequences(a);
  const Units near = units_from<QB, TK, kExtra>(a, loaded, 0);
  const Line line = make_line<QB, TK, kExtra, NW>(a, loaded, near);
  const int wg = (int)blockIdx.x;
  if (wg >= line.stretches())
    return;
  if (wave == 0)
    keep_sequences(loaded, kept);
  __syncthreads();
  const int begin = line.start(wg), end = line.end(wg);
  Lanes<DP> from;
  from.set(c);
  uint8_t* const mine = lds + wave * 2 * kTile;
  const uint32_t at = __builtin_amdgcn_readfirstlane(lds_addr(mine));
  const bool formed = a.softcap > 0.0f || a.slopes;
  Place p = locate<QB, TK, kExtra>(a, loaded, line, near, begin);
  int t0 = begin > p.at ? begin - p.at : 0;  // the unit's first tile in the stretch
  bool leading = true;
  while (true) {
    const Sequences seqs = kept_sequences(kept);  // anew for each unit: no registers under its products
    const Unit& u = p.unit;
    const int start = lane_value(seqs.start, u.seq);
    const int left = u.tiles - t0, room = end - p.at - t0, n = room < left ? room : left;
    if (n <= 0)
      return;  // the stretch ends before the unit's tiles
    const int first = lane_value(seqs.first, u.seq), cap = lane_value(seqs.cap, u.seq);
    const int ta = first + token_of(a, u.row) + 1, tb = first + token_of(a, u.row_end - 1) + 1;
    const int hi_least = ta < cap ? ta : cap, lo_most = a.window && tb > a.window ? tb - a.window : 0;
    Pages pages;
    pages.open(a, seqs, u.seq);
    if (c.dim != DP)  // chunks that are not loaded are zero (the buffers held sums before)
      for (int i = lane; i < 2 * kTile / 16; i += 64)
        reinterpret_cast<u4_t*>(mine)[i] = u4_t{0, 0, 0, 0};
    wait_lds();
    uint32_t there = 0;
    int64_t from_page[2] = {0, 0};
    const uint8_t* const k_head = uniform_ptr(static_cast<const uint8_t*>(c.k) + (int64_t)p.head * c.head_stride * 2);
    const uint8_t* const v_head = uniform_ptr(static_cast<const uint8_t*>(c.v) + (int64_t)p.head * c.head_stride * 2);
    const auto open = [&](int t) {
      const int key = u.lo + t * TK;
      pages.reach(a, key >> c.page_log);
      const int first_page = pages.page(key >> c.page_log), second_page = pages.page((key + 16) >> c.page_log);
      from_page[0] = Pages::bytes(c, first_page, key);
      from_page[1] = Pages::bytes(c, second_page, key + 16);
      there = (first_page >= 0 ? 1u : 0u) | (second_page >= 0 ? 2u : 0u);
    };
    const auto fetch_k = [&]() {
#pragma unroll
      for (int b = 0; b < 2; ++b)
        dma_k<DP>(c, from, k_head + from_page[b], at + b * (DP / 32) * 1024);
    };
    const auto fetch_v = [&]() {
#pragma unroll
      for (int b = 0; b < 2; ++b)
        dma_v<DP>(c, from, v_head + from_page[b], at + kTile + b * (DP / 32) * 1024);
    };
    const bool busy = u.hi > u.lo && wave < n;
    if (busy) {
      open(t0 + wave);
      fetch_k();
      fetch_v();
    }
    Rows<T, DP, NQ> rows;  // on their way with the first keys
    rows.load(a, seqs, u, p.head, u.row);
    Sums<DP, NQ> sums;
    sums.clear();
    if (busy) {
      for (int t = wave; t < n; t += NW) {
        const int key = u.lo + (t0 + t) * TK;
        const uint32_t here = there;
        const bool whole = key + TK <= hi_least && key >= lo_most && here == 3u, more = t + NW < n;
        wait_loads<kLoads>();  // K is here, V (kLoads transfers, whatever the head) may be on its way
        f4_t s[2][NQ];
        scores<T, DP, NQ, 2>(mine, rows, s, [](int) {});
        wait_lds();
        if (more) {
          open(t0 + t + NW);
          fetch_k();
        }
        finish_scores<T, DP, NQ, 2>(a, rows, key, whole, here, formed, s, sums.some);
        sums.weigh(s, [&](int y) { return formed ? 1.0f : rows.factor(y); });
        if (more)
          wait_loads_before_k<DP>(c);
        else
          wait_loads<0>();
        if (!whole && __any(odd_values<64, kTile>(mine + kTile, lane))) {
          mark_values<T, DP, NQ>(a, mine + kTile, rows, key, here, sums);
          wait_lds();
          clear_values<64, kTile>(mine + kTile, lane);
          wait_lds();
        }
        add_values<T, DP, NQ, true>(mine + kTile, s[0], s[1], sums);
        wait_lds();
        if (more)
          fetch_v();
      }
    }
    if (__builtin_expect(sums.far, 0))
      sum_again<T, DP, NQ, TK>(a, kept_sequences(kept), u, p.head, u.row, u.lo + (t0 + wave) * TK, u.lo + (t0 + n) * TK, NW * TK, sums);
    float l[NQ];
#pragma unroll
    for (int y = 0; y < NQ; ++y)
      l[y] = row_sum(sums.l[y]);
    if (__builtin_expect(__any(sums.odd(l)), 0))
      mark_again<DP, NQ>(a, kept_sequences(kept), u, p.head, u.row, u.lo + t0 * TK, u.lo + (t0 + n) * TK, sums);
    sums.settle();
    // The waves' sums of each 16 rows, joined by all threads.
#pragma unroll
    for (int y = 0; y < NQ; ++y) {
      if (g == 0) {
        sm[wave][16 * y + (lane & 15)] = sums.m[y];
        sl[wave][16 * y + (lane & 15)] = l[y];
      }
    }
    const bool done = n == u.tiles;
    const int64_t slot = 2 * (int64_t)wg + (leading ? 0 : 1);
    float* const buffer = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int y = 0; y < NQ; ++y) {
      __syncthreads();  // every wave's products are done, and the rows before these are out
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
        *reinterpret_cast<f4_t*>(buffer + (wave * 16 + (lane & 15)) * DP + 16 * d + 4 * g) = sums.o[y][d];
      __syncthreads();
      for (int i = tid; i < 16 * DP / 4; i += 64 * NW) {
        const int rr = i / (DP / 4), d = 4 * (i - rr * (DP / 4)), r = u.row + 16 * y + rr;
        if (r >= u.row_end || d >= c.dim)
          continue;
        float top = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w)
          top = fmaxf(top, sm[w][16 * y + rr]);
        f4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float f = share(sm[w][16 * y + rr], top);
          l = fmaf(f, sl[w][16 * y + rr], l);
          o += f * *reinterpret_cast<const f4_t*>(buffer + (w * 16 + rr) * DP + d);
        }
        if (done) {
          store4(out_row<T>(a, start, p.head, r) + d, row_values(o, l, top));
        } else {
          store_coherent4(part_row<DP, QB>(a, slot, 16 * y + rr) + d, o);
          if (d == 0) {
            float* ml = part_weights<DP, QB>(a, slot, 16 * y + rr);
            store_coherent(ml, top);
            store_coherent(ml + 1, l);
          }
        }
      }
    }
    if (!done)
      join_unit<T, DP, QB, kExtra, NW>(a, line, p, start, wave);
    if (p.at + t0 + n >= end)
      return;
    leading = false;
    t0 = 0;
    p = behind<QB, TK, kExtra>(a, kept_sequences(kept), p);
    __syncthreads();  // before the buffers and statistics are used again
  }
}

template <typename T, int DP>
hipError_t launch_t(hipStream_t s, const AttentionArgs& a) {
  if (a.row_tiles) {
    if constexpr (AttentionShape::most_row_tiles(DP) > 1) {
      if (a.row_tiles == 2)
        return dispatch(attention_rows_kernel<T, DP, 2, 4>, dim3(a.stretches), dim3(256), s, a);
      if (a.row_tiles == 3)
        return dispatch(attention_rows_kernel<T, DP, 3, 4>, dim3(a.stretches), dim3(256), s, a);
    }
    return dispatch(attention_rows_kernel<T, DP, 1, 4>, dim3(a.stretches), dim3(256), s, a);
  }
  constexpr bool kF = sizeof(T) == 4;
  constexpr int NQ = AttentionShape::chunk_tiles(DP, kF), NW = AttentionShape::chunk_waves(DP, kF), TK = AttentionShape::chunk_keys(DP, kF);
  return a.softcap > 0.0f || a.slopes ? dispatch(attention_chunk_kernel<T, DP, NQ, NW, TK, true>, dim3(a.stretches), dim3(64 * NW), s, a)
                                      : dispatch(attention_chunk_kernel<T, DP, NQ, NW, TK, false>, dim3(a.stretches), dim3(64 * NW), s, a);
}

template <typename T>
hipError_t launch_d(hipStream_t s, const AttentionArgs& a) {
  switch (AttentionShape::padded(a.cache.dim)) {
    case 64:
      return launch_t<T, 64>(s, a);
    case 96:
      return launch_t<T, 96>(s, a);
    case 128:
      return launch_t<T, 128>(s, a);
    case 192:
      return launch_t<T, 192>(s, a);
    default:
      return launch_t<T, 256>(s, a);
  }
}

}  // namespace

// Which kernel, how many query rows a unit has, how many workgroups: by the
// counts of new rows, the heads and the head size, which the host knows.  Returns the
// cache heads that a launch may take (the line's places have 32 bits; 0: not one).
int attention_plan(AttentionArgs& a, int dtype, int cus, size_t* floats) {
  const CacheArgs& c = a.cache;
  int most = 0;
  for (int s = 0; s < c.nq; ++s)
    most = c.count[s] > most ? c.count[s] : most;
  const int rows = most * a.group;
  const int dp = AttentionShape::padded(c.dim);
  a.row_tiles = rows <= 16 * AttentionShape::most_row_tiles(dp) ? (rows + 15) / 16 : 0;
  const bool f32 = dtype == kF32;
  const int qb = a.row_tiles ? 16 * a.row_tiles : 16 * AttentionShape::chunk_waves(dp, f32) * AttentionShape::chunk_tiles(dp, f32);
  const int tk = a.row_tiles ? 32 : AttentionShape::chunk_keys(dp, f32);
  a.units = 0;
  for (int s = 0; s < c.nq; ++s) {
    a.unit[s] = a.units;
    a.units += (int)(((int64_t)c.count[s] * a.group + qb - 1) / qb);
  }
  // No more workgroups than tiles: as many as a table holds, for every unit.
  const int extra = a.row_tiles ? AttentionShape::rows_extra : AttentionShape::chunk_extra;
  const int64_t tiles = (int64_t)a.units * ((((int64_t)c.width << c.page_log) + tk - 1) / tk + 1 + extra);
  const int wgs = a.row_tiles ? cus : 8 / AttentionShape::chunk_waves(dp, f32) * cus;
  a.stretches = tiles * c.heads < wgs ? (int)(tiles * c.heads) : wgs;
  const auto inverse = [](int y) { return y == 1 ? ~0u : (uint32_t)((1ull << 32) / (uint32_t)y); };
  a.group_inverse = inverse(a.group);
  a.stretches_inverse = inverse(a.stretches);
  *floats = 2 * (size_t)a.stretches * qb * (dp + 2);
  // Stretches of up to 8 tiles more than their share, 32-bit places.
  const int64_t places = (1ll << 31) - 1 - 16ll * wgs;
  return tiles > places ? 0 : (int)(places / tiles < (int64_t)c.heads ? places / tiles : c.heads);
}

hipError_t launch_attention(hipStream_t s, const AttentionArgs& a, int dtype) {
  return dtype == kF32 ? launch_d<float>(s, a) : launch_d<_Float16>(s, a);
}

}  // namespace q4k
