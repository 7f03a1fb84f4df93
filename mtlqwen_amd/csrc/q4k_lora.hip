// Low-rank adapters of a packed batch, one per sequence, beside a projection:
// u = x A^T (lora_shrink_kernel) and y = aux + s u B^T (lora_expand_kernel), both in
// one launch for single rows and few ranks (lora_token_kernel), and gate_kernel, the
// gated epilogue of a projection with adapters.
#include "q4k_device.h"

namespace q4k {
namespace {

constexpr int kLoraMaxSlices = 8;
// The one-launch kernel's rounds of 8 ranks and 4096 k, times rows (lora_plan), and
// the ranks that this leaves it, in powers of two: four lanes' eight.
constexpr int kTokenRounds = 3, kTokenRanks = 32;
static_assert(8 * kTokenRounds <= kTokenRanks, "ranks of the one-launch kernel");

// Up to 16 RT rows that lie in one sequence: the first row, the rows, and the
// sequence's adapter (-1: none) with its rank.
struct LoraBlock {
  int row, rows, adapter, rank;
  float scale;
};

__device__ __forceinline__ LoraBlock lora_block(const LoraArgs& a, int tile, int tile_rows) {
  // Up to 64 slots: a wave reads all their ranks and scales while the sequence's
  // adapter is on its way, not after it.
  const int lane = threadIdx.x & 63;
  const bool few = a.slots <= 64;
  int ranks = a.r;
  float scales = 1.0f;
  if (few && lane < a.slots) {
    if (a.ranks)
      ranks = a.ranks[lane];
    if (a.scales)
      scales = a.scales[lane];
  }
  // a.tile[q] = tiles before sequence q; constant indices, so that the tables
  // are read in one go.
  int q = 0, row = a.start[0], rows = a.count[0], first = 0;
#pragma unroll
  for (int i = 1; i < 8; ++i)
    if (i < a.nq && tile >= a.tile[i]) {
      q = i;
      row = a.start[i];
      rows = a.count[i];
      first = a.tile[i];
    }
  LoraBlock b;
  b.row = row + (tile - first) * tile_rows;
  b.rows = min(rows - (tile - first) * tile_rows, tile_rows);
  b.adapter = __builtin_amdgcn_readfirstlane(a.ids[q]);
  if (b.adapter < 0 || b.adapter >= a.slots)
    b.adapter = -1;
  const int slot = max(b.adapter, 0);
  if (few) {
    b.rank = __builtin_amdgcn_readlane(ranks, slot);
    b.scale = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scales), slot));
  } else {
    b.rank = a.ranks ? a.ranks[slot] : a.r;
    b.scale = a.scales ? a.scales[slot] : 1.0f;
  }
  b.rank = b.adapter < 0 ? 0 : min(max(b.rank, 0), a.r);
  if (b.rank == 0)
    b.adapter = -1;
  return b;
}

// Power of two that brings a largest magnitude m to [2^14, 2^15), and its
// inverse: values scaled by it split into two fp16 parts, hi = fp16(v) and lo =
// fp16(v - hi), that keep 22 of v's bits down to 2^-17 of the largest, and all but
// 2^-25 of a scaled value (2^-39 of the largest) below that.  (m below 2^-112, infinities and NaN: the
// nearest such power.)
__device__ __forceinline__ float split_scale(float m, float* inverse) {
  const int e = min(max((int)(__builtin_bit_cast(uint32_t, m) >> 23), 15), 254);
  *inverse = __builtin_bit_cast(float, (uint32_t)(e - 14) << 23);
  return __builtin_bit_cast(float, (uint32_t)(268 - e) << 23);
}

// The parts of N values scaled.  The low part of an infinity is finite (its
// difference is no number), so that the infinity stays one.
template <int N, typename H>
__device__ __forceinline__ void split(const float* v, float scale, H* hi, H* lo) {
  typedef float f2_t __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    const f2_t s = {v[e] * scale, v[e + 1] * scale};
    const h2_t h = __builtin_convertvector(s, h2_t);
    const f2_t d = {__builtin_amdgcn_fmed3f(fmaf((float)h[0], -1.0f, s[0]), -64.0f, 64.0f),
                    __builtin_amdgcn_fmed3f(fmaf((float)h[1], -1.0f, s[1]), -64.0f, 64.0f)};
    const h2_t l = __builtin_convertvector(d, h2_t);
    (*hi)[e] = h[0];
    (*hi)[e + 1] = h[1];
    (*lo)[e] = l[0];
    (*lo)[e + 1] = l[1];
  }
}

// The maximum with another lane's value: CTRL 0xB1, 0x4E: lanes ^ 1 and ^ 2; 0x120
// + n: n lanes on within 16.
template <int CTRL>
__device__ __forceinline__ float max_lane(float v) {
  return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true)));
}

// The 16 bytes of lane 4 (lane % 16) + lane / 16: loads give each four lanes 64
// contiguous bytes of one row (16 cache lines an instruction), the matrix
// instructions want lane % 16 to be the row (loaded so, every lane of a
// quarter wave is in a line of its own, 64 an instruction, and a CU takes in 13
// bytes a cycle: 3.9 us for 128 KB).
__device__ __forceinline__ u4_t to_rows(u4_t v, int from) {
  u4_t o;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    o[e] = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)v[e]);
  return o;
}

typedef uint32_t u4_any_t __attribute__((ext_vector_type(4), aligned(2)));

// ----------------------------------------------------------------------------
// One wave's share of u[row][j] = sum over k of x[row][k] A[j][k]: 16 rows, 16 NT
// ranks, `steps` times 32 k, from the addresses x and w on (row or rank lane / 4 of
// their tile, k 8 (lane % 4)), the loads of SEG steps on their way together.
// v_mfma_f32_16x16x32_f16, whose products are exact; fp32 x as two fp16 parts
// (split_scale), which costs two of these instructions where eight fp32 ones of
// twice the time each would be needed.  The scale of a row follows the largest
// value so far; the sums follow it where it changes.
// acc[t][c]: row 4 (lane / 16) + c, rank 16 t + lane % 16.
// ----------------------------------------------------------------------------
template <typename T, int NT, int SEG>
__device__ __forceinline__ void lora_sum(const T* x, const _Float16* w, int steps, int k, int live, int lane, f4_t* acc) {
  constexpr int kX = (int)sizeof(T) / 2;  // 16-byte loads of 8 values
  const int g = lane >> 4, from = 4 * (4 * (lane & 15) + g);
  float inverse, scale = split_scale(0.0f, &inverse);
#pragma unroll
  for (int t = 0; t < NT; ++t)
    acc[t] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = 0; s0 < steps; s0 += SEG) {
    u4_t wv[SEG][NT], xv[SEG][kX];
#pragma unroll
    for (int s = 0; s < SEG; ++s)
      if (s0 + s < steps)
#pragma unroll
        for (int h = 0; h < kX; ++h)
          xv[s][h] = *reinterpret_cast<const u4_any_t*>(x + 32 * (s0 + s) + 4 * h);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int s = 0; s < SEG; ++s)
        wv[s][t] = u4_t{0u, 0u, 0u, 0u};
      if (16 * t + (lane >> 2) < live)
#pragma unroll
        for (int s = 0; s < SEG; ++s)
          if (s0 + s < steps)
            wv[s][t] = *reinterpret_cast<const u4_any_t*>(w + (size_t)(16 * t) * k + 32 * (s0 + s));
    }
    if constexpr (kX == 2) {
      float m = 0.0f;
#pragma unroll
      for (int s = 0; s < SEG; ++s)
        if (s0 + s < steps)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            m = fmaxf(m, fabsf(__builtin_bit_cast(float, (uint32_t)xv[s][e >> 2][e & 3])));
      m = max_lane<0x4E>(max_lane<0xB1>(m));
      // Lanes 4 i .. 4 i + 3 hold row i: its scale stays with them.
      float undo;
      const float now = split_scale(m, &undo);
      if (__any(now < scale)) {
        const float ratio = now < scale ? now * inverse : 1.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float q = __shfl(ratio, 4 * (4 * g + c));
#pragma unroll
          for (int t = 0; t < NT; ++t)
            acc[t][c] *= q;
        }
        if (now < scale) {
          scale = now;
          inverse = undo;
        }
      }
    }
#pragma unroll
    for (int s = 0; s < SEG; ++s)
      if (s0 + s < steps) {
        h8_t a[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
          a[t] = __builtin_bit_cast(h8_t, to_rows(wv[s][t], from));
        if constexpr (kX == 1) {
          const h8_t v = __builtin_bit_cast(h8_t, to_rows(xv[s][0], from));
#pragma unroll
          for (int t = 0; t < NT; ++t)
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, a[t], acc[t], 0, 0, 0);
        } else {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            v[e] = __builtin_bit_cast(float, (uint32_t)xv[s][e >> 2][e & 3]);
          h8_t hi, lo;
          split<8>(v, scale, &hi, &lo);
          hi = __builtin_bit_cast(h8_t, to_rows(__builtin_bit_cast(u4_t, hi), from));
          lo = __builtin_bit_cast(h8_t, to_rows(__builtin_bit_cast(u4_t, lo), from));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, a[t], acc[t], 0, 0, 0);
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, a[t], acc[t], 0, 0, 0);
          }
        }
      }
  }
  if constexpr (kX == 2)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float undo = __shfl(inverse, 4 * (4 * g + c));
#pragma unroll
      for (int t = 0; t < NT; ++t)
        acc[t][c] *= undo;
    }
}

// The waves' sums of one row and rank, added in pairs.
template <int WAVES>
__device__ __forceinline__ float sum_waves(const float* p, int stride) {
  float v[WAVES];
#pragma unroll
  for (int w = 0; w < WAVES; ++w)
    v[w] = p[w * stride];
#pragma unroll
  for (int n = WAVES / 2; n > 0; n /= 2)
#pragma unroll
    for (int w = 0; w < n; ++w)
      v[w] += v[w + n];
  return v[0];
}

// K in slices: one workgroup per 16 rows, slice and 16 NT ranks; its eight waves
// take a part of the slice each and add their sums in LDS.  A is read once per 16
// rows, from the L2.  The kernel's own time: 333 ragged fp16 rows of rank 64, k =
// 4096, 5.0 us; 2048 fp32 rows of rank 64 19.2 (x alone would take 6.7 at the rate
// of a copy; sharing A between 64 rows through LDS, four slices of it on their way,
// took 16.5 and 4.7 for adding twice the slices, and more for fewer rows).
template <typename T, int NT, int SEG>
__global__ __launch_bounds__(512, 4) void lora_shrink_kernel(LoraArgs a) {
  constexpr int kSums = NT * 256, kWaves = 8;
  __shared__ float red[kWaves * kSums];
  const LoraBlock b = lora_block(a, blockIdx.x, 16);
  const int j0 = (int)blockIdx.z * 16 * NT;
  if (b.adapter < 0 || j0 >= b.rank)
    return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, i = lane & 15, g = lane >> 4;
  // Units of 32 k per wave.
  const int units = a.k / (32 * kWaves), u0 = (int)((int64_t)units * blockIdx.y / a.slices), u1 = (int)((int64_t)units * (blockIdx.y + 1) / a.slices);
  const int k0 = 32 * (kWaves * u0 + wave * (u1 - u0)) + 8 * (lane & 3);
  f4_t acc[NT];
  lora_sum<T, NT, SEG>(static_cast<const T*>(a.x) + (size_t)(b.row + min(lane >> 2, b.rows - 1)) * a.k + k0,
                       a.a + ((size_t)b.adapter * a.r + j0 + (lane >> 2)) * a.k + k0, u1 - u0, a.k, b.rank - j0, lane, acc);
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      red[wave * kSums + (4 * g + c) * (16 * NT) + 16 * t + i] = acc[t][c];
  __syncthreads();
  float* part = a.part + ((size_t)blockIdx.y * a.m + b.row) * a.rpad + j0;
  for (int o = tid; o < kSums; o += 64 * kWaves) {
    const int row = o / (16 * NT), j = o % (16 * NT);
    if (row < b.rows && j0 + j < b.rank)
      part[(size_t)row * a.rpad + j] = sum_waves<kWaves>(red + o, kSums);
  }
}

// ----------------------------------------------------------------------------
// y[row][n] = aux[row][n] + sum over j of (s u[row][j]) B[n][j] for up to 16 a.rt
// rows and 64 columns a step: u (scaled by s) lies in LDS as two fp16 parts per
// row (split_scale); v_mfma_f32_16x16x32_f16.  Tile p holds columns 4 i + p, so
// that lane i of a lane group ends up with four consecutive columns of rows 4
// (lane / 16) .. + 3, and 16 lanes read and write one contiguous piece of a row.
// NC = 0: up to 16 ranks, both parts of u in one instruction (k groups 0, 1 the
// high part, 2, 3 the low, B given twice); NC = 1, 2: up to 32 NC ranks; NC = 3:
// any number, B read anew for each row tile.  A wave takes every WAVES-th step of
// the workgroup's columns; the loads of its first B and aux are on their way
// before u is there, those of the next aux before its products.  The kernel's own
// time: 2048 fp32 rows of 12288, rank 64, with aux 48.1 us, 4.2 TB/s of aux and y (a
// copy reaches 5.05); 333 ragged fp16 rows of 6144 10.4 us: the chain of loads from
// the sequence's id to the sums and B, and the sums themselves, which every workgroup
// adds up anew from its rows' slices (8 here, 64 KB to a workgroup).
// ----------------------------------------------------------------------------
struct LoraU {
  _Float16* part[2];  // [16 rt][pad] each
  float* undo;        // [16 rt]
  int pad;
};

template <typename T, int NC, int WAVES, bool PAST>
struct LoraColumns {
  static constexpr int kChunks = NC == 0 ? 1 : NC == 3 ? 1 : NC, P = 4;
  typedef T vec_t __attribute__((ext_vector_type(P), aligned(sizeof(T))));
  const LoraArgs& a;
  const LoraBlock& b;
  const _Float16* w;
  int i, g, end;
  h8_t bv[P][kChunks];
  vec_t x[4];

  __device__ __forceinline__ LoraColumns(const LoraArgs& args, const LoraBlock& block, int lane, int last)
      : a(args), b(block), w(args.b + (size_t)max(block.adapter, 0) * args.n * args.r), i(lane & 15), g(lane >> 4), end(last) {}

  // Ranks j .. j + 7 of column n, zero behind the adapter's rank.
  __device__ __forceinline__ h8_t ranks8(int n, int j) const {
    h8_t v = h8_t{0, 0, 0, 0, 0, 0, 0, 0};
    if (j + 8 <= b.rank) {
      if (n < a.n)
        v = *reinterpret_cast<const h8_any_t*>(w + (size_t)n * a.r + j);
      return v;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n < a.n && j + e < b.rank)
        v[e] = w[(size_t)n * a.r + j + e];
    return v;
  }

  __device__ __forceinline__ void load_b(int n0) {
    if constexpr (NC != 3)
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          bv[p][c] = ranks8(n0 + P * i + p, NC == 0 ? 8 * (g & 1) : 32 * c + 8 * g);
  }

  __device__ __forceinline__ size_t at(int n0, int t, int c) const { return (size_t)(b.row + 16 * t + 4 * g + c) * a.n + n0 + P * i; }

  __device__ __forceinline__ void load_aux(int n0, int t) {
    if (a.aux && n0 + P * i < a.n)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (16 * t + 4 * g + c < b.rows) {
          const vec_t* from = reinterpret_cast<const vec_t*>(static_cast<const T*>(a.aux) + at(n0, t, c));
          if constexpr (PAST)
            x[c] = __builtin_nontemporal_load(from);
          else
            x[c] = *from;
        }
  }

  __device__ __forceinline__ void first(int n0) {
    if (n0 < end) {
      load_b(n0);
      load_aux(n0, 0);
    }
  }

  // All columns of the wave, from n0 on.
  __device__ __forceinline__ void run(int n0, const LoraU& u) {
    const int tiles = (b.rows + 15) >> 4;
    const _Float16* const frag = (NC == 0 && g >= 2 ? u.part[1] : u.part[0]) + i * u.pad + (NC == 0 ? 8 * (g & 1) : 8 * g);
    const _Float16* const low = u.part[1] + i * u.pad + 8 * g;
    while (n0 < end) {
      for (int t = 0; t < tiles; ++t) {
        const bool last = t + 1 == tiles;
        const int next = n0 + 16 * P * WAVES;
        f4_t acc[P];
#pragma unroll
        for (int p = 0; p < P; ++p)
          acc[p] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
        float undo[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (b.adapter >= 0) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            undo[c] = u.undo[16 * t + 4 * g + c];
          const int ro = 16 * t * u.pad;
          if constexpr (NC == 3) {
            for (int j = 0; j < b.rank; j += 32) {
              const h8_t hi = *reinterpret_cast<const h8_t*>(frag + ro + j), lo = *reinterpret_cast<const h8_t*>(low + ro + j);
#pragma unroll
              for (int p = 0; p < P; ++p) {
                const h8_t v = ranks8(n0 + P * i + p, j + 8 * g);
                acc[p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, v, acc[p], 0, 0, 0);
                acc[p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, v, acc[p], 0, 0, 0);
              }
            }
          } else {
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
              const h8_t hi = *reinterpret_cast<const h8_t*>(frag + ro + 32 * c);
#pragma unroll
              for (int p = 0; p < P; ++p)
                acc[p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, bv[p][c], acc[p], 0, 0, 0);
              if constexpr (NC != 0) {
                const h8_t lo = *reinterpret_cast<const h8_t*>(low + ro + 32 * c);
#pragma unroll
                for (int p = 0; p < P; ++p)
                  acc[p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, bv[p][c], acc[p], 0, 0, 0);
              }
            }
          }
        }
        if (last && next < end)
          load_b(next);
        vec_t y[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int p = 0; p < P; ++p) {
            float o = a.aux ? (float)x[c][p] : 0.0f;
            if (b.adapter >= 0)
              o = fmaf(acc[p][c], undo[c], o);
            y[c][p] = (T)o;
          }
        if (!last)
          load_aux(n0, t + 1);
        else if (next < end)
          load_aux(next, 0);
        if (n0 + P * i < a.n)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (16 * t + 4 * g + c < b.rows) {
              vec_t* to = reinterpret_cast<vec_t*>(static_cast<T*>(a.y) + at(n0, t, c));
              if constexpr (PAST)
                __builtin_nontemporal_store(y[c], to);
              else
                *to = y[c];
            }
      }
      n0 += 16 * P * WAVES;
    }
  }
};

// Rank columns of u's parts in LDS: a multiple of 32 (16 for NC = 0) and 8, so that
// the rows of a tile start in different banks.
__host__ __device__ inline int lora_upad(int r) {
  return (r <= 16 ? 16 : (r + 31) / 32 * 32) + 8;
}

__host__ __device__ inline size_t lora_ubytes(int rows, int r) {
  return (size_t)rows * (2 * lora_upad(r) * sizeof(_Float16) + sizeof(float));
}

// The second launch: one workgroup per 16 a.rt rows of a sequence and a.span
// columns.  2^a.glog lanes take one row of u, four ranks each (Q times), add the slices'
// sums, low slices first, and split them.
// S slices at most; the loads of up to W rows per lane group are on their way together.
// PAST: aux and y past the caches (lora_expand).
template <typename T, int NC, int S, bool PAST>
__global__ __launch_bounds__(256, S > 2 || (sizeof(T) == 4 && NC == 2) ? 3 : 4) void lora_expand_kernel(LoraArgs a) {
  extern __shared__ _Float16 lds[];
  const uint32_t outer = blockIdx.x / a.inner, inner = blockIdx.x - outer * a.inner;
  const uint32_t tile = a.by_rows ? outer : inner, piece = a.by_rows ? inner : outer;
  const LoraBlock b = lora_block(a, (int)tile, 16 * a.rt);
  if (b.adapter < 0 && a.aux == a.y)
    return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int start = (int)piece * a.span, n0 = start + 64 * wave;
  LoraU u;
  u.pad = lora_upad(a.r);
  u.part[0] = lds;
  u.part[1] = lds + 16 * a.rt * u.pad;
  u.undo = reinterpret_cast<float*>(lds + 32 * a.rt * u.pad);
  LoraColumns<T, NC, 4, PAST> cols(a, b, lane, min(start + a.span, a.n));
  cols.first(n0);
  if (b.adapter >= 0) {
    constexpr int Q = NC == 3 ? 2 : 1, W = S > 2 ? 2 / Q : 4 / Q;
    const float scale = b.scale;
    const int q = tid & ((1 << a.glog) - 1), width = u.pad - 8, stride = 256 >> a.glog, rows16 = (b.rows + 15) & ~15;
    for (int row0 = tid >> a.glog; row0 < rows16; row0 += W * stride) {
      f4_t v[W][Q][S];
#pragma unroll
      for (int r = 0; r < W; ++r)
#pragma unroll
        for (int h = 0; h < Q; ++h)
#pragma unroll
          for (int sl = 0; sl < S; ++sl) {
            const int row = row0 + r * stride, j = 4 * (q + (h << a.glog));
            v[r][h][sl] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (row < b.rows && j < b.rank && sl < a.slices)
              v[r][h][sl] = *reinterpret_cast<const f4_t*>(a.part + ((size_t)sl * a.m + b.row + row) * a.rpad + j);
          }
#pragma unroll
      for (int r = 0; r < W; ++r) {
        const int row = row0 + r * stride;
        float m = 0.0f;
#pragma unroll
        for (int h = 0; h < Q; ++h) {
          const int j = 4 * (q + (h << a.glog));
#pragma unroll
          for (int sl = 1; sl < S; ++sl)
            v[r][h][0] += v[r][h][sl];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[r][h][0][e] = j + e < b.rank ? v[r][h][0][e] * scale : 0.0f;
            m = fmaxf(m, fabsf(v[r][h][0][e]));
          }
        }
        for (int off = (1 << a.glog) >> 1; off > 0; off >>= 1)
          m = fmaxf(m, __shfl_xor(m, off));
        float inverse;
        const float up = split_scale(m, &inverse);
        if (row >= rows16)
          continue;
#pragma unroll
        for (int h = 0; h < Q; ++h) {
          const int j = 4 * (q + (h << a.glog));
          if (j < width) {
            const float x[4] = {v[r][h][0][0], v[r][h][0][1], v[r][h][0][2], v[r][h][0][3]};
            h4_t hi, lo;
            split<4>(x, up, &hi, &lo);
            *reinterpret_cast<h4_t*>(u.part[0] + row * u.pad + j) = hi;
            *reinterpret_cast<h4_t*>(u.part[1] + row * u.pad + j) = lo;
          }
        }
        if (q == 0)
          u.undo[row] = inverse;
      }
    }
    __syncthreads();
  }
  cols.run(n0, u);
}

// The sum of a wave's lanes, in lane 63: within rows of 16 lanes, then across them.
__device__ __forceinline__ float sum_lanes(float v) {
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x111, 0xf, 0xf, true));  // row_shr:1
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x112, 0xf, 0xf, true));  // row_shr:2
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x114, 0xf, 0xf, true));  // row_shr:4
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x118, 0xf, 0xf, true));  // row_shr:8
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x142, 0xa, 0xf, true));  // row_bcast:15
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x143, 0xc, 0xf, true));  // row_bcast:31
  return v;
}

// ----------------------------------------------------------------------------
// Sequences of few rows and few ranks (decode) in one launch: every workgroup
// forms u of its sequence's rows itself, on the vector units in fp32 (a wave
// takes 512 k of one rank row in one contiguous load, 8 k per lane), and writes
// a.span columns: 1 << a.glog lanes share a column's ranks, 8 each.  A second
// launch would cost the caller more than reading A once per workgroup costs the L2:
// 8 sequences of one fp16 row, rank 16, 4096 -> 12288: 5.9 us replayed and 7.0 a
// call, in two launches 8.1 and 9.5; what bounds it is latency (launch, id, A, sum, B).
// ----------------------------------------------------------------------------
template <typename T, int ROWS>
__global__ __launch_bounds__(512) void lora_token_kernel(LoraArgs a) {
  __shared__ float red[8][ROWS][kTokenRanks], us[ROWS][kTokenRanks];
  const LoraBlock b = lora_block(a, blockIdx.x, ROWS);
  if (b.adapter < 0 && a.aux == a.y)
    return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int share = lane & ((1 << a.glog) - 1), step = 512 >> a.glog;  // columns of a round of the workgroup
  const int end = min((int)(blockIdx.y + 1) * a.span, a.n);
  int n = (int)blockIdx.y * a.span + (tid >> a.glog);
  const _Float16* bw = a.b + (size_t)max(b.adapter, 0) * a.n * a.r + 8 * share;
  h8_t bv;
  T x0[ROWS];
  const auto load = [&](int col) {
    bv = h8_t{0, 0, 0, 0, 0, 0, 0, 0};
    if (col >= end)
      return;
    const _Float16* src = bw + (size_t)col * a.r;
    if (8 * share + 8 <= b.rank)
      bv = *reinterpret_cast<const h8_any_t*>(src);
    else
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * share + e < b.rank)
          bv[e] = src[e];
    if (a.aux)
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        if (r < b.rows && (r & ((1 << a.glog) - 1)) == share)
          x0[r] = static_cast<const T*>(a.aux)[(size_t)(b.row + r) * a.n + col];
  };
  load(n);
  float v[ROWS][8];
  if (b.adapter >= 0) {
    const float scale = b.scale;
    const T* x = static_cast<const T*>(a.x) + (size_t)b.row * a.k + 512 * wave + 8 * lane;
    const _Float16* w = a.a + (size_t)b.adapter * a.r * a.k + 512 * wave + 8 * lane;
    // Rounds of 8 ranks and 4096 k, the next one's ranks on their way.
    const int segments = (a.k + 4095) >> 12, rounds = ((b.rank + 7) >> 3) * segments;
    const int ke = 512 * wave + 8 * lane;
    h8_t wv[8], wn[8];
    const auto ranks = [&](int j0, int k0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        wn[j] = h8_t{0, 0, 0, 0, 0, 0, 0, 0};
        if (k0 + ke < a.k && j0 + j < b.rank)
          wn[j] = *reinterpret_cast<const h8_any_t*>(w + (size_t)(j0 + j) * a.k + k0);
      }
    };
    float acc[ROWS][8];
    ranks(0, 0);
    for (int round = 0, j0 = 0, k0 = 0; round < rounds; ++round) {
      if (segments > 1 || round == 0)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            v[r][e] = 0.0f;
          if (k0 + ke < a.k && r < b.rows)
            load8(x + (size_t)r * a.k + k0, v[r]);
        }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        wv[j] = wn[j];
      const bool last = k0 + 4096 >= a.k;
      const int j1 = last ? j0 + 8 : j0, k1 = last ? 0 : k0 + 4096;
      if (round + 1 < rounds)
        ranks(j1, k1);
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        if (r < b.rows)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float t = k0 == 0 ? 0.0f : acc[r][j];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              t = fmaf((float)wv[j][e], v[r][e], t);
            acc[r][j] = t;
            if (last) {
              const float s = sum_lanes(t);
              if (lane == 63)
                red[wave][r][j0 + j] = s;
            }
          }
      j0 = j1;
      k0 = k1;
    }
    __syncthreads();
    if (tid < ROWS * kTokenRanks) {
      const int r = tid / kTokenRanks, j = tid % kTokenRanks;
      us[r][j] = r < b.rows && j < b.rank ? sum_waves<8>(&red[0][r][j], ROWS * kTokenRanks) * scale : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[r][e] = us[r][8 * share + e];
  }
  for (; n < end; n += step) {
    float o[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      o[r] = 0.0f;
      if (b.adapter >= 0 && r < b.rows) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          o[r] = fmaf((float)bv[e], v[r][e], o[r]);
        for (int off = 1; off < 1 << a.glog; off <<= 1)
          o[r] += __shfl_xor(o[r], off);
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (r < b.rows && (r & ((1 << a.glog) - 1)) == share)
        static_cast<T*>(a.y)[(size_t)(b.row + r) * a.n + n] = (T)(a.aux ? (float)x0[r] + o[r] : o[r]);
    load(n + step);
  }
}

// y = silu(aux) * t, 8 elements per thread.
template <typename T>
__global__ __launch_bounds__(256) void gate_kernel(const T* t, const T* aux, T* y, size_t chunks) {
  typedef T t8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  for (size_t c = (size_t)blockIdx.x * 256 + threadIdx.x; c < chunks; c += (size_t)gridDim.x * 256) {
    float v[8], g[8];
    load8(t + 8 * c, v);
    load8(aux + 8 * c, g);
    t8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      o[i] = (T)(silu(g[i]) * v[i]);
    *reinterpret_cast<t8*>(y + 8 * c) = o;
  }
}

int lora_tiles(const LoraArgs& a, int rows) {
  int t = 0;
  for (int q = 0; q < a.nq; ++q)
    t += (a.count[q] + rows - 1) / rows;
  return t;
}

// Fills a.tile for tiles of `rows` rows and returns their number.
int lora_lay_tiles(LoraArgs& a, int rows) {
  int t = 0;
  for (int q = 0; q < a.nq; ++q) {
    a.tile[q] = t;
    t += (a.count[q] + rows - 1) / rows;
  }
  return t;
}

template <typename T>
hipError_t lora_token(hipStream_t s, LoraArgs a, int cus) {
  int rows = 1;
  for (int q = 0; q < a.nq; ++q)
    rows = a.count[q] > rows ? a.count[q] : rows;
  const int tile = rows <= 1 ? 1 : 2, tiles = lora_lay_tiles(a, tile);
  a.glog = a.r <= 8 ? 0 : a.r <= 16 ? 1 : 2;
  const int round = 512 >> a.glog, rounds = (a.n + round - 1) / round;
  // One workgroup per CU: replayed 5.9 us (rank 16, above), with two 7.4.
  const int64_t steps = ((int64_t)tiles * rounds + cus - 1) / cus;
  a.span = round * (int)steps;
  const dim3 grid(tiles, (a.n + a.span - 1) / a.span), block(512);
  return tile == 1 ? dispatch(lora_token_kernel<T, 1>, grid, block, s, a) : dispatch(lora_token_kernel<T, 2>, grid, block, s, a);
}

template <typename T>
hipError_t lora_shrink(hipStream_t s, LoraArgs a) {
  const int rt = (a.r + 15) / 16;
  const dim3 grid(lora_lay_tiles(a, 16), a.slices, (rt + 3) / 4), block(512);
  if (rt == 1)
    return dispatch(lora_shrink_kernel<T, 1, 4>, grid, block, s, a);
  if (rt == 2)
    return dispatch(lora_shrink_kernel<T, 2, 2>, grid, block, s, a);
  return dispatch(lora_shrink_kernel<T, 4, 2>, grid, block, s, a);
}

template <typename T, int S, bool PAST>
hipError_t lora_expand_nc(hipStream_t s, const LoraArgs& a, dim3 grid, dim3 block, size_t lds) {
  if (a.r <= 16)
    return dispatch_lds(lora_expand_kernel<T, 0, S, PAST>, grid, block, lds, s, a);
  if (a.r <= 32)
    return dispatch_lds(lora_expand_kernel<T, 1, S, PAST>, grid, block, lds, s, a);
  if (a.r <= 64)
    return dispatch_lds(lora_expand_kernel<T, 2, S, PAST>, grid, block, lds, s, a);
  return dispatch_lds(lora_expand_kernel<T, 3, S, PAST>, grid, block, lds, s, a);
}

template <typename T>
hipError_t lora_expand(hipStream_t s, LoraArgs a, int cus) {
  // Row tiles that share a load of B and u's sums: two where the sequences fill
  // them, four where that still leaves four workgroups per CU and u's parts take 64
  // KB at most, two workgroups to a CU's LDS (ranks up to 224); one for ranks beyond
  // 256.  Calls back to back, both launches, 4096 inputs, rank 64, with aux, one / two
  // / four tiles: 64 fp16 rows of one sequence, 12288 outputs, 10.3 / 11.2 / 14.4 us;
  // 333 ragged ones, 6144 outputs, 15.8 / 15.7 / 17.6; 2048 ragged ones, 12288
  // outputs, 68.9 / 60.5 / 49.4, fp32 81.5 / 77.7 / 66.3.
  const int64_t blocks = (int64_t)(a.m / 64) * ((a.n + 255) / 256);
  a.rt = a.r > 256 || a.m < 32 * a.nq ? 1 : a.m >= 64 * a.nq && blocks >= 4 * (int64_t)cus && lora_ubytes(64, a.r) <= 65536 ? 4 : 2;
  const int tiles = lora_lay_tiles(a, 16 * a.rt);
  // Columns of a workgroup: at least four workgroups per CU.
  int steps = (int)(((int64_t)tiles * ((a.n + 255) / 256)) / (4 * (int64_t)cus));
  steps = steps < 1 ? 1 : steps > 16 ? 16 : steps;
  a.span = 256 * steps;
  // Lanes of a row of u: four ranks each, twice beyond 256 ranks.
  const int quads = (lora_upad(a.r) - 8) / 4;
  a.glog = 2;
  while ((1 << a.glog) < quads && a.glog < 6)
    ++a.glog;
  // Workgroups side by side continue each other's rows, for the memory's sake (calls
  // as above, 2048 rows, fp32: 66.2 us, column by column 71.4; 128 fp16 rows 14.5 and
  // 15.0); with few rows they take the sequences in turn, so that each XCD's L2 holds
  // the B of its own (20 rows of 4 sequences: 9.95 us, row by row 10.2).
  const uint32_t cols = (uint32_t)((a.n + a.span - 1) / a.span);
  a.by_rows = a.m > 64;
  a.inner = a.by_rows ? cols : (uint32_t)tiles;
  const dim3 grid((uint32_t)tiles * cols), block(256);
  const size_t lds = lora_ubytes(16 * a.rt, a.r);
  // Outputs that outgrow the caches are written past them, and aux read past
  // them: from 64 MB of both on, where nothing reads y next; of y alone where aux
  // is y or a projection reads y next.  Calls back to back, 4096 inputs, rank 64,
  // past / through the caches: with aux, 25 MB each 29.3 / 26.9 us, 34 MB 40.4 /
  // 43.3, 50 MB 41.7 / 44.7, 101 MB 66.3 / 71.0; in place, 50 MB 41.4 / 38.4, 101 MB
  // 65.8 / 71.4; linear_lora, 50 MB 148 / 144, 101 MB 273 / 278.
  const size_t y_bytes = (size_t)a.m * a.n * sizeof(T);
  const bool past = (a.aux && a.aux != a.y && !a.reread ? 2 : 1) * y_bytes >= 64u << 20;
  if (a.slices <= 2)
    return past ? lora_expand_nc<T, 2, true>(s, a, grid, block, lds) : lora_expand_nc<T, 2, false>(s, a, grid, block, lds);
  return past ? lora_expand_nc<T, kLoraMaxSlices, true>(s, a, grid, block, lds)
              : lora_expand_nc<T, kLoraMaxSlices, false>(s, a, grid, block, lds);
}

}  // namespace

void lora_plan(LoraArgs& a, int cus) {
  // Rounds of the one-launch kernel (8 ranks of the stack, 4096 k, one row; the
  // ranks in use are on the device).  Replayed back to back, fp16, 4096 -> 12288, 8
  // sequences: 1 round 4.1 us against 8.8 in two launches, 2 rounds 5.9 (8.1), with
  // two rows 5.2 (8.9), 3 rounds 8.5 (9.1), 12288 -> 4096 6.0 (9.1), 4 rounds 7.9 (8.2)
  // with two rows and 9.1 (8.0) with 32 ranks.
  int rows = 0;
  for (int q = 0; q < a.nq; ++q)
    rows = a.count[q] > rows ? a.count[q] : rows;
  a.one = rows <= 2 && rows * ((a.r + 7) / 8) * ((a.k + 4095) / 4096) <= kTokenRounds;
  if (a.one)
    return;
  // Workgroups for every CU, each with at least 256 k.
  const int tiles = lora_tiles(a, 16) * ((a.r + 63) / 64);
  int want = (cus + tiles - 1) / (tiles > 0 ? tiles : 1);
  want = want > kLoraMaxSlices ? kLoraMaxSlices : want;
  want = want > a.k / 256 ? a.k / 256 : want;
  a.slices = want < 1 ? 1 : want;
}

hipError_t launch_lora_token(hipStream_t s, const LoraArgs& a, int dtype, int cus) {
  return dtype == kF32 ? lora_token<float>(s, a, cus) : lora_token<_Float16>(s, a, cus);
}

hipError_t launch_lora_shrink(hipStream_t s, const LoraArgs& a, int dtype) {
  return dtype == kF32 ? lora_shrink<float>(s, a) : lora_shrink<_Float16>(s, a);
}

hipError_t launch_lora_expand(hipStream_t s, const LoraArgs& a, int dtype, int cus) {
  return dtype == kF32 ? lora_expand<float>(s, a, cus) : lora_expand<_Float16>(s, a, cus);
}

hipError_t launch_gate(hipStream_t s, const void* t, const void* aux, void* y, size_t elems, int dtype) {
  const size_t chunks = elems / 8;
  const dim3 grid((unsigned)((chunks + 255) / 256 < 8192 ? (chunks + 255) / 256 : 8192)), block(256);
  if (dtype == kF32)
    return dispatch(gate_kernel<float>, grid, block, s, static_cast<const float*>(t), static_cast<const float*>(aux), static_cast<float*>(y), chunks);
  return dispatch(gate_kernel<_Float16>, grid, block, s, static_cast<const _Float16*>(t), static_cast<const _Float16*>(aux),
                  static_cast<_Float16*>(y), chunks);
}

}  // namespace q4k
