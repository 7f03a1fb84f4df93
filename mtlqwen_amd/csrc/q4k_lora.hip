// Low-rank adapters of a packed batch, one per sequence, beside a projection:
// lora_shrink_kernel (u = x A^T), lora_expand_kernel (y = aux + s u B^T) and
// gate_kernel (the gated epilogue of a projection with adapters).
#include "q4k_device.h"

namespace q4k {
namespace {

// A block of up to 16 rows that lie in one sequence: its first row, its rows,
// and the sequence's adapter (-1: none) with its rank.
struct LoraBlock {
  int row, rows, adapter, rank;
};

__device__ __forceinline__ LoraBlock lora_block(const LoraArgs& a, int tile, int tile_rows) {
  int q = 0, t = tile;
  while (q + 1 < a.nq) {
    const int tiles = (a.count[q] + tile_rows - 1) / tile_rows;
    if (t < tiles)
      break;
    t -= tiles;
    ++q;
  }
  LoraBlock b;
  b.row = a.start[q] + t * tile_rows;
  b.rows = min(a.count[q] - t * tile_rows, tile_rows);
  b.adapter = a.ids[q];
  if (b.adapter < 0 || b.adapter >= a.slots)
    b.adapter = -1;
  b.rank = b.adapter < 0 ? 0 : a.ranks ? min(max(a.ranks[b.adapter], 0), a.r) : a.r;
  if (b.rank == 0)
    b.adapter = -1;
  return b;
}

// ----------------------------------------------------------------------------
// u[row][j] = sum over k of x[row][k] A[j][k], in K-slices: one workgroup per
// 16 rows, slice and 16 * NT ranks; its eight waves share the slice's blocks of
// 256 k, 32 k each, and add their sums in LDS.  fp16 x: v_mfma_f32_16x16x32_f16,
// whose products are exact.  fp32 x: v_mfma_f32_16x16x4_f32 on A converted to
// fp32, so that x keeps its 24 bits and its range.
// ----------------------------------------------------------------------------
template <typename T, int NT>
__global__ __launch_bounds__(512) void lora_shrink_kernel(LoraArgs a) {
  __shared__ float red[8][NT * 256];
  const LoraBlock b = lora_block(a, blockIdx.x, 16);
  const int j0 = (int)blockIdx.z * 16 * NT;
  if (b.adapter < 0 || j0 >= b.rank)
    return;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, i = lane & 15, g = lane >> 4;
  const int nb = a.k >> 8, b0 = (int)((int64_t)nb * blockIdx.y / a.slices), b1 = (int)((int64_t)nb * (blockIdx.y + 1) / a.slices);
  const T* x = static_cast<const T*>(a.x) + (size_t)(b.row + min(i, b.rows - 1)) * a.k + 32 * wave + 8 * g;
  const _Float16* w = a.a + ((size_t)b.adapter * a.r + j0) * a.k + 32 * wave + 8 * g;
  f4_t acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
    acc[t] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  for (int kb = b0; kb < b1; ++kb) {
    h8_t wv[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      wv[t] = h8_t{0, 0, 0, 0, 0, 0, 0, 0};
      if (j0 + 16 * t + i < b.rank)
        wv[t] = *reinterpret_cast<const h8_any_t*>(w + (size_t)(16 * t + i) * a.k + kb * 256);
    }
    if constexpr (sizeof(T) == 2) {
      const h8_t xv = *reinterpret_cast<const h8_any_t*>(x + kb * 256);
#pragma unroll
      for (int t = 0; t < NT; ++t)
        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xv, wv[t], acc[t], 0, 0, 0);
    } else {
      float xv[8];
      load8(x + kb * 256, xv);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[e], (float)wv[t][e], acc[t], 0, 0, 0);
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      red[wave][(4 * g + c) * (16 * NT) + 16 * t + i] = acc[t][c];
  __syncthreads();
  float* part = a.part + ((size_t)blockIdx.y * a.m + b.row) * a.rpad + j0;
  for (int o = tid; o < 256 * NT; o += 512) {
    const int row = o / (16 * NT), j = o % (16 * NT);
    if (row < b.rows && j0 + j < b.rank) {
      float p[8];
#pragma unroll
      for (int wv = 0; wv < 8; ++wv)
        p[wv] = red[wv][o];
      part[(size_t)row * a.rpad + j] = sum8_pairs(p);
    }
  }
}

// ----------------------------------------------------------------------------
// y[row][n] = aux[row][n] + sum over j of (s u[row][j]) B[n][j]: one workgroup
// per 16 * RT rows of a sequence and 128 * CT columns.  The slices' sums are
// added (low slices first) into LDS, scaled, as fp32; the products are
// v_mfma_f32_16x16x4_f32 with B as the row operand, so that a lane ends up with
// consecutive columns of one row: two tiles cover 32 columns, lane group g
// holding 8g .. 8g + 7.  Rows without an adapter copy aux (or store zero).
// ----------------------------------------------------------------------------
template <typename T, int RT, int CT>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs a) {
  extern __shared__ float u[];  // [16 * RT][upad]
  const LoraBlock b = lora_block(a, blockIdx.x, 16 * RT);
  if (b.adapter < 0 && a.aux == a.y)
    return;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, i = lane & 15, g = lane >> 4;
  const int rtiles = (b.rank + 15) >> 4, upad = a.rpad + 4;
  if (b.adapter >= 0) {
    const float scale = a.scales ? a.scales[b.adapter] : 1.0f;
    for (int o = tid; o < 16 * RT * rtiles * 16; o += 256) {
      const int row = o / (rtiles * 16), j = o - row * (rtiles * 16);
      float s = 0.0f;
      if (row < b.rows && j < b.rank) {
        const float* p = a.part + (size_t)(b.row + row) * a.rpad + j;
        for (int sl = 0; sl < a.slices; ++sl)
          s += p[(size_t)sl * a.m * a.rpad];
        s *= scale;
      }
      u[row * upad + j] = s;
    }
    __syncthreads();
  }
  const _Float16* w = a.b + (size_t)max(b.adapter, 0) * a.n * a.r;
  typedef T t8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int n0 = ((int)blockIdx.y * CT + ct) * 128 + 32 * wave;
    if (n0 >= a.n)
      continue;
    const int nl = n0 + 8 * g;  // the lane's 8 columns
    f4_t acc[2][RT];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int t = 0; t < RT; ++t)
        acc[p][t] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    for (int jt = 0; jt < rtiles; ++jt) {
      const int j = 16 * jt + 4 * g;
      float bv[2][4];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int n = n0 + 8 * (i >> 2) + 4 * p + (i & 3);
        const _Float16* src = w + (size_t)n * a.r + j;
        if (n < a.n && j + 4 <= a.r) {
          const h4_t v = *reinterpret_cast<const h4_any_t*>(src);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            bv[p][e] = j + e < b.rank ? (float)v[e] : 0.0f;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            bv[p][e] = n < a.n && j + e < b.rank ? (float)src[e] : 0.0f;
        }
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const f4_t uv = *reinterpret_cast<const f4_t*>(&u[(16 * t + i) * upad + j]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int p = 0; p < 2; ++p)
            acc[p][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[p][e], uv[e], acc[p][t], 0, 0, 0);
      }
    }
    if (nl >= a.n)
      continue;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if (16 * t + i >= b.rows)
        continue;
      const size_t at = (size_t)(b.row + 16 * t + i) * a.n + nl;
      float o[8];
#pragma unroll
      for (int c = 0; c < 8; ++c)
        o[c] = acc[c >> 2][t][c & 3];
      if (a.aux) {
        float x[8];
        load8(static_cast<const T*>(a.aux) + at, x);
#pragma unroll
        for (int c = 0; c < 8; ++c)
          o[c] = b.adapter < 0 ? x[c] : x[c] + o[c];
      }
      t8 y;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        y[c] = (T)o[c];
      *reinterpret_cast<t8*>(static_cast<T*>(a.y) + at) = y;
    }
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

template <typename T>
hipError_t lora_shrink(hipStream_t s, const LoraArgs& a) {
  const int tiles = lora_tiles(a, 16), rt = (a.r + 15) / 16;
  if (rt == 1)
    return dispatch(lora_shrink_kernel<T, 1>, dim3(tiles, a.slices, 1), dim3(512), s, a);
  if (rt == 2)
    return dispatch(lora_shrink_kernel<T, 2>, dim3(tiles, a.slices, 1), dim3(512), s, a);
  return dispatch(lora_shrink_kernel<T, 4>, dim3(tiles, a.slices, (rt + 3) / 4), dim3(512), s, a);
}

template <typename T>
hipError_t lora_expand(hipStream_t s, const LoraArgs& a) {
  const int upad = a.rpad + 4;
  // Four row tiles share a load of B where the rows of a sequence fill them.
  if (a.m >= 64 * a.nq && (size_t)64 * upad * sizeof(float) <= 65536)
    return dispatch_lds(lora_expand_kernel<T, 4, 1>, dim3(lora_tiles(a, 64), (a.n + 127) / 128), dim3(256), 64 * upad * sizeof(float), s, a);
  return dispatch_lds(lora_expand_kernel<T, 1, 2>, dim3(lora_tiles(a, 16), (a.n + 255) / 256), dim3(256), 16 * upad * sizeof(float), s, a);
}

}  // namespace

int lora_slices(const LoraArgs& a, int cus) {
  // Two workgroups per CU, each at least one block of 256 k.
  const int tiles = lora_tiles(a, 16), nb = a.k / 256;
  const int want = (2 * cus + tiles - 1) / tiles;
  return want < 1 ? 1 : want > nb ? nb : want > 16 ? 16 : want;
}

hipError_t launch_lora_shrink(hipStream_t s, const LoraArgs& a, int dtype) {
  return dtype == kF32 ? lora_shrink<float>(s, a) : lora_shrink<_Float16>(s, a);
}

hipError_t launch_lora_expand(hipStream_t s, const LoraArgs& a, int dtype) {
  return dtype == kF32 ? lora_expand<float>(s, a) : lora_expand<_Float16>(s, a);
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
