// Attention of a packed batch's new tokens over a paged key/value cache.
#include "q4k_device.h"

namespace q4k {
namespace {

// One row and head: x_j = scale q.k_j, capped and biased, over the keys that the
// row sees, o = sum_j exp(x_j) v_j / sum_j exp(x_j), in one pass over the keys with
// the running maximum and sum.
template <typename T>
__global__ __launch_bounds__(256) void attention_kernel(AttentionArgs a) {
  __shared__ float so[4][256], sm[4], sl[4];
  const CacheArgs& c = a.cache;
  const int row = blockIdx.x, head = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int q = 0;
  while (q + 1 < c.nq && row >= c.start[q + 1])
    ++q;
  const int64_t pos = (int64_t)c.positions[q] + (row - c.start[q]);
  const int slot = c.slots ? c.slots[q] : q;
  const int64_t cap = (uint32_t)slot < (uint32_t)c.table_rows ? (int64_t)c.width << c.page_log : 0;
  const int64_t hi = pos + 1 < cap ? pos + 1 : cap, lo = a.window && pos + 1 > a.window ? pos + 1 - a.window : 0;
  const int kvh = head / a.group;
  float x[4], o[4] = {};
  for (int i = 0; i < 4; ++i)
    x[i] = lane + 64 * i < c.dim ? (float)(static_cast<const T*>(a.q) + (int64_t)row * a.q_row + (int64_t)head * a.q_head)[lane + 64 * i] : 0.0f;
  float m = -INFINITY, l = 0.0f;
  for (int64_t j = lo + wave; j < hi; j += 4) {
    const int32_t page = c.tables[(int64_t)slot * c.width + (j >> c.page_log)];
    if ((uint32_t)page >= c.pages)
      continue;
    const int64_t at = (int64_t)page * c.page_stride + (int64_t)kvh * c.head_stride + (j & ((1 << c.page_log) - 1)) * c.token_stride;
    float s = 0.0f;
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < c.dim)
        s = fmaf(x[i], (float)static_cast<const _Float16*>(c.k)[at + lane + 64 * i], s);
    for (int off = 32; off; off >>= 1)
      s += __shfl_xor(s, off);
    s *= a.scale;
    if (a.softcap > 0.0f)
      s = a.softcap * tanhf(s / a.softcap);
    if (a.slopes)
      s = fmaf(a.slopes[head], (float)(j - pos), s);
    // fmaxf leaves a NaN out; the weight, and with it the sums, takes it up.
    const float n = fmaxf(m, s), top = n == -INFINITY ? 0.0f : n, r = m == n ? 1.0f : expf(m - n), p = expf(s - top);
    l = l * r + p;
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < c.dim)
        o[i] = fmaf(p, (float)static_cast<const _Float16*>(c.v)[at + lane + 64 * i], o[i] * r);
    m = n;
  }
  for (int i = 0; i < 4; ++i)
    so[wave][lane + 64 * i] = o[i];
  sm[wave] = m;
  sl[wave] = l;
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= c.dim)
    return;
  const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float sum = 0.0f, y = 0.0f;
  for (int w = 0; w < 4; ++w) {
    const float f = sm[w] == top ? 1.0f : expf(sm[w] - top);
    sum += f * sl[w];
    y += f * so[w][d];
  }
  (static_cast<T*>(a.out) + (int64_t)row * a.out_row + (int64_t)head * a.out_head)[d] = (T)(sum == 0.0f ? 0.0f : y / sum);
}

}  // namespace

hipError_t launch_attention(hipStream_t s, const AttentionArgs& a, int dtype, int cus) {
  const dim3 grid(a.rows, a.heads);
  return dtype == kF32 ? dispatch(attention_kernel<float>, grid, dim3(256), s, a) : dispatch(attention_kernel<_Float16>, grid, dim3(256), s, a);
}

}  // namespace q4k
