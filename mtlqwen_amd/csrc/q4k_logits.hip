// Penalties for repeated tokens, biases and grammar masks on rows of logits:
// logits_kernel.
#include "q4k_device.h"

namespace q4k {
namespace {

// ----------------------------------------------------------------------------
// Row r, token v: seen = v among tokens [0, lengths[r]) of the row's text,
// c = its occurrences in [prompts[r], lengths[r]):
//   l1 = seen ? (l > 0 ? l / repetition : l * repetition) : l
//   l2 = c > 0 ? l1 - frequency c - presence : l1
//   l3 = l2 + the row's last bias entry for v (if any)
//   out = masked ? -inf : l3
//
// One read and one write of the row, bound by memory.  A workgroup owns
// T * E consecutive tokens, held in registers while it counts, in LDS, those of
// the row's text that fall into its range (a word per token: bit 31 = seen in
// the prompt, the low bits = c): integer counts, so the order of the atomics
// does not matter, and no count of the whole vocabulary is cleared, written or
// read.  The text is read once per workgroup, from the L2 after the first.
// ----------------------------------------------------------------------------
typedef int32_t i4_any_t __attribute__((ext_vector_type(4), aligned(4)));

template <int N>
__device__ __forceinline__ void clear_words(uint32_t* p, int tid, int threads) {
  for (int i = tid * 4; i < N; i += threads * 4)
    *reinterpret_cast<u4_t*>(p + i) = u4_t{0u, 0u, 0u, 0u};
}

template <typename T, int THREADS, int E>
__global__ __launch_bounds__(THREADS) void logits_kernel(LogitsArgs a) {
  constexpr int V = 16 / (int)sizeof(T), N = E / V, C = THREADS * E;
  typedef T vec_t __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  __shared__ uint32_t word[C];
  const int tid = threadIdx.x;
  const uint32_t row = blockIdx.y, base = blockIdx.x * (uint32_t)C;
  const T* in = static_cast<const T*>(a.in) + (int64_t)row * a.in_stride + base;
  T* out = static_cast<T*>(a.out) + (int64_t)row * a.out_stride + base;
  const uint32_t left = a.vocab - base;  // tokens from base to the row's end

  float v[N][V];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t at = (uint32_t)(j * THREADS + tid) * V;
    if (at + V <= left) {
      const vec_t x = *reinterpret_cast<const vec_t*>(in + at);
#pragma unroll
      for (int i = 0; i < V; ++i)
        v[j][i] = (float)x[i];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        v[j][i] = at + i < left ? (float)in[at + i] : 0.0f;
    }
  }

  // The row's text, clamped to the buffer: a slot or length outside it has none.
  int length = 0, prompt = 0;
  const int32_t* text = nullptr;
  if (a.tokens) {
    const int slot = a.slots ? a.slots[row] : (int)row;
    if (slot >= 0 && (uint32_t)slot < a.nslots) {
      text = a.tokens + (size_t)slot * a.capacity;
      length = min(max(a.lengths[row], 0), (int)a.capacity);
      prompt = a.prompts ? max(a.prompts[row], 0) : 0;
    }
  }
  if (length > 0) {
    clear_words<C>(word, tid, THREADS);
    __syncthreads();
    for (int i = tid * 4; i < length; i += THREADS * 4) {
      int32_t t[4];
      if (i + 4 <= length) {
        const i4_any_t x = *reinterpret_cast<const i4_any_t*>(text + i);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          t[e] = x[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          t[e] = i + e < length ? text[i + e] : -1;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t at = (uint32_t)t[e] - base;
        if (t[e] >= 0 && (uint32_t)t[e] < a.vocab && at < (uint32_t)C) {
          if (i + e >= prompt)
            atomicAdd(&word[at], 1u);
          else
            atomicOr(&word[at], 0x80000000u);
        }
      }
    }
    __syncthreads();
    const float rep = a.repetition ? a.repetition[row] : 1.0f;
    const float freq = a.frequency ? a.frequency[row] : 0.0f, pres = a.presence ? a.presence[row] : 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint32_t w = word[(j * THREADS + tid) * V + i], c = w & 0x7fffffffu;
        if (w && a.repetition)
          v[j][i] = v[j][i] > 0.0f ? v[j][i] / rep : v[j][i] * rep;
        if (c)
          v[j][i] = v[j][i] - freq * (float)c - pres;
      }
  }

  // The row's biases: of several entries for a token the last one counts.
  if (a.bias_offsets) {
    const int lo = min(max(a.bias_offsets[row], 0), (int)a.nbias), hi = min(max(a.bias_offsets[row + 1], 0), (int)a.nbias);
    if (lo < hi) {
      __syncthreads();
      clear_words<C>(word, tid, THREADS);
      __syncthreads();
      for (int i = lo + tid; i < hi; i += THREADS) {
        const int32_t t = a.bias_tokens[i];
        const uint32_t at = (uint32_t)t - base;
        if (t >= 0 && (uint32_t)t < a.vocab && at < (uint32_t)C)
          atomicMax(&word[at], (uint32_t)(i - lo) + 1u);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < N; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const uint32_t w = word[(j * THREADS + tid) * V + i];
          if (w)
            v[j][i] += a.bias_values[lo + (int)w - 1];
        }
    }
  }

  const int mrow = a.mask ? (a.mask_rows ? a.mask_rows[row] : (int)row) : -1;
  const bool masked = mrow >= 0 && (uint32_t)mrow < a.nmasks;
  const uint32_t* mask = masked ? a.mask + (size_t)mrow * a.mask_stride + (base >> 5) : nullptr;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t at = (uint32_t)(j * THREADS + tid) * V;
    if (at >= left)
      continue;
    const uint32_t allowed = masked ? mask[at >> 5] >> (at & 31u) : 0xffffffffu;
    vec_t y;
#pragma unroll
    for (int i = 0; i < V; ++i)
      y[i] = (T)((allowed >> i) & 1u ? v[j][i] : -__builtin_inff());
    if (at + V <= left) {
      *reinterpret_cast<vec_t*>(out + at) = y;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (at + i < left)
          out[at + i] = y[i];
    }
  }
}

template <typename T, int THREADS, int E>
hipError_t logits_dispatch(hipStream_t s, const LogitsArgs& a) {
  const uint32_t c = THREADS * E;
  return dispatch(logits_kernel<T, THREADS, E>, dim3((a.vocab + c - 1) / c, a.rows), dim3(THREADS), s, a);
}

template <typename T>
hipError_t logits_launch(hipStream_t s, const LogitsArgs& a, int cus) {
  // Large ranges read the text fewer times; small ones fill the card.
  if ((uint64_t)a.rows * a.vocab >= (uint64_t)cus * 2 * 16384)
    return logits_dispatch<T, 1024, 16>(s, a);
  return logits_dispatch<T, 256, 8>(s, a);
}

}  // namespace

hipError_t launch_logits(hipStream_t s, const LogitsArgs& a, int dtype, int cus) {
  return dtype == kF32 ? logits_launch<float>(s, a, cus) : logits_launch<_Float16>(s, a, cus);
}

}  // namespace q4k
