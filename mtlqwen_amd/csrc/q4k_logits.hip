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
// One read and one write of the row, bound by memory: 64 rows of 248320 fp32 take,
// replayed, 19.3 us with nothing else to do (6.6 TB/s, the inputs in the memory-side
// cache), 36.1 with texts of 32768 to 65536 tokens, 300 biases and masks, whose
// counting overlaps the copy in part.  A workgroup owns THREADS * E consecutive
// tokens, held in registers while it counts, in LDS, those of the row's text and
// biases that fall into its range.  One word per token: bit 31 = seen in the
// prompt; below it 31 - s bits with the number of the last bias entry (0: none);
// s low bits with c, s enough for the token buffer's capacity.  Integer counts
// and maxima, so the order of the atomics does not matter, and no count of the
// whole vocabulary is cleared, written or read.  A row of more biases than fit
// into 31 - s bits takes a second round through the words.  Workgroups of every
// other round of the CUs read their logits after the text, so that not all of
// them leave the memory idle while they count (the case above 36.6 -> 36.0 us, and
// 46.7 -> 44.6 with stores through the caches).  The text is read once per workgroup; the workgroups
// of a row sit a multiple of the row count apart, with 8 rows and their multiples
// on one XCD, whose L2 then serves every reading after the first.
// ----------------------------------------------------------------------------
typedef int32_t i4_any_t __attribute__((ext_vector_type(4), aligned(4)));

template <int N>
__device__ __forceinline__ void clear_words(uint32_t* p, int tid, int threads) {
  for (int i = tid * 4; i < N; i += threads * 4)
    *reinterpret_cast<u4_t*>(p + i) = u4_t{0u, 0u, 0u, 0u};
}

// The words of tokens text[lo, hi) that lie within `range` of `base`: the high
// bit set (SEEN), or one added.  K loads of four tokens in flight per thread;
// negative and foreign tokens lie past every range.
template <int THREADS, bool SEEN>
__device__ __forceinline__ void count_tokens(const int32_t* text, int lo, int hi, uint32_t base, uint32_t range, uint32_t spare,
                                             uint32_t* word, int tid) {
  constexpr int K = 4;
  for (int i0 = lo + tid * 4; i0 < hi; i0 += THREADS * 4 * K) {
    int32_t t[K][4];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = i0 + k * THREADS * 4;
      if (i + 4 <= hi) {
        const i4_any_t x = *reinterpret_cast<const i4_any_t*>(text + i);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          t[k][e] = x[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          t[k][e] = i + e < hi ? text[i + e] : -1;
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t at = (uint32_t)t[k][e] - base, to = at < range ? at : spare;
        if (SEEN)
          atomicOr(&word[to], 0x80000000u);
        else
          atomicAdd(&word[to], 1u);
      }
  }
}

template <typename T, int THREADS, int E>
__global__ __launch_bounds__(THREADS) void logits_kernel(LogitsArgs a) {
  constexpr int V = 16 / (int)sizeof(T), N = E / V, C = THREADS * E;
  typedef T vec_t __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  __shared__ uint32_t word[C + 64];
  const int tid = threadIdx.x;
  const uint32_t row = blockIdx.x, base = blockIdx.y * (uint32_t)C;
  const T* in = static_cast<const T*>(a.in) + (int64_t)row * a.in_stride + base;
  T* out = static_cast<T*>(a.out) + (int64_t)row * a.out_stride + base;
  const uint32_t left = a.vocab - base;  // tokens from base to the row's end
  const uint32_t range = left < (uint32_t)C ? left : (uint32_t)C, spare = C + (tid & 63);

  float v[N][V];
  auto load = [&]() {
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
  };
  const bool late = ((blockIdx.x + gridDim.x * blockIdx.y) / a.stagger) & 1u;
  if (!late)
    load();
  // What the row asks for: its text, clamped to the buffer (a slot or length
  // outside it has none), its biases and its mask.
  int length = 0, prompt = 0;
  const int32_t* text = nullptr;
  if (a.tokens) {
    const int slot = a.slots ? a.slots[row] : (int)row, len = a.lengths[row], given = a.prompts ? a.prompts[row] : 0;
    if (slot >= 0 && (uint32_t)slot < a.nslots) {
      text = a.tokens + (size_t)slot * a.capacity;
      length = min(max(len, 0), (int)a.capacity);
      prompt = min(max(given, 0), length);
    }
  }
  int lo = 0, nbias = 0;
  if (a.bias_offsets) {
    lo = min(max(a.bias_offsets[row], 0), (int)a.nbias);
    nbias = max(min(a.bias_offsets[row + 1], (int)a.nbias) - lo, 0);
  }
  const int mrow = a.mask ? (a.mask_rows ? a.mask_rows[row] : (int)row) : -1;
  const bool masked = mrow >= 0 && (uint32_t)mrow < a.nmasks;

  // Bit i of a word: the vector's value i is allowed.
  const uint32_t* mask = a.mask + (masked ? (size_t)mrow * a.mask_stride + (base >> 5) : 0);
  uint32_t allowed[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t at = (uint32_t)(j * THREADS + tid) * V;
    allowed[j] = masked && at < left ? mask[at >> 5] >> (at & 31u) : 0xffffffffu;
  }

  if (late && length <= 0 && nbias <= 0)
    load();
  if (length > 0 || nbias > 0) {
    const uint32_t bits = a.count_bits, biases = 0x7fffffffu >> bits;
    const bool packed = (uint32_t)nbias <= biases;
    clear_words<C>(word, tid, THREADS);
    __syncthreads();
    if (packed && nbias > 0) {
      for (int i = tid; i < nbias; i += THREADS) {
        const uint32_t at = (uint32_t)a.bias_tokens[lo + i] - base;
        if (at < range)
          atomicMax(&word[at], (uint32_t)(i + 1) << bits);
      }
      __syncthreads();
    }
    if (a.repetition)
      count_tokens<THREADS, true>(text, 0, prompt, base, range, spare, word, tid);
    count_tokens<THREADS, false>(text, prompt, length, base, range, spare, word, tid);
    if (late)
      load();
    __syncthreads();
    const float rep = a.repetition ? a.repetition[row] : 1.0f;
    const float freq = a.frequency ? a.frequency[row] : 0.0f, pres = a.presence ? a.presence[row] : 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint32_t w = word[(j * THREADS + tid) * V + i];
        if (w == 0)
          continue;
        const uint32_t c = w & ((1u << bits) - 1u), b = (w & 0x7fffffffu) >> bits;
        float x = v[j][i];
        if (a.repetition && (c || (w >> 31)))
          x = x > 0.0f ? x / rep : x * rep;
        if (c)
          x = x - freq * (float)c - pres;
        if (b)
          x += a.bias_values[lo + (int)b - 1];
        v[j][i] = x;
      }
    if (!packed) {
      __syncthreads();
      clear_words<C>(word, tid, THREADS);
      __syncthreads();
      for (int i = tid; i < nbias; i += THREADS) {
        const uint32_t at = (uint32_t)a.bias_tokens[lo + i] - base;
        if (at < range)
          atomicMax(&word[at], (uint32_t)i + 1u);
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

#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t at = (uint32_t)(j * THREADS + tid) * V;
    if (at >= left)
      continue;
    vec_t y;
#pragma unroll
    for (int i = 0; i < V; ++i)
      y[i] = (T)((allowed[j] >> i) & 1u ? v[j][i] : -__builtin_inff());
    if (at + V <= left) {
      if constexpr (THREADS > 512)  // past the caches, which such outputs outgrow: 44.6 -> 36.1 us
        __builtin_nontemporal_store(y, reinterpret_cast<vec_t*>(out + at));
      else
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
  return dispatch(logits_kernel<T, THREADS, E>, dim3(a.rows, (a.vocab + c - 1) / c), dim3(THREADS), s, a);
}

template <typename T>
hipError_t logits_launch(hipStream_t s, const LogitsArgs& a, int cus) {
  // Large ranges read the text fewer times, small ones fill the card: 4096 tokens
  // to a workgroup, or 16384 once every CU has one of those, or half of them where
  // texts may be long.  Replayed, fp32, 248320 tokens, texts up to 65536 / 4000: 1 row
  // 9.0 / 5.9 us (16384: 11.3 / 8.5), 8 rows 13.0 / 7.5 (11.9 / 9.0), 16 rows 19.8 /
  // 11.5 (13.7 / 11.1), 32 rows 32.1 / 17.7 (18.8 / 13.3).
  const uint64_t logits = (uint64_t)a.rows * a.vocab, fill = (uint64_t)cus * 16384;
  if (logits >= fill || (a.tokens && a.capacity > 32768 && logits >= fill / 2))
    return logits_dispatch<T, 1024, 16>(s, a);
  return logits_dispatch<T, 512, 8>(s, a);
}

}  // namespace

hipError_t launch_logits(hipStream_t s, LogitsArgs a, int dtype, int cus) {
  a.stagger = (uint32_t)cus;
  a.count_bits = 1;
  while (a.count_bits < 31 && (a.capacity >> a.count_bits) != 0)
    ++a.count_bits;
  return dtype == kF32 ? logits_launch<float>(s, a, cus) : logits_launch<_Float16>(s, a, cus);
}

}  // namespace q4k
