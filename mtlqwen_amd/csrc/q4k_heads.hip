// Rotary positions of attention heads, alone or after the RMS norm of each
// query and key head: heads_kernel.
//
// Both read and write every value once, so they are bound by memory; what
// decides is that a row's angles are made once for many heads.
#include "q4k_device.h"

namespace q4k {
namespace {

// ----------------------------------------------------------------------------
// One head of `dim` values x, position p, h = rot / 2, pair i < h turned by
// p f_i (f = inv_freq): with c = scale cos(p f_i) and n = scale sin(p f_i),
//   half layout (INTER = 0):   y[i] = x[i] c - x[i + h] n, y[i + h] = x[i + h] c + x[i] n
//   interleaved (INTER = 1):   the same of x[2i] and x[2i + 1]
// and y[d] = x[d] for d >= rot.  NORM: x is x * w / sqrt(sum(x^2) / dim + eps)
// first, in fp32, without a rounding in between.
//
// A lane holds two vectors of V values (a "slot"): of the rotated part the two
// that turn into each other, behind it two neighbours; glog = log2 of the lanes
// of a head, so that a wave reduces the sums of squares of its heads without
// LDS.  P slots per lane cover heads that 64 lanes of one slot do not.
//
// A workgroup takes U rows per lane and every gridDim.y-th group of hb heads of
// them: its angles are made once, in LDS, for all those heads, and the values of
// the next group are asked for before the present one's are used.
// Angles are 64-bit products of the position and the frequency in turns: at
// position 2^20 a product in 32 bits would be off by 0.06 rad, at any position
// below 2^31 this one is by 5e-7.  The fraction enters the function in 32 bits, and
// what that rounding left, d rad, as c - n d and n + c d (d^2 < 1e-14): without it
// (9.4e-8 rad) a value near zero would keep few of its bits.
// ----------------------------------------------------------------------------
template <typename T, int V>
struct VecOf {
  typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  static __device__ __forceinline__ float get(const type& v, int i) { return (float)v[i]; }
  static __device__ __forceinline__ void set(type& v, int i, float x) { v[i] = (T)x; }
};
template <typename T>
struct VecOf<T, 1> {
  typedef T type;
  static __device__ __forceinline__ float get(const type& v, int) { return (float)v; }
  static __device__ __forceinline__ void set(type& v, int, float x) { v = (T)x; }
};

// The calls that fill the card (two rows per lane) write past the caches: what they
// write outgrows them.  Replayed back to back, through the caches -> past them: norm
// and rotation of 8192 rows of 40 heads of 128, fp16, 38.2 -> 33.9 us, 4.95 TB/s
// (2048 rows 10.2 -> 9.0); rotation alone, fp32, 66.9 -> 63.9 us, 5.25 TB/s, where a
// copy of 1 GiB reaches 5.05.
template <int U, typename V>
__device__ __forceinline__ void put(V* p, V v) {
  if constexpr (U > 1)
    __builtin_nontemporal_store(v, p);
  else
    *p = v;
}

template <typename T, int V, int P, int U, bool NORM, bool INTER>
__global__ __launch_bounds__(256) void heads_kernel(HeadsArgs a) {
  extern __shared__ float cs[];  // [rows of the workgroup][2][h]: cosines, sines
  typedef VecOf<T, V> vec;
  typedef typename vec::type vec_t;
  const int tid = threadIdx.x, lane = tid & ((1 << a.glog) - 1), slot = tid >> a.glog;
  const int hb = 1 << a.hblog, rb = 256 >> (a.glog + a.hblog);
  const uint32_t row0 = blockIdx.x * (uint32_t)(rb * U) + (uint32_t)(slot >> a.hblog);
  const int h = a.rot >> 1, nslots = a.nslots, rslots = INTER ? 0 : h / V;
  const uint32_t heads = a.heads[0] + a.heads[1], hstep = gridDim.y * (uint32_t)hb;

  int o1[P], o2[P];
  bool on1[P], on2[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int j = lane + (p << a.glog);
    o1[p] = INTER ? 2 * V * j : j < rslots ? V * j : a.rot + 2 * V * (j - rslots);
    o2[p] = !INTER && j < rslots ? o1[p] + h : o1[p] + V;
    on1[p] = j < nslots && o1[p] < a.dim;
    on2[p] = on1[p] && o2[p] < a.dim;
  }

  vec_t r1[U][P], r2[U][P];
  const auto load = [&](uint32_t head) {
    const bool key = head >= a.heads[0];
    const T* in = static_cast<const T*>(key ? a.in[1] : a.in[0]) + (int64_t)(key ? head - a.heads[0] : head) * (key ? a.head_in[1] : a.head_in[0]);
    const int64_t row_in = key ? a.row_in[1] : a.row_in[0];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t row = row0 + (uint32_t)(u * rb);
      const T* x = in + (int64_t)row * row_in;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        if (head < heads && row < a.rows && on1[p])
          r1[u][p] = *reinterpret_cast<const vec_t*>(x + o1[p]);
        if (head < heads && row < a.rows && on2[p])
          r2[u][p] = *reinterpret_cast<const vec_t*>(x + o2[p]);
      }
    }
  };
  uint32_t head = blockIdx.y * (uint32_t)hb + (uint32_t)(slot & (hb - 1));
  load(head);

  // The angles of the workgroup's rows.
  for (int i = tid; i < rb * U * h; i += 256) {
    const int r = i / h, f = i - r * h;
    const uint32_t row = blockIdx.x * (uint32_t)(rb * U) + (uint32_t)r;
    if (row < a.rows) {
      const double turns = (double)a.positions[row] * (a.inv_freq[f] * 0.15915494309189533577);
      const double part = turns - rint(turns);
      const float near = (float)part, d = 6.2831853f * (float)(part - (double)near);
      float s, c;
      sincospif(2.0f * near, &s, &c);
      cs[(2 * r) * h + f] = a.scale * fmaf(-s, d, c);
      cs[(2 * r + 1) * h + f] = a.scale * fmaf(c, d, s);
    }
  }
  __syncthreads();

  float w1[NORM ? P : 1][V], w2[NORM ? P : 1][V];
  int weights = -1;
  for (uint32_t first = blockIdx.y * (uint32_t)hb; first < heads; first += hstep) {
    const bool key = head >= a.heads[0], live = head < heads;
    T* out = static_cast<T*>(key ? a.out[1] : a.out[0]) + (int64_t)(key ? head - a.heads[0] : head) * (key ? a.head_out[1] : a.head_out[0]);
    const int64_t row_out = key ? a.row_out[1] : a.row_out[0];
    if constexpr (NORM) {
      if (weights != (int)key) {
        weights = (int)key;
        typedef VecOf<float, V> fvec;
        const float* w = key ? a.w[1] : a.w[0];
#pragma unroll
        for (int p = 0; p < P; ++p) {
          if (live && on1[p]) {
            const typename fvec::type t = *reinterpret_cast<const typename fvec::type*>(w + o1[p]);
#pragma unroll
            for (int i = 0; i < V; ++i)
              w1[p][i] = fvec::get(t, i);
          }
          if (live && on2[p]) {
            const typename fvec::type t = *reinterpret_cast<const typename fvec::type*>(w + o2[p]);
#pragma unroll
            for (int i = 0; i < V; ++i)
              w2[p][i] = fvec::get(t, i);
          }
        }
      }
    }
    float v1[U][P][V], v2[U][P][V];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v1[u][p][i] = on1[p] ? vec::get(r1[u][p], i) : 0.0f;
          v2[u][p][i] = on2[p] ? vec::get(r2[u][p], i) : 0.0f;
        }
    head += hstep;
    if (first + hstep < heads)
      load(head);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t row = row0 + (uint32_t)(u * rb);
      if constexpr (NORM) {
        float ss = 0.0f;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int i = 0; i < V; ++i)
            ss = fmaf(v1[u][p][i], v1[u][p][i], fmaf(v2[u][p][i], v2[u][p][i], ss));
        for (int off = (1 << a.glog) >> 1; off > 0; off >>= 1)
          ss += __shfl_xor(ss, off);
        const float r = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            v1[u][p][i] = v1[u][p][i] * r * w1[p][i];
            v2[u][p][i] = v2[u][p][i] * r * w2[p][i];
          }
      }
      if (row >= a.rows || !live)
        continue;
      const float* ct = cs + 2 * ((slot >> a.hblog) + u * rb) * h;
      const float* st = ct + h;
      T* y = out + (int64_t)row * row_out;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        if (on1[p] && o1[p] < a.rot) {
          if constexpr (!INTER || V == 1) {
            const int f = INTER ? o1[p] >> 1 : o1[p];
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float c = ct[f + i], n = st[f + i], x1 = v1[u][p][i], x2 = v2[u][p][i];
              v1[u][p][i] = x1 * c - x2 * n;
              v2[u][p][i] = x2 * c + x1 * n;
            }
          } else {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
              const float c = ct[(o1[p] + i) >> 1], n = st[(o1[p] + i) >> 1], x1 = v1[u][p][i], x2 = v1[u][p][i + 1];
              v1[u][p][i] = x1 * c - x2 * n;
              v1[u][p][i + 1] = x2 * c + x1 * n;
            }
            if (o2[p] < a.rot) {
#pragma unroll
              for (int i = 0; i < V; i += 2) {
                const float c = ct[(o2[p] + i) >> 1], n = st[(o2[p] + i) >> 1], x1 = v2[u][p][i], x2 = v2[u][p][i + 1];
                v2[u][p][i] = x1 * c - x2 * n;
                v2[u][p][i + 1] = x2 * c + x1 * n;
              }
            }
          }
        }
        vec_t y1, y2;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          vec::set(y1, i, v1[u][p][i]);
          vec::set(y2, i, v2[u][p][i]);
        }
        if (on1[p])
          put<U>(reinterpret_cast<vec_t*>(y + o1[p]), y1);
        if (on2[p])
          put<U>(reinterpret_cast<vec_t*>(y + o2[p]), y2);
      }
    }
  }
}

// The widest vector that a head's layout allows: chunks of V values must not
// straddle the halves (or the end) of the rotated part, nor the head's end.
int heads_vec(int dim, int rot, bool inter, int widest) {
  for (int v = widest; v > 1; v >>= 1)
    if (dim % v == 0 && (inter ? rot : rot / 2) % v == 0)
      return v;
  return 1;
}

template <typename T, bool NORM, bool INTER>
hipError_t heads_launch(hipStream_t s, HeadsArgs a, int cus) {
  constexpr int kWide = 16 / (int)sizeof(T);
  constexpr uint32_t kDeep = 2;
  int v = heads_vec(a.dim, a.rot, INTER, kWide);
  auto slots_of = [&](int vec) {
    const int turned = INTER ? 0 : a.rot / (2 * vec), rest = INTER ? a.dim : a.dim - a.rot;
    return turned + (rest + 2 * vec - 1) / (2 * vec);
  };
  if (v != kWide || slots_of(v) > 64)
    v = v >= 2 ? 2 : 1;
  a.nslots = slots_of(v);
  const uint32_t heads = a.heads[0] + a.heads[1];
  a.glog = 0;
  while ((1 << a.glog) < a.nslots && a.glog < 6)
    ++a.glog;
  // Heads side by side: as many as a workgroup holds and the heads fill to an
  // eighth, so that few lanes idle.
  a.hblog = 8 - a.glog;
  while (a.hblog > 0 && ((heads + (1u << a.hblog) - 1) >> a.hblog << a.hblog) - heads > heads / 8)
    --a.hblog;
  const uint32_t rb = 256u >> (a.glog + a.hblog), groups = (heads + (1u << a.hblog) - 1) >> a.hblog;
  // Two rows per lane, and as many head groups per workgroup, as leave every CU
  // four workgroups.  Replayed, with norms, fp16, stores through the caches: 821
  // rows of 20 heads of 256 5.8 us, with two 6.6, with eight 5.8; 8192 rows of 40
  // heads of 128 38.2 us, with two 38.2, with eight 40.7, and 38.1 with one row per
  // lane, whose stores stay in the caches.  Heads that 16 bytes do not divide take
  // four- and two-byte accesses and one row: 8192 fp16 rows of 40 heads of 80 with 40
  // rotated 65 us, with 80 rotated (16 bytes) 23.
  const uint64_t want = 4ull * (uint32_t)cus;
  const bool deep = v == kWide && (uint64_t)((a.rows + kDeep * rb - 1) / (kDeep * rb)) * groups >= want &&
                    (size_t)rb * kDeep * a.rot * sizeof(float) <= 32768;
  const uint32_t rows = rb * (deep ? kDeep : 1u), blocks = (a.rows + rows - 1) / rows;
  const uint64_t split = (want + blocks - 1) / blocks;
  const dim3 grid(blocks, split < groups ? (uint32_t)split : groups), block(256);
  const size_t lds = (size_t)rows * a.rot * sizeof(float);
  if (v == kWide && deep)
    return dispatch_lds(heads_kernel<T, kWide, 1, kDeep, NORM, INTER>, grid, block, lds, s, a);
  if (v == kWide)
    return dispatch_lds(heads_kernel<T, kWide, 1, 1, NORM, INTER>, grid, block, lds, s, a);
  if (v == 2)
    return dispatch_lds(heads_kernel<T, 2, 4, 1, NORM, INTER>, grid, block, lds, s, a);
  return dispatch_lds(heads_kernel<T, 1, 8, 1, NORM, INTER>, grid, block, lds, s, a);
}

template <typename T>
hipError_t heads_launch_t(hipStream_t s, const HeadsArgs& a, bool norm, bool inter, int cus) {
  if (norm)
    return inter ? heads_launch<T, true, true>(s, a, cus) : heads_launch<T, true, false>(s, a, cus);
  return inter ? heads_launch<T, false, true>(s, a, cus) : heads_launch<T, false, false>(s, a, cus);
}

}  // namespace

hipError_t launch_heads(hipStream_t s, const HeadsArgs& a, bool norm, bool inter, int dtype, int cus) {
  return dtype == kF32 ? heads_launch_t<float>(s, a, norm, inter, cus) : heads_launch_t<_Float16>(s, a, norm, inter, cus);
}

}  // namespace q4k
