// The paged key/value cache besides the attention that reads it: keys and
// values of new tokens into their pages (cache_write_kernel), slots that take
// over the states of others (cache_assign_kernel), pages moved to the front of
// the pool (cache_compact_kernel), and the copies that the last two ask for.
#include "q4k_device.h"

namespace q4k {
namespace {

// ----------------------------------------------------------------------------
// Row t of sequence q goes to position p = positions[q] + t: token p % page_size
// of page tables[slot of q][p / page_size], rounded to fp16 (the cache's type;
// half a step, 2^-11 of the value).  A lane moves 8 values of one head; keys and
// values of a row are 2 * heads * dim / 8 lanes next to each other.  Bound by
// memory: every value is read and written once.
// ----------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void cache_write_kernel(CacheArgs c, CacheRows in, uint32_t per_row, uint32_t rows) {
  const uint32_t chunks = (uint32_t)c.dim >> 3;
  const uint64_t item = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t row = (uint32_t)(item / per_row);
  if (row >= rows)
    return;
  uint32_t at = (uint32_t)(item - (uint64_t)row * per_row);
  const bool value = at >= (per_row >> 1);
  at -= value ? per_row >> 1 : 0;
  const uint32_t head = at / chunks, d = (at - head * chunks) << 3;
  const T* x = static_cast<const T*>(value ? in.v : in.k) + (int64_t)row * (value ? in.v_row : in.k_row) + (int64_t)head * (value ? in.v_head : in.k_head) + d;
  float f[8];
  load8(x, f);
  int q = 0;
  while (q + 1 < c.nq && row >= (uint32_t)c.start[q + 1])
    ++q;
  const int64_t pos = (int64_t)c.positions[q] + (row - (uint32_t)c.start[q]);
  const int slot = c.slots ? c.slots[q] : q;
  if (pos < 0 || pos >> c.page_log >= c.width || (uint32_t)slot >= (uint32_t)c.table_rows)
    return;
  const int32_t page = c.tables[(int64_t)slot * c.width + (pos >> c.page_log)];
  if ((uint32_t)page >= c.pages)
    return;
  _Float16* y = static_cast<_Float16*>(value ? c.v : c.k) + (int64_t)page * c.page_stride + (int64_t)head * c.head_stride +
                (pos & ((1 << c.page_log) - 1)) * c.token_stride + d;
  h8_t h;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    h[i] = (_Float16)f[i];
  *reinterpret_cast<h8_t*>(y) = h;
}

// ----------------------------------------------------------------------------
// Tables.  One workgroup of 1024 threads per call: which pages are held is a
// bit per page in LDS (up to 2^18 pages, 32 KB), so nothing about the pool is
// kept between calls, and pages are found by counting bits: `rank` holds, per word,
// the pages counted before it.  What each step reads it reads with all threads at once,
// over slots and entries alike, so that narrow tables are bound by latency (64 slots of 8
// entries 6.3 us); wide ones by what one CU gets through, a division and 8 bytes an
// entry and walk: 64 slots of 512 entries 46 us assigned and 38 compacted, of 4096 entries 291 and
// 252 (2.1 MB of tables, a microsecond of the card's memory).
// ----------------------------------------------------------------------------
constexpr int kTableThreads = 1024;
constexpr int kWords = (int)kMaxPages / 32;

// Sum over the threads before this one, and over all of them.  `sums` holds 16
// words; free for the next call behind the caller's next barrier.
__device__ __forceinline__ uint32_t scan_before(uint32_t v, uint32_t* sums, uint32_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t s = v;
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t o = __shfl_up(s, off);
    s += lane >= off ? o : 0;
  }
  if (lane == 63)
    sums[wave] = s;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kTableThreads / 64; ++w) {
    const uint32_t x = sums[w];
    before += w < wave ? x : 0;
    all += x;
  }
  __syncthreads();
  *total = all;
  return before + s - v;
}

__device__ __forceinline__ bool bit_of(const uint32_t* bits, uint32_t p) {
  return (bits[p >> 5] >> (p & 31)) & 1;
}

__device__ __forceinline__ void set_bit(uint32_t* bits, uint32_t p) {
  atomicOr(&bits[p >> 5], 1u << (p & 31));
}

__device__ __forceinline__ int words_of(const TableArgs& a) {
  return (int)((a.pages + 31) >> 5);
}

// rank[w] = set bits in the words before w; their number.  Ends with a barrier.
__device__ __forceinline__ uint32_t count_bits(const uint32_t* bits, uint32_t* rank, int words, uint32_t* sums) {
  const int each = (words + kTableThreads - 1) / kTableThreads, from = threadIdx.x * each;
  uint32_t n = 0, all;
  for (int w = from; w < from + each && w < words; ++w)
    n += __popc(bits[w]);
  uint32_t before = scan_before(n, sums, &all);
  for (int w = from; w < from + each && w < words; ++w) {
    rank[w] = before;
    before += __popc(bits[w]);
  }
  __syncthreads();
  return all;
}

// Set bits before page p.
__device__ __forceinline__ uint32_t rank_of(const uint32_t* bits, const uint32_t* rank, uint32_t p) {
  return rank[p >> 5] + __popc(bits[p >> 5] & ((1u << (p & 31)) - 1));
}

// A slot's tokens: not negative, no more than its table holds.
__device__ __forceinline__ int32_t tokens_of(int32_t length, const TableArgs& a) {
  const int64_t most = (int64_t)a.width << a.page_log;
  return length < 0 ? 0 : length > most ? (int32_t)most : length;
}

// Calls f(slot, entry) for all entries of all slots, the threads side by side.
template <typename F>
__device__ __forceinline__ void each_entry(const TableArgs& a, const F& f) {
  const uint32_t all = (uint32_t)a.slots * (uint32_t)a.width;  // below 2^31: checked by the caller
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < all; i += kTableThreads) {
    const uint32_t s = i / (uint32_t)a.width;
    f((int)s, (int)(i - s * (uint32_t)a.width));
  }
}

// What a workgroup copies of a block at a time.
constexpr uint32_t kCopyBytes = 16384;

template <int THREADS = 256>
__device__ __forceinline__ void copy_bytes(const uint8_t* from, uint8_t* to, uint32_t bytes) {
  constexpr int kDeep = 4;
  u4_t v[kDeep];
  for (uint32_t at = threadIdx.x * 16; at < bytes; at += THREADS * 16 * kDeep) {
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
      if (at + i * THREADS * 16 < bytes)
        v[i] = *reinterpret_cast<const u4_t*>(from + at + i * THREADS * 16);
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
      if (at + i * THREADS * 16 < bytes)
        *reinterpret_cast<u4_t*>(to + at + i * THREADS * 16) = v[i];
  }
}

// Slot s takes the first lengths[p] tokens of its parent p.  Pages full of tokens are
// shared.  A page that is not full will be written on, so it can stay with one
// slot only: with the lowest of those that hold it, unless another holds it as a
// full page; the others get a page of their own and a copy (page_fork_kernel).
// Then, slot by slot, the lowest free pages for counts[s] more tokens.
__global__ __launch_bounds__(kTableThreads) void cache_assign_kernel(TableArgs a, PoolArgs pool) {
  __shared__ uint32_t bits[kWords], rank[kWords], sums[16], before[kMaxSlots + 1];
  __shared__ unsigned long long beyond;  // pages that tables have no entries for
  __shared__ __attribute__((aligned(16))) int32_t last[kMaxSlots];
  __shared__ int32_t parent[kMaxSlots], full[kMaxSlots], first[kMaxSlots], kept[kMaxSlots];
  const int tid = threadIdx.x, words = words_of(a);
  for (int w = tid; w < words; w += kTableThreads)
    bits[w] = 0;
  int32_t length = 0, tail = -1;
  bool part = false;
  if (tid < a.slots) {
    const int32_t p = a.parents ? a.parents[tid] : tid;
    const bool live = (uint32_t)p < (uint32_t)a.slots;
    length = live ? tokens_of(a.lengths[p], a) : 0;
    part = length & ((1 << a.page_log) - 1);
    parent[tid] = live ? p : 0;
    full[tid] = length >> a.page_log;
    a.new_lengths[tid] = length;
    if (part)
      tail = a.tables[(int64_t)p * a.width + full[tid]];
  }
  last[tid] = (uint32_t)tail < a.pages ? tail : -1;
  if (tid == 0)
    beyond = 0;
  __syncthreads();
  each_entry(a, [&](int s, int e) {
    if (e < full[s]) {
      const uint32_t p = (uint32_t)a.tables[(int64_t)parent[s] * a.width + e];
      if (p < a.pages)
        set_bit(bits, p);
    }
  });
  bool keep = last[tid] >= 0;
  const int4* lasts = reinterpret_cast<const int4*>(last);
#pragma unroll 4
  for (int s = 0; s < (a.slots + 3) / 4; ++s) {  // the slots before this one
    const int4 o = lasts[s];
    keep = keep && !((4 * s < tid && o.x == last[tid]) | (4 * s + 1 < tid && o.y == last[tid]) | (4 * s + 2 < tid && o.z == last[tid]) |
                     (4 * s + 3 < tid && o.w == last[tid]));
  }
  __syncthreads();
  keep = keep && !bit_of(bits, (uint32_t)last[tid]);
  __syncthreads();
  uint32_t wants = 0;
  if (tid < a.slots) {
    if (keep)
      set_bit(bits, (uint32_t)last[tid]);
    // A page that the parent's table lacks stays lacking.
    const int32_t from = full[tid] + (part && (keep || last[tid] < 0));
    const int32_t count = a.counts ? a.counts[tid] : 0;
    const int64_t need = ((int64_t)length + (count > 0 ? count : 0) + (1 << a.page_log) - 1) >> a.page_log;
    const int64_t most = need < a.width ? need : a.width;
    wants = most > from ? (uint32_t)(most - from) : 0;
    if (need > most)
      atomicAdd(&beyond, (unsigned long long)(need - most));
    first[tid] = from;
    kept[tid] = keep;
  }
  uint32_t asked;
  const uint32_t mine = scan_before(wants, sums, &asked);
  if (tid < a.slots)
    before[tid] = mine;
  if (tid == 0)
    before[a.slots] = asked;
  const uint32_t there = a.pages - count_bits(bits, rank, words, sums);
  if (tid == 0 && a.missing) {
    const unsigned long long n = beyond + (asked > there ? asked - there : 0);
    *a.missing = n < 0x7fffffff ? (int32_t)n : 0x7fffffff;
  }
  // Request r of slot s (before[s] <= r < before[s + 1]) takes the r-th free page.
  const uint32_t given = asked < there ? asked : there;
  for (uint32_t p0 = 0; p0 < a.pages && p0 - rank[p0 >> 5] < given; p0 += kTableThreads) {
    const uint32_t p = p0 + tid;
    if (p >= a.pages || bit_of(bits, p))
      continue;
    const uint32_t r = p - rank_of(bits, rank, p);
    if (r >= given)
      continue;
    int lo = 0, hi = a.slots;  // before[lo] <= r < before[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      (before[mid] <= r ? lo : hi) = mid;
    }
    a.new_tables[(int64_t)lo * a.width + first[lo] + (r - before[lo])] = (int32_t)p;
  }
  each_entry(a, [&](int s, int e) {
    const bool asks = e >= first[s] && e - first[s] < (int)(before[s + 1] - before[s]);
    if (asks && before[s] + (uint32_t)(e - first[s]) < given)
      return;  // given above
    const bool old = e < full[s] || (e == full[s] && kept[s]);
    const int32_t p = old ? a.tables[(int64_t)parent[s] * a.width + e] : -1;
    a.new_tables[(int64_t)s * a.width + e] = (uint32_t)p < a.pages ? p : -1;
  });
  // One slot alone: only a last page that its table lists as a full one too is copied,
  // by this workgroup.  Hardly a call has one, and a launch for it takes 2 us.
  if (a.slots != 1 || last[0] < 0 || kept[0])
    return;
  __threadfence_block();
  __syncthreads();
  const int32_t target = a.new_tables[full[0]];
  if (target < 0)
    return;
  const uint64_t page = (uint64_t)pool.blocks * pool.block_bytes;
  const uint32_t bytes = (uint32_t)(a.new_lengths[0] & ((1 << a.page_log) - 1)) * pool.token_bytes;
  for (uint32_t b = 0; b < pool.blocks; ++b)
    copy_bytes<kTableThreads>(pool.data + (uint64_t)last[0] * page + (uint64_t)b * pool.block_bytes,
                              pool.data + (uint64_t)target * page + (uint64_t)b * pool.block_bytes, bytes);
}

// The pages that cache_assign_kernel gave in place of ones that are shared: what
// their slots hold of them, `part` tokens of every block.  Every workgroup lists the slots
// that fork and takes its share of all their blocks, up to kCopyBytes of one at a time:
// a launch of no more workgroups than the card holds, whatever the slots.  256 slots that
// fork nothing, pages of 4 MB, take 18.6 us a call so, and 115 with a workgroup for each slot and
// kCopyBytes of a page; 64 slots half of which fork 12.6 and 13.2, 8 slots 9.0 and 8.5.
__global__ __launch_bounds__(256) void page_fork_kernel(TableArgs a, PoolArgs p) {
  __shared__ int32_t source[kMaxSlots], target[kMaxSlots], part[kMaxSlots];
  __shared__ int found[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int forks = 0;
  for (int s0 = 0; s0 < a.slots; s0 += 256) {
    const int s = s0 + (int)threadIdx.x;
    const int32_t from = s >= a.slots ? -1 : a.parents ? a.parents[s] : s;
    int32_t src = -1, dst = -1, tokens = 0;
    if ((uint32_t)from < (uint32_t)a.slots) {
      const int32_t length = tokens_of(a.lengths[from], a), full = length >> a.page_log;
      tokens = length & ((1 << a.page_log) - 1);
      if (tokens) {
        src = a.tables[(int64_t)from * a.width + full];
        dst = a.new_tables[(int64_t)s * a.width + full];
      }
    }
    const bool copies = (uint32_t)src < a.pages && (uint32_t)dst < a.pages && src != dst;
    const uint64_t mine = __ballot(copies);
    if (lane == 0)
      found[wave] = __popcll(mine);
    __syncthreads();
    int at = forks + __popcll(mine & ((1ull << lane) - 1));
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      at += w < wave ? found[w] : 0;
      forks += found[w];
    }
    if (copies) {
      source[at] = src;
      target[at] = dst;
      part[at] = tokens;
    }
    __syncthreads();
  }
  const uint64_t page = (uint64_t)p.blocks * p.block_bytes, all = (uint64_t)p.blocks * p.parts;
  const auto copy = [&](auto each) {  // of a fork; 64-bit quotients only where they are needed
    for (decltype(each) i = blockIdx.x; i < (uint32_t)forks * each; i += gridDim.x) {
      const uint32_t f = (uint32_t)(i / each);
      const auto rest = i - f * each, block = rest / p.parts;
      const uint64_t at = (uint64_t)(rest - block * p.parts) * kCopyBytes, off = (uint64_t)block * p.block_bytes + at;
      const uint64_t bytes = (uint64_t)part[f] * p.token_bytes;
      if (at < bytes)
        copy_bytes(p.data + (uint64_t)source[f] * page + off, p.data + (uint64_t)target[f] * page + off,
                   (uint32_t)(bytes - at < kCopyBytes ? bytes - at : kCopyBytes));
    }
  };
  if ((uint64_t)forks * all < (1ull << 31))
    copy((uint32_t)all);
  else
    copy(all);
}

// Of the n pages held by any slot, the i-th at or behind page n moves to the i-th
// free one before it: no page is read that another is written over.  moves[0]
// = their number, then the pairs.
__global__ __launch_bounds__(kTableThreads) void cache_compact_kernel(TableArgs a, int32_t* moves) {
  __shared__ uint32_t bits[kWords], rank[kWords], sums[16];
  __shared__ int32_t held[kMaxSlots];
  const int tid = threadIdx.x, words = words_of(a);
  for (int w = tid; w < words; w += kTableThreads)
    bits[w] = 0;
  if (tid < a.slots)
    held[tid] = (int32_t)(((int64_t)tokens_of(a.lengths[tid], a) + (1 << a.page_log) - 1) >> a.page_log);
  __syncthreads();
  each_entry(a, [&](int s, int e) {
    if (e < held[s]) {
      const uint32_t p = (uint32_t)a.tables[(int64_t)s * a.width + e];
      if (p < a.pages)
        set_bit(bits, p);
    }
  });
  __syncthreads();
  const uint32_t used = count_bits(bits, rank, words, sums);
  const uint32_t low = used < a.pages ? rank_of(bits, rank, used) : used;  // pages that stay
  if (tid == 0) {
    moves[0] = (int32_t)(used - low);
    if (a.missing)
      *a.missing = (int32_t)used;
  }
  for (uint32_t p = tid; p < a.pages; p += kTableThreads) {
    const uint32_t r = rank_of(bits, rank, p);
    const bool is = bit_of(bits, p);
    if (p < used ? !is : is)
      moves[p < used ? 2 + 2 * (p - r) : 1 + 2 * (r - low)] = (int32_t)p;
  }
  __threadfence_block();
  __syncthreads();
  each_entry(a, [&](int s, int e) {
    const uint32_t p = e < held[s] ? (uint32_t)a.tables[(int64_t)s * a.width + e] : ~0u;
    int32_t to = p < a.pages ? (int32_t)p : -1;
    if (p < a.pages && p >= used)
      to = moves[2 + 2 * (rank_of(bits, rank, p) - low)];
    a.new_tables[(int64_t)s * a.width + e] = to;
  });
}

__global__ __launch_bounds__(256) void page_move_kernel(const int32_t* moves, PoolArgs p) {
  const uint64_t page = (uint64_t)p.blocks * p.block_bytes, at = (uint64_t)blockIdx.x * kCopyBytes;
  const uint32_t bytes = (uint32_t)(page - at < kCopyBytes ? page - at : kCopyBytes);
  const int n = moves[0];
  for (int i = blockIdx.y; i < n; i += gridDim.y)
    copy_bytes(p.data + (uint64_t)moves[1 + 2 * i] * page + at, p.data + (uint64_t)moves[2 + 2 * i] * page + at, bytes);
}

}  // namespace

hipError_t launch_cache_write(hipStream_t s, const CacheArgs& c, const CacheRows& in, uint32_t rows, int dtype) {
  const uint32_t per_row = 2 * c.heads * (uint32_t)c.dim / 8;
  const dim3 grid((uint32_t)(((uint64_t)rows * per_row + 255) / 256)), block(256);
  return dtype == kF32 ? dispatch(cache_write_kernel<float>, grid, block, s, c, in, per_row, rows)
                       : dispatch(cache_write_kernel<_Float16>, grid, block, s, c, in, per_row, rows);
}

hipError_t launch_cache_assign(hipStream_t s, const TableArgs& a, const PoolArgs& p) {
  return dispatch(cache_assign_kernel, dim3(1), dim3(kTableThreads), s, a, p);
}

hipError_t launch_page_fork(hipStream_t s, const TableArgs& a, PoolArgs p, int cus) {
  p.parts = (p.block_bytes + kCopyBytes - 1) / kCopyBytes;
  const uint64_t all = (uint64_t)p.blocks * p.parts * (uint64_t)a.slots, most = 8ull * (uint64_t)cus;
  return dispatch(page_fork_kernel, dim3((uint32_t)(all < most ? all : most)), dim3(256), s, a, p);
}

hipError_t launch_cache_compact(hipStream_t s, const TableArgs& a, int32_t* moves) {
  return dispatch(cache_compact_kernel, dim3(1), dim3(kTableThreads), s, a, moves);
}

hipError_t launch_page_move(hipStream_t s, const int32_t* moves, const PoolArgs& p, uint32_t pages, int cus) {
  const uint32_t parts = (uint32_t)(((uint64_t)p.blocks * p.block_bytes + kCopyBytes - 1) / kCopyBytes);
  const uint32_t want = (16u * (uint32_t)cus + parts - 1) / parts, most = pages / 2 > 0 ? pages / 2 : 1;
  return dispatch(page_move_kernel, dim3(parts, want < most ? want : most), dim3(256), s, moves, p);
}

}  // namespace q4k
