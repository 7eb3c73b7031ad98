// Log probability of one given token per row, the row's entropy and its best
// alternatives, from one pass over the logits.
//
//   m = max x, S = sum e^(x-m), T = sum (x-m) e^(x-m)
//   log p(t) = x_t - m - log S,   entropy = log S - T / S
//
// Bound: the logits are read once from HBM. A block takes kChunk consecutive entries of
// a row into registers, so maxima, sums and the chunk's best entries come from that one
// read; a second, small kernel joins a row's parts in order. Each warp sums relative to
// its own maximum (one redux), so without alternatives no thread waits for another warp;
// an entry costs an exponential (16 a cycle and SM, 70% of the time the read takes for
// bf16) and about six other instructions, two entries at a time where there are packed
// forms. The grid depends on V alone and each thread owns fixed entries of it, so a row
// gives the same bits alone or among others, whatever its alignment.
#include <type_traits>

#include "common.cuh"
#include "host_util.h"

namespace rb {
namespace lp {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kBytes = 128;                  // of a row per thread
template <typename T>
struct Shape {
  static constexpr int kPer = kBytes / sizeof(T);   // entries per thread: 32 fp32, 64 bf16
  static constexpr int kChunk = kThreads * kPer;
  static constexpr int W = 16 / sizeof(T);          // entries of a 16-byte piece
};
constexpr int kMaxTop = RB_LOGPROBS_MAX_TOP;
constexpr float kLog2E = 1.4426950408889634f;

// One warp's entries: maximum (a NaN if there is one), S, T.
struct Stat { float m, s, t, pad; };

// Order of the alternatives as one integer: larger value first (NaN above all,
// -0 equal to 0), then lower index. 0 is below every key.
__device__ __forceinline__ uint64_t key_of(float x, int index) {
  uint32_t u = __float_as_uint(x + 0.0f);
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  if (x != x) u = 0xFFFFFFFFu;
  return (static_cast<uint64_t>(u) << 32) | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ int index_of(uint64_t key) { return static_cast<int>(~static_cast<uint32_t>(key)); }
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t u = static_cast<uint32_t>(key >> 32);
  if (u == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u);
}

__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t min64(uint64_t a, uint64_t b) { return a < b ? a : b; }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float smaller(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return max64(a, b); }
__device__ __forceinline__ uint64_t smaller(uint64_t a, uint64_t b) { return min64(a, b); }
// 32 values, one per lane, descending by lane (bitonic network).
template <typename K>
__device__ __forceinline__ K warp_sort_desc(K k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d > 0; d >>= 1) {
      const K o = __shfl_xor_sync(0xffffffffu, k, d);
      const bool up = (lane & size) != 0 && size < 32, low = (lane & d) == 0;
      k = (low != up) ? larger(k, o) : smaller(k, o);
    }
  return k;
}
// The 32 largest of two descending lists, descending.
template <typename K>
__device__ __forceinline__ K warp_merge_desc(K a, K b) {
  const int lane = threadIdx.x & 31;
  K k = larger(a, __shfl_sync(0xffffffffu, b, 31 - lane));   // a bitonic list
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const K o = __shfl_xor_sync(0xffffffffu, k, d);
    k = (lane & d) == 0 ? larger(k, o) : smaller(k, o);
  }
  return k;
}

// 2^((x - m) log2 e): the difference first, so that a large m costs no accuracy
__device__ __forceinline__ float exp_diff(float d) { return fast_exp2(d * kLog2E); }
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float warp_max_nan(float a) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(a));
  return r;
}

// A thread's entries stay as they were read (bf16 packed) and are widened at each use.
// Thread t owns entries base + (j * kThreads + t) * W + e, e < W, j < 8: one 16-byte load
// per j where the row allows it. Entries past the row and excluded ones are -inf.
template <typename T>
struct Entries {
  uint32_t raw[kBytes / 4];
  __device__ __forceinline__ float operator[](int i) const {
    if (sizeof(T) == 4) return __uint_as_float(raw[i]);
    return __uint_as_float((i & 1) ? (raw[i / 2] & 0xFFFF0000u) : (raw[i / 2] << 16));
  }
  __device__ __forceinline__ void clear(int i) {   // entry i: -inf
    if (sizeof(T) == 4) raw[i] = 0xFF800000u;
    else raw[i / 2] = (i & 1) ? ((raw[i / 2] & 0xFFFFu) | 0xFF800000u) : ((raw[i / 2] & 0xFFFF0000u) | 0xFF80u);
  }
  __device__ __forceinline__ static int at(int i) {   // entry i: offset in the chunk
    constexpr int W = Shape<T>::W;
    return ((i / W) * kThreads + static_cast<int>(threadIdx.x)) * W + i % W;
  }
  __device__ __forceinline__ float max() const {      // a NaN if there is one
    if (sizeof(T) == 4) {
      float m = __uint_as_float(raw[0]);
#pragma unroll
      for (int i = 1; i < kBytes / 4; ++i) m = max_nan(m, __uint_as_float(raw[i]));
      return m;
    }
    uint32_t m = raw[0];
#pragma unroll
    for (int i = 1; i < kBytes / 4; ++i) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(raw[i]));
    return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u));
  }
  __device__ __forceinline__ void load(const T* row, int base, int V, int off, int size) {
    constexpr int W = Shape<T>::W;
    const bool vec = (reinterpret_cast<uintptr_t>(row + base) & 15u) == 0;
    if (vec && base + Shape<T>::kChunk <= V) {
#pragma unroll
      for (int j = 0; j < kBytes / 16; ++j) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(row + base) + j * kThreads + threadIdx.x);
        raw[4 * j] = v.x;
        raw[4 * j + 1] = v.y;
        raw[4 * j + 2] = v.z;
        raw[4 * j + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < kBytes / 16; ++j) {
        const int i0 = base + at(j * W);
        if (vec && i0 + W <= V) {
          const uint4 v = __ldcs(reinterpret_cast<const uint4*>(row + i0));
          raw[4 * j] = v.x;
          raw[4 * j + 1] = v.y;
          raw[4 * j + 2] = v.z;
          raw[4 * j + 3] = v.w;
        } else {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            if (sizeof(T) == 4) {
              raw[4 * j + w] = i0 + w < V ? reinterpret_cast<const uint32_t*>(row)[i0 + w] : 0xFF800000u;
            } else {
              const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
              const uint32_t lo = i0 + 2 * w < V ? h[i0 + 2 * w] : 0xFF80u, hi = i0 + 2 * w + 1 < V ? h[i0 + 2 * w + 1] : 0xFF80u;
              raw[4 * j + w] = lo | (hi << 16);
            }
          }
        }
      }
    }
    if (base < off + size && base + Shape<T>::kChunk > off) {
#pragma unroll
      for (int i = 0; i < Shape<T>::kPer; ++i) {
        const int x = base + at(i);
        if (x >= off && x - off < size) clear(i);
      }
    }
  }
};

// The chunk's best entries. A limit that at least `top` entries reach and few others do:
// the top-th largest of 32 maxima, one per lane number. Entries from the limit up go to
// shared memory in any order (their keys differ) and are ranked by counting. Where many
// tie at the limit, the lowest indices among them are taken, in order; where too many
// lie above it, or a NaN is among them, the best entry is taken `top` times.
constexpr int kCand = 1024;
struct TopShared {
  float maxima[kWarps][32];
  float limit;
  int found, warp_count[kWarps];
  uint64_t cand[kCand], round;
};
// A thread's candidates are found as a bit mask over its registers and read again from
// memory by number: few threads have any, and code that takes every register apart is long.
template <typename T>
__device__ __forceinline__ void choose(const Entries<T>& x, float mine, bool nan, const T* row, int base, int V, int off, int size,
                                       int top, TopShared& sh, uint64_t* out) {
  constexpr int kPer = Shape<T>::kPer, W = Shape<T>::W;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float limit = sh.limit;
  auto value = [&](int i) {
    const int at = base + x.at(i);
    if (at >= V || (at >= off && at - off < size)) return -INFINITY;
    return sizeof(T) == 4 ? reinterpret_cast<const float*>(row)[at] : bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(row)[at]);
  };
  auto push = [&](int i, float v) {
    const int c = atomicAdd(&sh.found, 1);
    if (c < kCand) sh.cand[c] = key_of(v, base + x.at(i));
  };
  // at -inf there are always too many
  const bool crowded = limit == -INFINITY;
  if (mine >= limit && !crowded && !nan) {   // entries past the row are -inf: below the limit
    uint64_t bits = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) bits |= static_cast<uint64_t>(x[i] >= limit) << i;
#pragma unroll 1
    for (; bits; bits &= bits - 1) {
      const int i = __ffsll(bits) - 1;
      push(i, value(i));
    }
  }
  __syncthreads();
  int n = sh.found;
  if (n > kCand || crowded || nan) {   // the same in every thread, as is every branch below
    __syncthreads();
    if (threadIdx.x == 0) sh.found = 0;
    __syncthreads();
    if (mine > limit && !nan) {
#pragma unroll 1
      for (int i = 0; i < kPer; ++i) {
        const float v = value(i);
        if (v > limit) push(i, v);
      }
    }
    __syncthreads();
    n = sh.found;
    if (nan || n > kCand - kMaxTop) {
      uint64_t last = ~0ull;
#pragma unroll 1
      for (int r = 0; r < top; ++r) {
        if (threadIdx.x == 0) sh.round = 0;
        __syncthreads();
        uint64_t k = 0;
#pragma unroll 1
        for (int i = 0; i < kPer; ++i) {
          const uint64_t c = base + x.at(i) < V ? key_of(value(i), base + x.at(i)) : 0;
          if (c < last) k = max64(k, c);
        }
        atomicMax(reinterpret_cast<unsigned long long*>(&sh.round), static_cast<unsigned long long>(k));
        __syncthreads();
        last = sh.round;
        if (threadIdx.x == 0) out[r] = last;
        __syncthreads();
      }
      return;
    }
    int ties = 0;         // taken so far, in index order: j, then thread, then entry
#pragma unroll 1
    for (int j = 0; j < kBytes / 16 && ties < top; ++j) {
      int here = 0;
#pragma unroll 1
      for (int e = 0; e < W; ++e) here += value(j * W + e) == limit && base + x.at(j * W + e) < V;
      int sum = here;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      if (lane == 31) sh.warp_count[warp] = sum;
      __syncthreads();
      int at = ties + sum - here, all = 0;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) at += sh.warp_count[w];
        all += sh.warp_count[w];
      }
#pragma unroll 1
      for (int e = 0; e < W; ++e) {
        const int pos = base + x.at(j * W + e);
        if (value(j * W + e) == limit && pos < V && at < top) sh.cand[n + at++] = key_of(limit, pos);
      }
      ties += all;
      __syncthreads();
    }
    n += min(ties, top);
  }
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t k = sh.cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += sh.cand[j] > k;
    if (rank < top) out[rank] = k;
  }
  for (int i = n + static_cast<int>(threadIdx.x); i < top; i += kThreads) out[i] = 0;   // a chunk shorter than top
}

// Blocks of an SM, by what fits without much spilling: more of them hide each other's waits
// (rows of 152,064: 512 fp32 without alternatives 47 us = 6.6 TB/s, 2,000 bf16 103-110 us = 5.5-5.9;
// with 20 alternatives 128 fp32 20.7 us, 512 bf16 58 us = 2.7 TB/s).
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, TOP ? (sizeof(T) == 4 ? 5 : 4) : 6)
    chunk_kernel(const T* __restrict__ logits, int64_t ld, int V, int off, int size, int top, int chunks,
                 Stat* __restrict__ stats, uint64_t* __restrict__ best) {
  __shared__ typename std::conditional<TOP, TopShared, int>::type shared;
  pdl_wait();
  pdl_trigger();
  const int chunk = blockIdx.x % chunks, row = blockIdx.x / chunks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, base = chunk * Shape<T>::kChunk;
  Entries<T> x;
  x.load(logits + row * ld, base, V, off, size);
  const float mine = x.max();
  const float m = warp_max_nan(mine);
  if constexpr (TOP) {
    if (threadIdx.x == 0) shared.found = 0;
    shared.maxima[warp][lane] = mine;
    __syncthreads();
    if (warp == 0) {
      float k = mine;
#pragma unroll
      for (int w = 1; w < kWarps; ++w) k = fmaxf(k, shared.maxima[w][lane]);
      k = warp_sort_desc(k);
      if (lane == top - 1) shared.limit = k;
    }
  }
  // relative to the warp's maximum; an entry of -inf weighs nothing (a finite number times 0)
  const float ref = (m == -INFINITY || m == INFINITY) ? 0.f : m;
  const uint64_t minus = pair(-ref, -ref), log2e = pair(kLog2E, kLog2E);
  uint64_t s2 = pair(0.f, 0.f), t2 = pair(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < Shape<T>::kPer; i += 2) {
    float a, b;
    unpair(add2(pair(x[i], x[i + 1]), minus), a, b);
    const uint64_t d = pair(fmaxf(a, -1e30f), fmaxf(b, -1e30f));
    unpair(mul2(d, log2e), a, b);
    const uint64_t e = pair(fast_exp2(a), fast_exp2(b));
    s2 = add2(s2, e);
    t2 = fma2(d, e, t2);
  }
  float s0, s1, t0, t1;
  unpair(s2, s0, s1);
  unpair(t2, t0, t1);
  const float s = warp_sum(s0 + s1), t = warp_sum(t0 + t1);
  if (lane == 0) *reinterpret_cast<float4*>(stats + static_cast<int64_t>(blockIdx.x) * kWarps + warp) = make_float4(m, s, t, 0.f);
  if constexpr (TOP) {
    const bool nan = __syncthreads_or(mine != mine);
    choose<T>(x, mine, nan, logits + row * ld, base, V, off, size, top, shared, best + static_cast<int64_t>(blockIdx.x) * top);
  }
}

// The row's sums in order, by one warp, and the chunks' best entries: a block per row with
// alternatives (warp 0 has the sums, the others share the lists meanwhile), a warp per row
// without.
template <bool TOP>
constexpr int kJoinWarps = TOP ? 9 : 4;
template <typename T, bool TOP>
__global__ void __launch_bounds__(32 * kJoinWarps<TOP>)
    join_kernel(const T* __restrict__ logits, int64_t ld, int M, int V, const int64_t* __restrict__ tokens, int off,
                int size, int top, int chunks, const Stat* __restrict__ stats, const uint64_t* __restrict__ best,
                float* __restrict__ logprob, float* __restrict__ entropy, float* __restrict__ top_lp,
                int64_t* __restrict__ top_ids) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = TOP ? blockIdx.x : blockIdx.x * kJoinWarps<TOP> + warp;
  if (row >= M) return;
  __shared__ uint64_t lists[TOP ? kJoinWarps<TOP> - 1 : 1][32];
  if constexpr (TOP) {
    if (warp > 0) {
      const uint64_t* b = best + static_cast<int64_t>(row) * chunks * top;
      uint64_t k = 0;
#pragma unroll 4
      for (int c = warp - 1; c < chunks; c += kJoinWarps<TOP> - 1)
        k = warp_merge_desc(k, lane < top ? b[static_cast<int64_t>(c) * top + lane] : uint64_t(0));
      lists[warp - 1][lane] = k;
      __syncthreads();
      return;
    }
  }
  const int64_t parts = static_cast<int64_t>(chunks) * kWarps;
  const float4* st = reinterpret_cast<const float4*>(stats + row * parts);
  // running (m, s, t) per lane: one pass over the row's parts
  float m = -INFINITY, s = 0.f, t = 0.f;
#pragma unroll 4
  for (int64_t c = lane; c < parts; c += 32) {
    const float4 x = st[c];
    const float hi = max_nan(m, x.x), ref = (hi == -INFINITY || hi == INFINITY) ? 0.f : hi;
    // a side of -inf has nothing in it
    const float da = fmaxf(m - ref, -1e30f), db = fmaxf(x.x - ref, -1e30f);
    const float wa = exp_diff(da), wb = exp_diff(db);
    t = wa * fmaf(da, s, t) + wb * fmaf(db, x.y, x.z);
    s = wa * s + wb * x.y;
    m = hi;
  }
  const float top_m = warp_max_nan(m), ref = (top_m == -INFINITY || top_m == INFINITY) ? 0.f : top_m;
  const float d = fmaxf(m - ref, -1e30f), w = exp_diff(d);
  t = warp_sum(w * fmaf(d, s, t));
  s = warp_sum(w * s);
  const float nan_f = __uint_as_float(0x7FC00000u);
  const bool bad = top_m != top_m || top_m == -INFINITY || top_m == INFINITY;
  const float logs = logf(s);
  if (lane == 0) {
    const int64_t tok = tokens[row];
    float v = nan_f;
    if (!bad && tok >= 0 && tok < V) {
      float x = -INFINITY;
      if (tok < off || tok - off >= size) {
        if (sizeof(T) == 4) x = reinterpret_cast<const float*>(logits)[row * ld + tok];
        else x = bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(logits)[row * ld + tok]);
      }
      v = x - top_m - logs;
    }
    logprob[row] = v;
    entropy[row] = bad ? nan_f : logs - t / s;
  }
  if constexpr (TOP) {
    __syncthreads();
    uint64_t k = lists[0][lane];
#pragma unroll
    for (int w = 1; w < kJoinWarps<TOP> - 1; ++w) k = warp_merge_desc(k, lists[w][lane]);
    if (lane < top) {
      top_lp[static_cast<int64_t>(row) * top + lane] = bad ? nan_f : value_of(k) - top_m - logs;
      top_ids[static_cast<int64_t>(row) * top + lane] = index_of(k);
    }
  }
}

__host__ inline int64_t chunks_of(int V, int chunk) { return (static_cast<int64_t>(V) + chunk - 1) / chunk; }

template <typename T>
int run(const void* logits, int64_t ld, int M, int V, const int64_t* tokens, int off, int size, int top, float* logprob,
        float* entropy, float* top_lp, int64_t* top_ids, void* ws, cudaStream_t st) {
  const int chunks = static_cast<int>(chunks_of(V, Shape<T>::kChunk));
  const T* x = static_cast<const T*>(logits);
  Stat* stats = static_cast<Stat*>(ws);
  uint64_t* best = reinterpret_cast<uint64_t*>(stats + static_cast<int64_t>(M) * chunks * kWarps);
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(M) * chunks));
  auto go = [&](auto chunk, auto join, int rows_per_block, int threads) {
    const int r = launch_k(chunk, grid, dim3(kThreads), 0, st, true, x, ld, V, off, size, top, chunks, stats, best);
    if (r != RB_OK) return r;
    return launch_k(join, dim3((M + rows_per_block - 1) / rows_per_block), dim3(threads), 0, st, true, x, ld, M, V, tokens,
                    off, size, top, chunks, stats, best, logprob, entropy, top_lp, top_ids);
  };
  return top > 0 ? go(chunk_kernel<T, true>, join_kernel<T, true>, 1, 32 * kJoinWarps<true>)
                 : go(chunk_kernel<T, false>, join_kernel<T, false>, kJoinWarps<false>, 32 * kJoinWarps<false>);
}

}  // namespace lp

size_t logprobs_workspace(int M, int V, int top) {
  if (M <= 0 || V <= 0 || top < 0) return 0;   // of fp32's chunks, the smaller ones
  return static_cast<size_t>(M) * lp::chunks_of(V, lp::Shape<float>::kChunk) * (sizeof(lp::Stat) * lp::kWarps + sizeof(uint64_t) * top);
}

int logprobs_launch(const void* logits, int dtype, int64_t ld, int M, int V, const int64_t* tokens, int off, int size,
                    int top, float* logprob, float* entropy, float* top_lp, int64_t* top_ids, void* ws,
                    cudaStream_t st) {
  if (static_cast<int64_t>(M) * lp::chunks_of(V, lp::Shape<float>::kChunk) > INT32_MAX) return RB_ERR_CAPACITY;
  if (V > INT32_MAX - lp::Shape<uint16_t>::kChunk) return RB_ERR_CAPACITY;
  if (off > V) off = V;
  if (size > V - off) size = V - off;
  return dtype == RB_F32 ? lp::run<float>(logits, ld, M, V, tokens, off, size, top, logprob, entropy, top_lp, top_ids, ws, st)
                         : lp::run<uint16_t>(logits, ld, M, V, tokens, off, size, top, logprob, entropy, top_lp, top_ids, ws, st);
}

}  // namespace rb
