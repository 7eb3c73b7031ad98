// Log probability of one given token per row, the row's entropy and its best
// alternatives, from one pass over the logits.
//
//   m = max x, S = sum e^(x-m), T = sum (x-m) e^(x-m)
//   log p(t) = x_t - m - log S,   entropy = log S - T / S
//
// Bound: the logits are read once from HBM. A block takes kChunk consecutive
// entries of a row into registers, so max, sums and the chunk's best entries come
// from that one read; a second, small kernel joins a row's chunks in order. The
// chunk grid depends on V alone and each thread owns fixed entries of it, so a row
// gives the same bits alone or among others, whatever its alignment.
#include "common.cuh"
#include "host_util.h"

namespace rb {
namespace lp {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kPer = 32;                     // entries per thread
constexpr int kChunk = kThreads * kPer;      // 8192
constexpr int kMaxTop = RB_LOGPROBS_MAX_TOP;
constexpr float kLog2E = 1.4426950408889634f;

// One chunk: max, S, T and whether a NaN was seen, then the best `top` keys.
struct Stat { float m, s, t; int nan; };

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
// 32 keys, one per lane, descending by lane (bitonic network).
__device__ __forceinline__ uint64_t warp_sort_desc(uint64_t k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d > 0; d >>= 1) {
      const uint64_t o = __shfl_xor_sync(0xffffffffu, k, d);
      const bool up = (lane & size) != 0 && size < 32, low = (lane & d) == 0;
      k = (low != up) ? max64(k, o) : min64(k, o);
    }
  return k;
}
// The 32 largest of two descending lists, descending.
__device__ __forceinline__ uint64_t warp_merge_desc(uint64_t a, uint64_t b) {
  const int lane = threadIdx.x & 31;
  uint64_t k = max64(a, __shfl_sync(0xffffffffu, b, 31 - lane));   // a bitonic list
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const uint64_t o = __shfl_xor_sync(0xffffffffu, k, d);
    k = (lane & d) == 0 ? max64(k, o) : min64(k, o);
  }
  return k;
}

// 2^((x - m) log2 e): the difference first, so that a large m costs no accuracy
__device__ __forceinline__ float exp_diff(float d) { return fast_exp2(d * kLog2E); }

// Sum over the block in a fixed order; every thread gets it.
__device__ __forceinline__ float block_sum(float v, float* buf) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) s += buf[w];
  return s;
}

// Thread t owns entries base + (j * kThreads + t) * W + e, e < W, j < kPer / W (W
// entries are 16 bytes): one 16-byte load where the row allows it.
template <typename T>
__device__ __forceinline__ void load_chunk(const T* row, int base, int V, int off, int size, float (&x)[kPer]) {
  constexpr int W = 16 / sizeof(T);
  const bool vec = (reinterpret_cast<uintptr_t>(row + base) & 15u) == 0;
#pragma unroll
  for (int j = 0; j < kPer / W; ++j) {
    const int i0 = base + (j * kThreads + static_cast<int>(threadIdx.x)) * W;
    if (vec && i0 + W <= V) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4*>(row + i0));
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < W; ++e)
        x[j * W + e] = sizeof(T) == 4 ? __uint_as_float(u[e * sizeof(T) / 4])
                                      : __uint_as_float((e & 1) ? (u[e / 2] & 0xFFFF0000u) : (u[e / 2] << 16));
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) {
        if (i0 + e >= V) x[j * W + e] = -INFINITY;
        else if (sizeof(T) == 4) x[j * W + e] = reinterpret_cast<const float*>(row)[i0 + e];
        else x[j * W + e] = bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(row)[i0 + e]);
      }
    }
    if (i0 < off + size && i0 + W > off) {
#pragma unroll
      for (int e = 0; e < W; ++e)
        if (i0 + e >= off && i0 + e - off < size) x[j * W + e] = -INFINITY;
    }
  }
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads)
    chunk_kernel(const T* __restrict__ logits, int64_t ld, int V, int off, int size, int top, int chunks,
                 Stat* __restrict__ stats, uint64_t* __restrict__ best) {
  constexpr int W = 16 / sizeof(T);
  __shared__ float buf[kWarps];
  __shared__ uint64_t lists[kWarps][32];
  __shared__ uint64_t limit;
  __shared__ int found;
  __shared__ uint64_t cand[TOP ? kMaxTop * kPer : 1];
  pdl_wait();
  pdl_trigger();
  const int chunk = blockIdx.x % chunks, row = blockIdx.x / chunks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float x[kPer];
  load_chunk(logits + row * ld, chunk * kChunk, V, off, size, x);

  float m = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    m = fmaxf(m, x[i]);
    nan |= x[i] != x[i];
  }
  uint64_t mine = 0;
  if (TOP) {   // the thread's best key
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int at = chunk * kChunk + ((i / W) * kThreads + static_cast<int>(threadIdx.x)) * W + i % W;
      if (at < V) mine = max64(mine, key_of(x[i], at));
    }
    if (threadIdx.x == 0) found = 0;
    lists[warp][lane] = warp_sort_desc(mine);
  }
  m = warp_max(m);
  if (lane == 0) buf[warp] = m;
  nan = __syncthreads_or(nan);
  m = buf[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) m = fmaxf(m, buf[w]);
  if (TOP && warp == 0) {
    // The top-th best of the threads' best keys: at least `top` entries reach it,
    // and only the threads whose own best does can hold one of them.
    uint64_t k = lists[0][lane];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) k = warp_merge_desc(k, lists[w][lane]);
    if (lane == top - 1) limit = k;
  }
  const float ref = (m == -INFINITY || m == INFINITY) ? 0.f : m;
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const float d = x[i] - ref, e = exp_diff(d);
    s += e;
    t += e > 0.f ? d * e : 0.f;   // an excluded or vanishing entry adds nothing
  }
  s = block_sum(s, buf);
  t = block_sum(t, buf);
  if (threadIdx.x == 0) stats[blockIdx.x] = Stat{m, s, t, nan};
  if (TOP) {
    const uint64_t lim = limit;   // written before block_sum's barriers
    if (mine >= lim && mine != 0) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int at = chunk * kChunk + ((i / W) * kThreads + static_cast<int>(threadIdx.x)) * W + i % W;
        const uint64_t k = at < V ? key_of(x[i], at) : 0;
        if (k != 0 && k >= lim) cand[atomicAdd(&found, 1)] = k;   // at most top threads come here
      }
    }
    __syncthreads();
    const int n = found;
    uint64_t* out = best + static_cast<int64_t>(blockIdx.x) * top;
    for (int i = threadIdx.x; i < n; i += kThreads) {   // the order of cand[] does not matter: keys differ
      const uint64_t k = cand[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += cand[j] > k;
      if (rank < top) out[rank] = k;
    }
    for (int i = n + static_cast<int>(threadIdx.x); i < top; i += kThreads) out[i] = 0;   // a chunk shorter than top
  }
}

// One warp per row: the chunks in order.
constexpr int kJoinWarps = 4;
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps)
    join_kernel(const T* __restrict__ logits, int64_t ld, int M, int V, const int64_t* __restrict__ tokens, int off,
                int size, int top, int chunks, const Stat* __restrict__ stats, const uint64_t* __restrict__ best,
                float* __restrict__ logprob, float* __restrict__ entropy, float* __restrict__ top_lp,
                int64_t* __restrict__ top_ids) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, row = blockIdx.x * kJoinWarps + (threadIdx.x >> 5);
  if (row >= M) return;
  const Stat* st = stats + static_cast<int64_t>(row) * chunks;
  float m = -INFINITY;
  int nan = 0;
  for (int c = lane; c < chunks; c += 32) {
    m = fmaxf(m, st[c].m);
    nan |= st[c].nan;
  }
  m = warp_max(m);
  nan = __any_sync(0xffffffffu, nan);
  float s = 0.f, t = 0.f;
  for (int c = lane; c < chunks; c += 32) {
    const Stat x = st[c];
    if (x.m == -INFINITY) continue;
    const float d = x.m - m, w = exp_diff(d);
    s = fmaf(w, x.s, s);
    t = fmaf(w, fmaf(d, x.s, x.t), t);
  }
  s = warp_sum(s);
  t = warp_sum(t);
  const float nan_f = __uint_as_float(0x7FC00000u);
  const bool bad = nan || m == -INFINITY || m == INFINITY;
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
      v = x - m - logs;
    }
    logprob[row] = v;
    entropy[row] = bad ? nan_f : logs - t / s;
  }
  if (top > 0) {
    uint64_t k = 0;
    for (int c = 0; c < chunks; ++c) {
      const uint64_t* b = best + (static_cast<int64_t>(row) * chunks + c) * top;
      k = warp_merge_desc(k, lane < top ? b[lane] : 0);
    }
    if (lane < top) {
      top_lp[static_cast<int64_t>(row) * top + lane] = bad ? nan_f : value_of(k) - m - logs;
      top_ids[static_cast<int64_t>(row) * top + lane] = index_of(k);
    }
  }
}

__host__ inline int64_t chunks_of(int V) { return (static_cast<int64_t>(V) + kChunk - 1) / kChunk; }

template <typename T>
int run(const void* logits, int64_t ld, int M, int V, const int64_t* tokens, int off, int size, int top, float* logprob,
        float* entropy, float* top_lp, int64_t* top_ids, void* ws, cudaStream_t st) {
  const int chunks = static_cast<int>(chunks_of(V));
  const T* x = static_cast<const T*>(logits);
  Stat* stats = static_cast<Stat*>(ws);
  uint64_t* best = reinterpret_cast<uint64_t*>(stats + static_cast<int64_t>(M) * chunks);
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(M) * chunks));
  const int r = top > 0 ? launch_k(chunk_kernel<T, true>, grid, dim3(kThreads), 0, st, true, x, ld, V, off, size, top,
                                   chunks, stats, best)
                        : launch_k(chunk_kernel<T, false>, grid, dim3(kThreads), 0, st, true, x, ld, V, off, size, top,
                                   chunks, stats, best);
  if (r != RB_OK) return r;
  return launch_k(join_kernel<T>, dim3((M + kJoinWarps - 1) / kJoinWarps), dim3(32 * kJoinWarps), 0, st, true, x, ld, M,
                  V, tokens, off, size, top, chunks, stats, best, logprob, entropy, top_lp, top_ids);
}

}  // namespace lp

size_t logprobs_workspace(int M, int V, int top) {
  if (M <= 0 || V <= 0 || top < 0) return 0;
  return static_cast<size_t>(M) * lp::chunks_of(V) * (sizeof(lp::Stat) + sizeof(uint64_t) * top);
}

int logprobs_launch(const void* logits, int dtype, int64_t ld, int M, int V, const int64_t* tokens, int off, int size,
                    int top, float* logprob, float* entropy, float* top_lp, int64_t* top_ids, void* ws,
                    cudaStream_t st) {
  if (static_cast<int64_t>(M) * lp::chunks_of(V) > INT32_MAX) return RB_ERR_CAPACITY;
  if (V > INT32_MAX - lp::kChunk) return RB_ERR_CAPACITY;
  if (off > V) off = V;
  if (size > V - off) size = V - off;
  return dtype == RB_F32 ? lp::run<float>(logits, ld, M, V, tokens, off, size, top, logprob, entropy, top_lp, top_ids, ws, st)
                         : lp::run<uint16_t>(logits, ld, M, V, tokens, off, size, top, logprob, entropy, top_lp, top_ids, ws, st);
}

}  // namespace rb
