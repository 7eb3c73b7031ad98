// Pages of a KV cache: reserving room (new pages, and a copy of a partly filled
// page that others share), writing tokens, committing, forking, compacting an
// accepted path, truncating and freeing. The whole state lives in device memory
// (rb_kv_pages in the header), so every call is asynchronous and can be captured.
//
// What bounds them: moving K / V is HBM traffic (each byte read once, written
// once, in 16-byte pieces); everything else is latency, hence one block that
// plans a call and as few launches as the order of the steps allows, chained by
// programmatic dependent launch. A call is all or nothing: the plan checks every
// entry first, and a call that cannot be served raises the state's status word and
// changes nothing. Writing has no plan: it leaves out the tokens that have no place, and
// a commit of such a token is refused.
//
// Measured (28 layers, 4 kv heads of 128, bf16, pages of 16): 1,024 drafted tokens of four
// sequences truncated, reserved, written (59 MB in, 59 MB out) and compacted 36 us; 16
// samples forked off two prompts, their last pages copied, one token each, 19 us.
#include <algorithm>

#include "common.cuh"
#include "host_util.h"
#include "kv_pages.cuh"

namespace rb {
namespace kvp {

constexpr int kPlanThreads = 1024;
constexpr int kHash = 2 * RB_PAGES_MAX_LIST;   // open addressing at load <= 1/2

__device__ __forceinline__ void refuse(const PagesDev& s, int code) { atomicCAS(s.status, 0, code); }

// A sequence's pages and tokens, within what its row of the table can hold whatever the
// caller's state says.
__device__ __forceinline__ int held_of(const PagesDev& s, int seq) { return min(max(s.held[seq], 0), s.max_pages); }
__device__ __forceinline__ int length_of(const PagesDev& s, int seq) { return min(max(s.lengths[seq], 0), s.max_pages * s.page_size); }

// Inserts v into an open-addressed set of kHash words (-1 = empty); false if it was there.
__device__ __forceinline__ bool set_insert(int* set, int v) {
  int at = (static_cast<uint32_t>(v) * 2654435761u) % kHash;
  for (;;) {
    const int old = atomicCAS(&set[at], -1, v);
    if (old == -1) return true;
    if (old == v) return false;
    at = at + 1 == kHash ? 0 : at + 1;
  }
}
__device__ __forceinline__ bool set_has(const int* set, int v) {
  int at = (static_cast<uint32_t>(v) * 2654435761u) % kHash;
  for (;;) {
    if (set[at] == v) return true;
    if (set[at] == -1) return false;
    at = at + 1 == kHash ? 0 : at + 1;
  }
}

// Every sequence of the list exists and none is named twice. Block-wide; the
// result is the same in every thread. `set` holds the list afterwards.
__device__ bool check_list(const PagesDev& s, const int32_t* seqs, int n, int* set) {
  for (int i = threadIdx.x; i < kHash; i += blockDim.x) set[i] = -1;
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int q = seqs[i];
    bad |= q < 0 || q >= s.max_seqs || !set_insert(set, q);
  }
  return !__syncthreads_or(bad);
}

__host__ __device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Exclusive prefix sum over the block (kPlanThreads threads); `total` in every thread.
__device__ int block_scan(int v, int* total, int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();   // the last use of warp_sums is over
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  *total = warp_sums[31];
  return x - v + (warp ? warp_sums[warp - 1] : 0);
}

// ---------------------------------------------------------------- reserve
// One block: entry i of the list (thread i) needs a copy of its partly filled page
// if that is shared, plus new pages up to length + count. The pages taken are the
// lowest free ones, given out in list order. `copies[3 i]` = (page to copy or -1,
// its copy, filled slots) for the copy kernel that follows.
__global__ void __launch_bounds__(kPlanThreads)
    reserve_plan(const PagesDev s, const int32_t* __restrict__ seqs, const int32_t* __restrict__ counts, int n,
                 int32_t* __restrict__ copies, int32_t* __restrict__ taken) {
  __shared__ int set[kHash];
  __shared__ int shared_page[kPlanThreads];   // the shared, partly filled page entry i would write to, or -1
  __shared__ int4 give[kPlanThreads];         // entry i: sequence, its pages before the call, first of taken[], how many
  __shared__ int warp_sums[32];
  pdl_wait();
  pdl_trigger();
  const int i = threadIdx.x, ps = s.page_size;
  if (i < n) copies[3 * i] = -1;
  if (!check_list(s, seqs, n, set)) {
    if (i == 0) refuse(s, RB_PAGES_BAD_SEQUENCE);
    return;
  }
  int seq = 0, len = 0, held = 0, count = 0, page = -1;
  bool bad = false;
  if (i < n) {
    seq = seqs[i];
    len = length_of(s, seq);
    held = held_of(s, seq);
    count = counts[i];
    bad = count < 0 || count > static_cast<int64_t>(s.max_pages) * ps - len;
    if (!bad && count > 0 && len % ps != 0) {
      const int p = s.table[static_cast<int64_t>(seq) * s.max_pages + len / ps];
      if (p >= 0 && p < s.pages && s.refs[p] > 1) page = p;
    }
  }
  shared_page[i] = page;
  if (__syncthreads_or(bad)) {
    if (i == 0) refuse(s, RB_PAGES_BAD_COUNT);
    return;
  }
  if (page >= 0) {   // the last of those who ask keeps the page if nobody else holds it
    int asking = 0;
    bool last = true;
    for (int j = 0; j < n; ++j) {
      if (shared_page[j] != page) continue;
      ++asking;
      last &= j <= i;
    }
    if (last && asking == s.refs[page]) page = -1;
  }
  const int cow = page >= 0;
  int fresh = i < n ? max(0, static_cast<int>((static_cast<int64_t>(len) + count + ps - 1) / ps) - held) : 0;
  fresh = min(fresh, s.pages + 1);   // more than there are: the sum stays within 32 bits (view() bounds the pages)
  int total;
  const int at = block_scan(cow + fresh, &total, warp_sums);
  give[i] = make_int4(seq, held, at + cow, fresh);
  // the lowest `total` free pages
  int found = 0;
  for (int base = 0; found < total && base < s.pages; base += 4 * kPlanThreads) {
    const int p0 = base + 4 * i;
    int free_mask = 0, here;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (p0 + e < s.pages && s.refs[p0 + e] == 0) free_mask |= 1 << e;
    int rank = found + block_scan(__popc(free_mask), &here, warp_sums);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (free_mask >> e & 1) {
        if (rank < total) taken[rank] = p0 + e;
        ++rank;
      }
    found += here;
  }
  if (found < total) {   // the same in every thread
    if (i == 0) refuse(s, RB_PAGES_NONE_FREE);
    return;
  }
  __syncthreads();       // taken[] and give[] written; every read of refs[] above is over
  if (cow) {
    const int copy = taken[at];
    s.table[static_cast<int64_t>(seq) * s.max_pages + len / ps] = copy;
    s.refs[copy] = 1;
    atomicSub(&s.refs[page], 1);
    copies[3 * i + 1] = copy;
    copies[3 * i + 2] = len % ps;
    copies[3 * i] = page;
  }
  if (i < n) s.held[seq] = held + fresh;
  for (int e = i >> 5; e < n; e += kPlanThreads / 32) {   // a warp per entry
    const int4 g = give[e];
    for (int j = i & 31; j < g.w; j += 32) {
      const int p = taken[g.z + j];
      s.table[static_cast<int64_t>(g.x) * s.max_pages + g.y + j] = p;
      s.refs[p] = 1;
    }
  }
}

// Block (i, layer * 2 + kv): the filled slots of entry i's copied page, every head.
__global__ void __launch_bounds__(256) copy_pages(const PagesDev s, const int32_t* __restrict__ copies) {
  pdl_wait();
  pdl_trigger();
  const int32_t* c = copies + 3 * blockIdx.x;
  const int from = c[0];
  if (from < 0) return;
  const int vecs = s.row_bytes / 16, run = c[2] * vecs;   // 16-byte pieces of one head's filled slots
  const int64_t head = static_cast<int64_t>(s.page_size) * vecs, page = head * s.kv_heads;
  uint4* base = reinterpret_cast<uint4*>(s.store) + static_cast<int64_t>(blockIdx.y) * s.pages * page;
  const uint4* src = base + from * page;
  uint4* dst = base + c[1] * page;
  for (int x = threadIdx.x; x < run * s.kv_heads; x += blockDim.x) {
    const int64_t at = x / run * head + x % run;
    dst[at] = src[at];
  }
}

// ---------------------------------------------------------------- write
// A warp per token and `each` layers (finding the place costs several trips to memory, the
// data one): token t belongs to entry i with offsets[i] <= t <
// offsets[i + 1] (no offsets: t itself) and goes to position length + t - offsets[i].
// Tokens before offsets[0] or from offsets[n] on belong to nobody.
constexpr int kWriteWarps = 4;
struct WriteSrc {
  const uint8_t* p;
  int64_t s_layer, s_token, s_head;   // bytes
};
__global__ void __launch_bounds__(32 * kWriteWarps)
    write_tokens(const PagesDev s, const WriteSrc k, const WriteSrc v, const int32_t* __restrict__ seqs,
                 const int32_t* __restrict__ offsets, int n, int tokens, int layer0, int layers, int each) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * kWriteWarps + (threadIdx.x >> 5);
  if (t >= tokens || n == 0) return;
  int i = t, j = 0;
  if (offsets) {
    int lo = 0, hi = n;   // the last entry whose offset is <= t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (offsets[mid] <= t) lo = mid; else hi = mid - 1;
    }
    i = lo;
    j = t - offsets[i];
    if (j < 0 || i >= n) return;
  } else if (t >= n) {
    return;
  }
  const int seq = seqs[i];
  bool twice = false;   // the same sequence under another entry
  for (int e = lane; e < n; e += 32) twice |= e != i && seqs[e] == seq;
  if (seq < 0 || seq >= s.max_seqs || __any_sync(0xffffffffu, twice)) {
    if (lane == 0) refuse(s, RB_PAGES_BAD_SEQUENCE);
    return;
  }
  const int64_t pos = static_cast<int64_t>(length_of(s, seq)) + j;
  const int64_t idx = pos / s.page_size;
  if (idx >= held_of(s, seq)) {
    if (lane == 0) refuse(s, RB_PAGES_BAD_COUNT);
    return;
  }
  const int page = s.table[static_cast<int64_t>(seq) * s.max_pages + idx];
  if (page < 0 || page >= s.pages || s.refs[page] != 1) {
    if (lane == 0) refuse(s, RB_PAGES_SHARED);
    return;
  }
  const int vecs = s.row_bytes / 16, per = s.kv_heads * vecs;
  const int64_t head = static_cast<int64_t>(s.page_size) * vecs;
  const int64_t side = static_cast<int64_t>(s.pages) * s.kv_heads * head;
  uint4* dst0 = reinterpret_cast<uint4*>(s.store) + static_cast<int64_t>(page) * s.kv_heads * head + (pos % s.page_size) * vecs;
  const int begin = blockIdx.y * each, end = min(layers, begin + each);
  const uint8_t* kt = k.p + t * k.s_token;
  const uint8_t* vt = v.p + t * v.s_token;
  for (int x0 = lane; x0 < per; x0 += 64) {   // two pieces a lane, four layers: up to sixteen loads before their stores
    const int h0 = x0 / vecs, c0 = x0 % vecs, x1 = x0 + 32, h1 = x1 / vecs, c1 = x1 % vecs;
    const bool two = x1 < per;
    const int64_t d0 = h0 * head + c0, d1 = h1 * head + c1;
    const int64_t k0 = h0 * k.s_head + c0 * 16, k1 = h1 * k.s_head + c1 * 16, v0 = h0 * v.s_head + c0 * 16, v1 = h1 * v.s_head + c1 * 16;
    for (int l0 = begin; l0 < end; l0 += 4) {
      uint4 a[4][4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (l0 + e < end) {
          const uint8_t* ks = kt + (l0 + e) * k.s_layer;
          const uint8_t* vs = vt + (l0 + e) * v.s_layer;
          a[e][0] = __ldcs(reinterpret_cast<const uint4*>(ks + k0));
          a[e][1] = __ldcs(reinterpret_cast<const uint4*>(vs + v0));
          if (two) {
            a[e][2] = __ldcs(reinterpret_cast<const uint4*>(ks + k1));
            a[e][3] = __ldcs(reinterpret_cast<const uint4*>(vs + v1));
          }
        }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (l0 + e < end) {
          uint4* dst = dst0 + static_cast<int64_t>(layer0 + l0 + e) * 2 * side;
          dst[d0] = a[e][0];
          dst[side + d0] = a[e][1];
          if (two) {
            dst[d1] = a[e][2];
            dst[side + d1] = a[e][3];
          }
        }
    }
  }
}

// ---------------------------------------------------------------- commit
// A sequence takes only what a write could have put there: every position within the pages it
// holds, on pages that nobody else does. So a round whose reserve or write was refused (the
// host need not look in between) does not make tokens of what was never written. A warp per entry
// looks at the pages.
__global__ void __launch_bounds__(kPlanThreads)
    commit_plan(const PagesDev s, const int32_t* __restrict__ seqs, const int32_t* __restrict__ counts, int n) {
  __shared__ int set[kHash];
  pdl_wait();
  pdl_trigger();
  if (!check_list(s, seqs, n, set)) {
    if (threadIdx.x == 0) refuse(s, RB_PAGES_BAD_SEQUENCE);
    return;
  }
  const int i = threadIdx.x;
  int64_t len = 0;
  bool bad = false, shared = false;
  if (i < n) {
    len = static_cast<int64_t>(length_of(s, seqs[i])) + counts[i];
    bad = counts[i] < 0 || len > static_cast<int64_t>(held_of(s, seqs[i])) * s.page_size;
  }
  if (__syncthreads_or(bad)) {
    if (i == 0) refuse(s, RB_PAGES_BAD_COUNT);
    return;
  }
  for (int e = i >> 5; e < n; e += kPlanThreads / 32) {
    const int from = length_of(s, seqs[e]), to = from + counts[e];   // within the held pages: 32 bits
    const int32_t* row = s.table + static_cast<int64_t>(seqs[e]) * s.max_pages;
    for (int x = from / s.page_size + (i & 31); x < ceil_div(to, s.page_size) && to > from; x += 32) {
      const int p = row[x];
      shared |= p < 0 || p >= s.pages || s.refs[p] != 1;
    }
  }
  if (__syncthreads_or(shared)) {
    if (i == 0) refuse(s, RB_PAGES_SHARED);
    return;
  }
  if (i < n) s.lengths[seqs[i]] = static_cast<int>(len);
}

// ---------------------------------------------------------------- fork
// Plan: every pair is valid (sources exist, targets are distinct, empty and no
// source of the call); ok[0] tells the pairs' blocks, unless (`share`) the plan's block,
// a warp per pair, shares the pages itself.
__global__ void __launch_bounds__(kPlanThreads)
    fork_plan(const PagesDev s, const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int n,
              int32_t* __restrict__ ok, bool share) {
  __shared__ int set[kHash];
  pdl_wait();
  pdl_trigger();
  bool good = check_list(s, dst, n, set);
  const int i = threadIdx.x;
  bool bad = false;
  if (good && i < n) {
    const int a = src[i];
    bad = a < 0 || a >= s.max_seqs || set_has(set, a) || held_of(s, dst[i]) != 0 || length_of(s, dst[i]) != 0;
  }
  good = !__syncthreads_or(bad) && good;
  if (i == 0) {
    ok[0] = good;
    if (!good) refuse(s, RB_PAGES_BAD_SEQUENCE);
  }
  if (!good || !share) return;
  for (int e = i >> 5; e < n; e += kPlanThreads / 32) {
    const int a = src[e], d = dst[e], len = length_of(s, a), pages = ceil_div(len, s.page_size);
    for (int x = i & 31; x < pages; x += 32) {
      const int p = s.table[static_cast<int64_t>(a) * s.max_pages + x];
      s.table[static_cast<int64_t>(d) * s.max_pages + x] = p;
      if (p >= 0 && p < s.pages) atomicAdd(&s.refs[p], 1);
    }
    if ((i & 31) == 0) {
      s.lengths[d] = len;
      s.held[d] = pages;
    }
  }
}
// Block (x, pair): the pages that hold the source's tokens become the target's too.
__global__ void __launch_bounds__(256)
    fork_share(const PagesDev s, const int32_t* __restrict__ src, const int32_t* __restrict__ dst,
               const int32_t* __restrict__ ok) {
  pdl_wait();
  pdl_trigger();
  if (!ok[0]) return;
  const int a = src[blockIdx.y], d = dst[blockIdx.y];
  const int len = length_of(s, a), pages = ceil_div(len, s.page_size);
  for (int x = blockIdx.x * blockDim.x + threadIdx.x; x < pages; x += gridDim.x * blockDim.x) {
    const int p = s.table[static_cast<int64_t>(a) * s.max_pages + x];
    s.table[static_cast<int64_t>(d) * s.max_pages + x] = p;
    if (p >= 0 && p < s.pages) atomicAdd(&s.refs[p], 1);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    s.lengths[d] = len;
    s.held[d] = pages;
  }
}

// Gives back the pages of `seq` from its `keep`-th on (block-wide).
__device__ void release(const PagesDev& s, int seq, int keep, int held) {
  int32_t* row = s.table + static_cast<int64_t>(seq) * s.max_pages;
  for (int x = keep + threadIdx.x; x < held; x += blockDim.x) {
    const int p = row[x];
    row[x] = -1;
    if (p >= 0 && p < s.pages) atomicSub(&s.refs[p], 1);
  }
}

// ---------------------------------------------------------------- truncate / free
// Block i serves entry i and checks the whole list itself: what the checks read
// (length >= new length) stays true while other blocks apply theirs.
__global__ void __launch_bounds__(256)
    truncate_seqs(const PagesDev s, const int32_t* __restrict__ seqs, const int32_t* __restrict__ lengths, int n) {
  __shared__ int set[kHash];
  pdl_wait();
  pdl_trigger();
  if (!check_list(s, seqs, n, set)) {
    if (threadIdx.x == 0) refuse(s, RB_PAGES_BAD_SEQUENCE);
    return;
  }
  bool bad = false;
  if (lengths)
    for (int i = threadIdx.x; i < n; i += blockDim.x) bad |= lengths[i] < 0 || lengths[i] > length_of(s, seqs[i]);
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) refuse(s, RB_PAGES_BAD_COUNT);
    return;
  }
  const int seq = seqs[blockIdx.x], len = lengths ? lengths[blockIdx.x] : 0;
  const int keep = ceil_div(len, s.page_size), held = held_of(s, seq);
  release(s, seq, keep, held);
  __syncthreads();
  if (threadIdx.x == 0) {
    s.lengths[seq] = len;
    if (keep < held) s.held[seq] = keep;
  }
}

// ---------------------------------------------------------------- compact
// Plan: block i checks entry i (every block checks the list) and says so in flags[i].
__global__ void __launch_bounds__(256)
    compact_plan(const PagesDev s, const int32_t* __restrict__ seqs, const int32_t* __restrict__ paths, int64_t ld,
                 int width, const int32_t* __restrict__ counts, int n, int32_t* __restrict__ flags) {
  __shared__ int set[kHash];
  pdl_wait();
  pdl_trigger();
  if (!check_list(s, seqs, n, set)) {
    if (threadIdx.x == 0) {
      refuse(s, RB_PAGES_BAD_SEQUENCE);
      flags[blockIdx.x] = 1;
    }
    return;
  }
  const int seq = seqs[blockIdx.x], m = counts[blockIdx.x], len = length_of(s, seq);
  const int64_t room = static_cast<int64_t>(held_of(s, seq)) * s.page_size - len;
  const int32_t* path = paths + blockIdx.x * ld;
  bool bad = m < 0 || m > width, shared = false;
  if (!bad)
    for (int j = threadIdx.x; j < m; j += blockDim.x) {
      const int a = path[j];
      const bool wrong = a < 0 || a >= room || (j > 0 && path[j - 1] >= a);
      bad |= wrong;
      if (wrong) continue;
      for (const int at : {a, j}) {   // j <= a < room
        const int p = s.table[static_cast<int64_t>(seq) * s.max_pages + (static_cast<int64_t>(len) + at) / s.page_size];
        shared |= p < 0 || p >= s.pages || (at == j && s.refs[p] != 1);
      }
    }
  bad = __syncthreads_or(bad);
  shared = __syncthreads_or(shared);
  if (threadIdx.x == 0) {
    flags[blockIdx.x] = bad || shared;
    if (bad || shared) refuse(s, bad ? RB_PAGES_BAD_COUNT : RB_PAGES_SHARED);
  }
}
// Whether any entry's plan found fault; block-wide.
__device__ __forceinline__ bool refused(const int32_t* flags, int n) {
  int any = 0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) any |= flags[i];
  return __syncthreads_or(any);
}
// Block (x, entry): thread = one 16-byte piece of one (layer, side, head); tokens in
// ascending order, sixteen loads before their stores: a source lies at or after its
// target, and after every earlier target, so no store meets a later load's source.
constexpr int kMoveThreads = 128;
__global__ void __launch_bounds__(kMoveThreads)
    compact_move(const PagesDev s, const int32_t* __restrict__ seqs, const int32_t* __restrict__ paths, int64_t ld,
                 const int32_t* __restrict__ counts, int n, const int32_t* __restrict__ flags) {
  __shared__ int64_t from[kMoveThreads], to[kMoveThreads];   // offsets of a slot in a head's pages, in pieces
  pdl_wait();
  pdl_trigger();
  if (refused(flags, n)) return;
  const int seq = seqs[blockIdx.y], m = counts[blockIdx.y], len = length_of(s, seq);
  const int vecs = s.row_bytes / 16;
  const int64_t head = static_cast<int64_t>(s.page_size) * vecs, page = head * s.kv_heads;
  const int64_t x = static_cast<int64_t>(blockIdx.x) * kMoveThreads + threadIdx.x;
  const bool live = x < static_cast<int64_t>(s.layers) * 2 * s.kv_heads * vecs;
  const int64_t side = x / (s.kv_heads * vecs);
  const int h = static_cast<int>(x / vecs % s.kv_heads), c = static_cast<int>(x % vecs);
  uint4* base = reinterpret_cast<uint4*>(s.store) + side * s.pages * page + h * head + c;
  const int32_t* row = s.table + static_cast<int64_t>(seq) * s.max_pages;
  for (int j0 = 0; j0 < m; j0 += kMoveThreads) {
    const int j = j0 + threadIdx.x, cnt = min(kMoveThreads, m - j0);
    __syncthreads();
    if (j < m) {
      const int64_t a = static_cast<int64_t>(len) + paths[blockIdx.y * ld + j], b = static_cast<int64_t>(len) + j;
      from[threadIdx.x] = row[a / s.page_size] * page + a % s.page_size * vecs;
      to[threadIdx.x] = row[b / s.page_size] * page + b % s.page_size * vecs;
    }
    __syncthreads();
    if (!live) continue;
    for (int e0 = 0; e0 < cnt; e0 += 16) {
      uint4 val[16];
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (e0 + e < cnt) val[e] = base[from[e0 + e]];
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (e0 + e < cnt) base[to[e0 + e]] = val[e];
    }
  }
}
// Block i: the accepted tokens count, pages past them go back.
__global__ void __launch_bounds__(256)
    compact_finish(const PagesDev s, const int32_t* __restrict__ seqs, const int32_t* __restrict__ counts, int n,
                   const int32_t* __restrict__ flags) {
  pdl_wait();
  pdl_trigger();
  if (refused(flags, n)) return;
  const int seq = seqs[blockIdx.x], len = length_of(s, seq) + counts[blockIdx.x];
  const int keep = ceil_div(len, s.page_size), held = held_of(s, seq);
  release(s, seq, keep, held);
  __syncthreads();
  if (threadIdx.x == 0) {
    s.lengths[seq] = len;
    if (keep < held) s.held[seq] = keep;
  }
}

// ---------------------------------------------------------------- host side
int view(const rb_kv_pages* a, PagesDev* s) {
  if (!a || !a->store || !a->table || !a->lengths || !a->held || !a->refs || !a->status) return RB_ERR_INVALID_ARG;
  if (a->layers <= 0 || a->pages <= 0 || a->kv_heads <= 0 || a->page_size <= 0 || a->head_dim <= 0 ||
      a->max_seqs <= 0 || a->max_pages <= 0)
    return RB_ERR_INVALID_ARG;
  if (a->elem_bytes != 2 && a->elem_bytes != 4) return RB_ERR_UNSUPPORTED;
  const int64_t row = static_cast<int64_t>(a->head_dim) * a->elem_bytes;
  if (row % 16 != 0 || !aligned16(a->store)) return RB_ERR_UNSUPPORTED;
  // a page's pieces, a sequence's tokens and a layer's lists are counted in 32 bits
  if (row * a->page_size * a->kv_heads > (INT64_C(1) << 30) || a->page_size * static_cast<int64_t>(a->max_pages) > (INT64_C(1) << 30) ||
      a->layers > 16384 || a->pages > (1 << 20))
    return RB_ERR_CAPACITY;
  *s = PagesDev{static_cast<uint8_t*>(a->store), a->layers, a->pages, a->kv_heads, a->page_size, static_cast<int>(row),
                a->max_seqs, a->max_pages, a->table, a->lengths, a->held, a->refs, a->status};
  return RB_OK;
}
int check_n(int n) { return n < 0 ? RB_ERR_INVALID_ARG : n > RB_PAGES_MAX_LIST ? RB_ERR_CAPACITY : RB_OK; }

}  // namespace kvp

using namespace kvp;

size_t kv_pages_workspace(const rb_kv_pages* a) {
  PagesDev s;
  if (view(a, &s) != RB_OK) return 0;
  return (static_cast<size_t>(s.pages) + 3 * RB_PAGES_MAX_LIST) * sizeof(int32_t);
}

int kv_pages_reserve(const rb_kv_pages* a, const int32_t* seqs, const int32_t* counts, int n, void* ws, size_t bytes,
                     cudaStream_t st) {
  PagesDev s;
  int r = view(a, &s);
  if (r == RB_OK) r = check_n(n);
  if (r != RB_OK || n == 0) return r;
  if (!seqs || !counts) return RB_ERR_INVALID_ARG;
  if (!ws || bytes < kv_pages_workspace(a)) return RB_ERR_WORKSPACE;
  int32_t* copies = static_cast<int32_t*>(ws);
  r = launch_k(reserve_plan, dim3(1), dim3(kPlanThreads), 0, st, true, s, seqs, counts, n, copies,
               copies + 3 * RB_PAGES_MAX_LIST);
  if (r != RB_OK) return r;
  return launch_k(copy_pages, dim3(n, s.layers * 2), dim3(256), 0, st, true, s, copies);
}

int kv_pages_write(const rb_kv_pages* a, const rb_kv_tokens* x, const int32_t* seqs, const int32_t* offsets, int n,
                   cudaStream_t st) {
  PagesDev s;
  int r = view(a, &s);
  if (r == RB_OK) r = check_n(n);
  if (r != RB_OK) return r;
  if (!x || x->tokens < 0 || x->layer0 < 0 || x->layers < 0 || x->layer0 > s.layers - x->layers) return RB_ERR_INVALID_ARG;
  if (n == 0 || x->tokens == 0 || x->layers == 0) return RB_OK;
  if (!seqs || !x->k || !x->v) return RB_ERR_INVALID_ARG;
  const int64_t es = a->elem_bytes;
  for (int64_t v : {x->skl, x->skt, x->skh, x->svl, x->svt, x->svh})
    if (v * es % 16 != 0) return RB_ERR_UNSUPPORTED;
  if (!aligned16(x->k) || !aligned16(x->v)) return RB_ERR_UNSUPPORTED;
  const WriteSrc k{static_cast<const uint8_t*>(x->k), x->skl * es, x->skt * es, x->skh * es};
  const WriteSrc v{static_cast<const uint8_t*>(x->v), x->svl * es, x->svt * es, x->svh * es};
  // about 16 warps an SM before a warp takes more layers; four at a time are in flight
  const int64_t work = static_cast<int64_t>(x->tokens) * x->layers / (device_sm_count() * 16);
  const int each = static_cast<int>(work < 1 ? 1 : work > 8 ? 8 : work);
  return launch_k(write_tokens, dim3(ceil_div(x->tokens, kWriteWarps), ceil_div(x->layers, each)), dim3(32 * kWriteWarps), 0,
                  st, true, s, k, v, seqs, offsets, n, x->tokens, x->layer0, x->layers, each);
}

int kv_pages_commit(const rb_kv_pages* a, const int32_t* seqs, const int32_t* counts, int n, cudaStream_t st) {
  PagesDev s;
  int r = view(a, &s);
  if (r == RB_OK) r = check_n(n);
  if (r != RB_OK || n == 0) return r;
  if (!seqs || !counts) return RB_ERR_INVALID_ARG;
  return launch_k(commit_plan, dim3(1), dim3(kPlanThreads), 0, st, true, s, seqs, counts, n);
}

int kv_pages_fork(const rb_kv_pages* a, const int32_t* src, const int32_t* dst, int n, void* ws, size_t bytes,
                  cudaStream_t st) {
  PagesDev s;
  int r = view(a, &s);
  if (r == RB_OK) r = check_n(n);
  if (r != RB_OK || n == 0) return r;
  if (!src || !dst) return RB_ERR_INVALID_ARG;
  if (!ws || bytes < kv_pages_workspace(a)) return RB_ERR_WORKSPACE;
  int32_t* ok = static_cast<int32_t*>(ws);
  // up to 16 passes of the plan's block over the tables cost less than a second launch
  const bool share = static_cast<int64_t>(n) * s.max_pages <= 16 * kPlanThreads;
  r = launch_k(fork_plan, dim3(1), dim3(kPlanThreads), 0, st, true, s, src, dst, n, ok, share);
  if (r != RB_OK || share) return r;
  return launch_k(fork_share, dim3(std::min(8, ceil_div(s.max_pages, 256)), n), dim3(256), 0, st, true, s, src, dst,
                  ok);
}

int kv_pages_truncate(const rb_kv_pages* a, const int32_t* seqs, const int32_t* lengths, int n, cudaStream_t st) {
  PagesDev s;
  int r = view(a, &s);
  if (r == RB_OK) r = check_n(n);
  if (r != RB_OK || n == 0) return r;
  if (!seqs) return RB_ERR_INVALID_ARG;
  return launch_k(truncate_seqs, dim3(n), dim3(256), 0, st, true, s, seqs, lengths, n);
}

int kv_pages_compact(const rb_kv_pages* a, const int32_t* seqs, const int32_t* paths, int64_t ld, int width,
                     const int32_t* counts, int n, void* ws, size_t bytes, cudaStream_t st) {
  PagesDev s;
  int r = view(a, &s);
  if (r == RB_OK) r = check_n(n);
  if (r != RB_OK) return r;
  if (width < 0 || (width > 0 && ld < width)) return RB_ERR_INVALID_ARG;
  if (n == 0) return RB_OK;
  if (!seqs || !counts || (width > 0 && !paths)) return RB_ERR_INVALID_ARG;
  if (!ws || bytes < kv_pages_workspace(a)) return RB_ERR_WORKSPACE;
  int32_t* flags = static_cast<int32_t*>(ws);
  r = launch_k(compact_plan, dim3(n), dim3(256), 0, st, true, s, seqs, paths, ld, width, counts, n, flags);
  if (r != RB_OK) return r;
  const int64_t pieces = static_cast<int64_t>(s.layers) * 2 * s.kv_heads * (s.row_bytes / 16);
  r = launch_k(compact_move, dim3(static_cast<unsigned>((pieces + kMoveThreads - 1) / kMoveThreads), n), dim3(kMoveThreads),
               0, st, true, s, seqs, paths, ld, counts, n, flags);
  if (r != RB_OK) return r;
  return launch_k(compact_finish, dim3(n), dim3(256), 0, st, true, s, seqs, counts, n, flags);
}

}  // namespace rb
