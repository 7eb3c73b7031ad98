// Attention of one new token per sequence over a paged KV cache.
//
//   out[b, h] = sum_t softmax_t(q[b, h] . k_t * scale) v_t,   t < length of sequence b
//
// Bound: every cached K and V row is read once from HBM for all heads of its group
// (4 D flops per 2 D elements and query head: far below the tensor ridge). The length is
// cut into chunks at absolute positions whose size depends on the sequence's own length
// only; every chunk leaves its (accumulator, max, sum), and a second kernel joins them in
// chunk order, so a sequence gives the same bits alone or in any batch. A warp works for
// itself: it takes consecutive chunks (as many as the launch has too many of) in tiles of
// 16 keys through its own ring of asynchronous copies, which runs on across chunks.
//
// bf16: S^T = K Q^T and O^T = V^T P^T on m16n8k16 tiles, so that the group's heads are the
// 8 (or 16) columns: a group of up to 8 wastes no rows and needs half the accumulators. P
// enters as two bf16 parts (hi + lo), so a weight is good to 2^-16 and the result is
// rounded once, at the end. fp32: three tf32 products per term, each step from zero and
// added in fp32. Where pages hold whole tiles, a tile arrives as TMA boxes, else row by row.
//
// Measured (both launches, one B200): 64 bf16 sequences of 512 to 12,000 tokens, 32 / 8 heads,
// 286 us = 5.5 TB/s (with heads as rows and blocks of four warps 335); 256 of 1,024 tokens 5.1
// TB/s; one of 120,000 4.7 TB/s; one of 4,133, 28 / 4 heads, 14 us, of which most is latency.
#include <type_traits>

#include "common.cuh"
#include "host_util.h"

namespace rb {
namespace pg {

constexpr int kD = 128;
constexpr int kThreads = 32;               // a block is one warp: they share nothing, and spread evenly
constexpr int kKeys = 16;                  // keys of a tile
constexpr int kRows = 16;                  // query heads of a block
constexpr int kMinChunk = 32, kMaxChunk = 2048;

// Keys per chunk of a sequence of `len` tokens: in bf16 64 up to 4,096 tokens, then doubled
// each time the length is four times larger; in fp32, whose keys are twice as long and cost
// several times the instructions, 32 up to 16,384. A chunk's result costs G x 520 bytes written and read against 512 bytes a key
// (bf16): 6% of the traffic for a group of 4 at 64. A single sequence pays where the size doubles, as half
// as many warps read it: 4,096 tokens of 28 / 4 heads take 11.6 us, 4,097 take 14.6.
__host__ __device__ constexpr int kGrow(int es) { return es == 2 ? 1 : 16; }
__host__ __device__ inline int chunk_of(int len, int es) {
  int c = kMinChunk * 4 / es;
  while (c < kMaxChunk && static_cast<int64_t>(kGrow(es)) * c * c < len) c *= 2;
  return c;
}
__host__ __device__ inline int chunks_of(int len, int es) {
  const int c = chunk_of(len, es);
  return len / c + (len % c != 0);
}
// Upper bound of chunks_of over every length up to `len`.
__host__ inline int max_chunks(int len, int es) {
  int n = 1;
  for (int c = kMinChunk * 4 / es;; c *= 2) {   // the longest length each size serves
    const int64_t top = c < kMaxChunk ? static_cast<int64_t>(kGrow(es)) * c * c : len;
    const int x = static_cast<int>(top < len ? top : len);
    const int k = chunks_of(x, es);
    n = k > n ? k : n;
    if (x == len) return n;
  }
}

struct Dev {
  const void* q;
  int64_t sqb, sqh;
  const void *k, *v;
  int64_t skp, skh, sks, svp, svh, svs;   // strides of pages, heads, slots (elements)
  const int32_t *table, *lengths, *seqs;
  int64_t ld_table;
  int B, H, HK, pages, page_size, width, rows, ahead, max_len;
  int es;                                  // bytes of an element
  int splits, per_warp;                    // chunks a sequence may have; consecutive chunks a warp takes
  void* out;
  int64_t sob, soh;
  float scale2;                            // sm_scale * log2 e
};

// The table row of batch entry b and how many of its tokens are read.
__device__ __forceinline__ int length_of(const Dev& p, int b, int* row) {
  const int r = p.seqs ? p.seqs[b] : b;
  *row = r;
  if (r < 0 || r >= p.rows) return 0;
  const int64_t len = static_cast<int64_t>(p.lengths[r]) + p.ahead;
  return static_cast<int>(len < 0 ? 0 : len > p.max_len ? p.max_len : len);
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

// The weights' sum of a chunk none of whose tokens has a page: tells it from one whose scores are
// all -inf, whose sum is 0 (and whose sequence, if nothing else is in it, has no value: 0 / 0).
constexpr float kNothing = -1.f;

// What a warp works on: consecutive chunks of one sequence and kv head.
struct Item {
  int b, kvh, h0, nh;        // batch entry, kv head, first query head and how many
  int len, chunk, chunks;    // tokens read, keys per chunk, chunks of the sequence
  int c0, k0, k1;            // first chunk of the warp, its keys
  const int32_t* table;      // the sequence's row
};
__device__ __forceinline__ bool item_of(const Dev& p, Item* it) {
  const int G = p.H / p.HK, tiles = (G + kRows - 1) / kRows;
  it->b = blockIdx.z;
  it->kvh = blockIdx.y / tiles;
  const int g0 = blockIdx.y % tiles * kRows;
  it->h0 = it->kvh * G + g0;
  it->nh = min(kRows, G - g0);
  int row;
  it->len = length_of(p, it->b, &row);
  it->table = p.table + row * p.ld_table;
  it->chunk = chunk_of(it->len, p.es);
  it->chunks = chunks_of(it->len, p.es);
  it->c0 = blockIdx.x * p.per_warp;
  if (it->c0 >= it->chunks) return false;
  it->k0 = it->c0 * it->chunk;
  it->k1 = min(static_cast<int64_t>(it->len), it->k0 + static_cast<int64_t>(p.per_warp) * it->chunk);
  return true;
}

// Where a chunk's result goes: accumulators [B, H, splits, kD], then (max, sum) [B, H, splits].
__device__ __forceinline__ float* acc_at(const Dev& p, float* part, const Item& it, int r, int c) {
  return part + ((static_cast<int64_t>(it.b) * p.H + it.h0 + r) * p.splits + c) * kD;
}
__device__ __forceinline__ float2* ml_at(const Dev& p, float* part, const Item& it, int r, int c) {
  return reinterpret_cast<float2*>(part + static_cast<int64_t>(p.B) * p.H * p.splits * kD) +
         (static_cast<int64_t>(it.b) * p.H + it.h0 + r) * p.splits + c;
}
template <typename T>
__device__ __forceinline__ T* out_at(const Dev& p, const Item& it, int r) {
  return static_cast<T*>(p.out) + it.b * p.sob + (it.h0 + r) * p.soh;
}
template <typename T>
__device__ __forceinline__ void write_empty(const Dev& p, const Item& it) {   // by the sequence's first warp
  if (it.c0 != 0) return;
  for (int x = threadIdx.x & 31; x < it.nh * kD; x += 32) out_at<T>(p, it, x / kD)[x % kD] = T(0);
}

// Row r of chunk c again, by one warp and key by key. A product in several parts turns an
// infinity into a NaN (infinity times a second part of zero) that the plain product is
// not; a row that came out NaN is settled here. A weight that is zero, or that a later
// maximum makes zero, turns an attended infinity or NaN into a NaN, as in the tiles.
template <typename T>
__device__ __noinline__ void redo_row(const Dev& p, const Item& it, float* part, int r, int c) {
  const int lane = threadIdx.x & 31, d = lane * 4;
  auto load = [&](const void* base, int64_t at, float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      x[e] = sizeof(T) == 4 ? static_cast<const float*>(base)[at + d + e]
                            : bf16_bits_to_f32(static_cast<const uint16_t*>(base)[at + d + e]);
  };
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  load(p.q, it.b * p.sqb + (it.h0 + r) * p.sqh, q);
  const int end = min(static_cast<int64_t>(it.len), (c + static_cast<int64_t>(1)) * it.chunk);
  for (int key = c * it.chunk; key < end; ++key) {
    const int page = it.table[key / p.page_size], slot = key % p.page_size;
    if (page < 0 || page >= p.pages) continue;
    float k[4], v[4];
    load(p.k, page * p.skp + it.kvh * p.skh + slot * p.sks, k);
    load(p.v, page * p.svp + it.kvh * p.svh + slot * p.svs, v);
    const float s = warp_sum(fmaf(q[0], k[0], fmaf(q[1], k[1], fmaf(q[2], k[2], q[3] * k[3])))) * p.scale2;
    const float mx = fmaxf(m, s), ref = mx == -INFINITY ? 0.f : mx;
    const float a = fast_exp2(m - ref), x = fast_exp2(s - ref);
    m = mx;
    l = fmaf(l, a, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(o[e], a, x * v[e]);
  }
  if (it.chunks == 1) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (sizeof(T) == 4) out_at<float>(p, it, r)[d + e] = o[e] / l;
      else out_at<uint16_t>(p, it, r)[d + e] = f32_to_bf16_bits(o[e] / l);
    }
  } else {
    *reinterpret_cast<float4*>(acc_at(p, part, it, r, c) + d) = make_float4(o[0], o[1], o[2], o[3]);
    if (lane == 0) *ml_at(p, part, it, r, c) = make_float2(m, l);
  }
}

// A tile in shared memory, K then V. From TMA boxes: blocks of 128 bytes of all 16 rows,
// 16-byte pieces swizzled by row & 7. Gathered: whole rows, 16 bytes apart beyond their
// length. Either way eight rows' pieces of one column lie in different banks.
constexpr int kQPitch = kD + 4;
template <typename T, bool kTma>
struct Ring {
  // Tiles in a warp's ring. fp32 tiles are twice as large and take long to compute: eight warps
  // an SM with a tile each hide more than five with two (32 sequences of 2,048 tokens, 28 / 4
  // heads: 91 us against 124; one of 4,133: 15 either way).
  static constexpr int kStages = sizeof(T) == 2 ? 3 : 1;
  static constexpr int kRow = kD * sizeof(T);
  static constexpr int kSide = kKeys * (kTma ? kRow : kRow + 16), kTile = 2 * kSide;
  // ring, mbarriers, fp32: the tile's weights and the queries (pitches free of bank conflicts)
  static constexpr int smem(int nt) {
    return 1024 + kStages * kTile + 64 + (sizeof(T) == 4 ? (kKeys * (nt == 1 ? 12 : 20) + nt * 8 * kQPitch) * 4 : 0);
  }
  __device__ __forceinline__ static uint32_t at(uint32_t side, int row, int piece) {
    return kTma ? side + (piece >> 3) * (kKeys * 128) + row * 128 + (((piece & 7) ^ (row & 7)) * 16) : side + row * (kRow + 16) + piece * 16;
  }
};
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int slot, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(bar)
      : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {   // an 8 x 8 bf16 matrix, one register a lane
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// x = hi + lo: hi rounded to tf32's 11 bits by integer arithmetic (the conversion
// instruction is several times slower), lo what is left, which the tensor core cuts to 11
// bits: good to 2^-22 of x. A NaN survives in lo; an infinity gives one.
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(   // not volatile: independent products may pass one another
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
struct Split4 {
  uint32_t hi[4], lo[4];
  __device__ __forceinline__ explicit Split4(const uint32_t (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) split(__uint_as_float(x[e]), hi[e], lo[e]);
  }
};
struct Split2 {
  uint32_t hi[2], lo[2];
  __device__ __forceinline__ Split2(float a, float b) {
    split(a, hi[0], lo[0]);
    split(b, hi[1], lo[1]);
  }
};
__device__ __forceinline__ void mma_3tf32(float (&d)[4], const Split4& a, const Split2& b) {
  float t[4];                          // from zero: the tensor core's own additions truncate, so they are kept short
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(t[0]), "=f"(t[1]), "=f"(t[2]), "=f"(t[3])
      : "r"(a.lo[0]), "r"(a.lo[1]), "r"(a.lo[2]), "r"(a.lo[3]), "r"(b.hi[0]), "r"(b.hi[1]), "f"(0.f));
  mma_tf32(t, a.hi, b.lo[0], b.lo[1]);
  mma_tf32(t, a.hi, b.hi[0], b.hi[1]);
#pragma unroll
  for (int e = 0; e < 4; ++e) d[e] += t[e];
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// NT: columns of 8 query heads. kTma: pages hold whole tiles (page size % 16 == 0), so a tile
// lies in one page; else its rows are gathered one by one.
template <typename T, int NT, bool kTma>
__global__ void __launch_bounds__(kThreads, 8)
    paged_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const Dev p,
               float* __restrict__ part) {
  extern __shared__ uint8_t raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int lane = threadIdx.x, g = lane >> 2, c = lane & 3;
  using R = Ring<T, kTma>;
  constexpr int kStages = R::kStages, kTile = R::kTile, kSide = R::kSide, kPieces = R::kRow / 16;
  const uint32_t ring = smem_u32(sm), bars = ring + kStages * kTile;
  if (lane == 0) {
    if (kTma) {
      tma_prefetch_desc(&tk);
      tma_prefetch_desc(&tv);
    }
    for (int i = 0; i < kStages; ++i) mbar_init(bars + i * 8, 1);
    fence_mbar_init();
  }
  __syncwarp();
  pdl_wait();
  pdl_trigger();
  Item it;
  if (!item_of(p, &it)) {
    if (it.len == 0) write_empty<T>(p, it);
    return;
  }
  const int tiles = (it.k1 - it.k0 + kKeys - 1) / kKeys, per_chunk = it.chunk / kKeys;
  // the page of tile t (kTma: of the tile; else of this lane's key), looked up one tile ahead
  auto page_at = [&](int t) {
    const int key = it.k0 + t * kKeys + (kTma ? 0 : lane & 15);
    if (key >= it.k1) return -1;
    const int x = it.table[key / p.page_size];
    return x < p.pages ? x : -1;           // -1: no page, its tokens are left out
  };
  auto get = [&](int t, int page, int stage) -> uint32_t {   // starts tile t; which of its keys there are
    const uint32_t dst = ring + stage * kTile;
    const int key = it.k0 + t * kKeys;
    const uint32_t bar = bars + stage * 8;
    const int n = it.k1 - key;
    if (kTma) {
      if (lane == 0) {
        if (page >= 0) {
          const int slot = key % p.page_size;
          mbar_arrive_expect_tx(bar, kTile);
#pragma unroll
          for (int x = 0; x < R::kRow / 128; ++x) {
            tma_box(dst + x * kKeys * 128, &tk, bar, x * 128 / sizeof(T), slot, it.kvh, page);
            tma_box(dst + kSide + x * kKeys * 128, &tv, bar, x * 128 / sizeof(T), slot, it.kvh, page);
          }
        } else {
          mbar_arrive(bar);
        }
      }
      return page < 0 ? 0u : n < kKeys ? (1u << n) - 1u : 0xFFFFu;
    }
    // a row a lane: the lower sixteen fetch K, the others V; rows that do not exist become zeros
    const uint32_t valid = __ballot_sync(0xffffffffu, page >= 0) & 0xFFFFu;
    const int row = lane & 15, slot = (key + row) % p.page_size;
    const uint32_t to = dst + (lane >> 4) * kSide + row * (R::kRow + 16);
    if (page < 0) {
      for (int x = 0; x < kPieces; ++x) asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(to + x * 16), "r"(0) : "memory");
      fence_proxy_async_smem();   // a later copy may land here
    }
    if (lane == 0) mbar_arrive_expect_tx(bar, __popc(valid) * 2 * R::kRow);
    __syncwarp();
    if (page >= 0) {
      const T* from = lane < 16 ? static_cast<const T*>(p.k) + page * p.skp + it.kvh * p.skh + slot * p.sks
                                : static_cast<const T*>(p.v) + page * p.svp + it.kvh * p.svh + slot * p.svs;
      bulk_load(to, from, R::kRow, bar);
    }
    return valid;
  };

  constexpr int kPitch = NT == 1 ? 12 : 20;   // fp32 weights, [key][head]: free of bank conflicts
  float* weights = reinterpret_cast<float*>(sm + kStages * kTile + 64);
  uint32_t* queries = reinterpret_cast<uint32_t*>(weights + kKeys * kPitch);
  uint32_t there[kStages];                 // which keys there are of tiles t, t + 1, ...
  int page = page_at(0);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    there[i] = i < tiles ? get(i, page, i) : 0;
    page = page_at(i + 1);
  }
  // Queries as B fragments: column g of each eight (heads past the group are zero). A step
  // is 32 bytes of a row: 16 bf16 or 8 fp32; either way lane c has bytes 4 c and 16 + 4 c.
  // fp32 has them in shared memory.
  constexpr int kSteps = kD * sizeof(T) / 32;
  const uint32_t* q = static_cast<const uint32_t*>(p.q) + (it.b * p.sqb + it.h0 * p.sqh) * sizeof(T) / 4;
  uint32_t qb[NT][sizeof(T) == 2 ? kSteps : 1][2];
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int kk = 0; kk < kSteps; ++kk)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          qb[n][kk][e] = n * 8 + g < it.nh ? q[(n * 8 + g) * p.sqh / 2 + kk * 8 + e * 4 + c] : 0u;
  } else {
#pragma unroll 4
    for (int r = 0; r < NT * 8; ++r)
      *reinterpret_cast<uint4*>(queries + r * kQPitch + lane * 4) =
          r < it.nh ? *reinterpret_cast<const uint4*>(q + r * p.sqh + lane * 4) : make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  // O^T: rows = dims 16 d + g, + 8; columns = heads 8 n + 2 c, + 1, as are m and l (l: this lane's keys)
  float o[kD / 16][NT][4], m[NT][2], l[NT][2];
  auto reset = [&] {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int d = 0; d < kD / 16; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][n][e] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }
  };
  reset();
  int left = per_chunk, chunk = it.c0;
  bool some = false;                       // a token of the chunk has a page; the same in every lane
  uint32_t phase = 0;
  for (int t0 = 0; t0 < tiles; t0 += kStages, phase ^= 1) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
      const int t = t0 + s;
      if (t >= tiles) break;
      constexpr int kAhead = kStages - 1;
      there[kAhead] = t + kAhead < tiles ? get(t + kAhead, page, s == 0 ? kAhead : s - 1) : 0;   // into the stage read last
      page = page_at(t + kAhead + 1);
      const uint32_t live = there[0];
      const uint32_t K = ring + s * kTile, V = K + kSide;
      if (!__all_sync(0xffffffffu, mbar_wait_spin(bars + s * 8, phase, 0x321))) {   // an error flag is up: see the copies out
        for (int x = t; x < min(tiles, t + kStages); ++x) mbar_wait(bars + x % kStages * 8, x / kStages & 1, 0x321);
        return;
      }
      if (kTma && live != 0xFFFFu && live != 0u) {
        // slots past the last token hold whatever was there: zero weights would not silence it
        const int n = __popc(live);
        for (int x = lane; x < kKeys * kPieces; x += 32)
          if (x / kPieces >= n)
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(R::at(V, x / kPieces, x % kPieces)), "r"(0) : "memory");
      }
      __syncwarp();
      some |= live != 0u;
      if (live) {   // the same in every lane
        float sc[NT][4], odd[NT][4];   // bf16: the odd steps apart, which halves the chain of dependent products
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[n][e] = odd[n][e] = 0.f;
        const int kr = lane & 15;                                   // ldmatrix rows: keys 0-7, 8-15, then the next 8 dims
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) {   // ldmatrix moves 8 x 4 fp32 blocks as it moves 8 x 8 bf16 ones
          uint32_t a[4];
          ldsm4(R::at(K, kr, kk * 2 + (lane >> 4)), a);
          if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_bf16(kk & 1 ? odd[n] : sc[n], a, qb[n][kk]);
          } else {
            const Split4 as(a);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint32_t* qr = queries + (n * 8 + g) * kQPitch + kk * 8 + c;
              mma_3tf32(sc[n], as, Split2(__uint_as_float(qr[0]), __uint_as_float(qr[4])));
            }
          }
        }
        uint32_t hi[NT][2], lo[NT][2];   // bf16 weights as B fragments, in two parts
        float alpha[NT][2];
        bool same = true;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {   // column 2 c + e: this lane has keys g and g + 8
            float& x = sc[n][e];
            float& y = sc[n][2 + e];
            x = (live >> g & 1) ? (x + odd[n][e]) * p.scale2 : -INFINITY;
            y = (live >> (g + 8) & 1) ? (y + odd[n][2 + e]) * p.scale2 : -INFINITY;
            float mx = fmaxf(x, y);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            mx = fmaxf(mx, m[n][e]);
            const float ref = mx == -INFINITY ? 0.f : mx;
            alpha[n][e] = fast_exp2(m[n][e] - ref);
            same &= alpha[n][e] == 1.f;
            m[n][e] = mx;
            x = fast_exp2(x - ref);
            y = fast_exp2(y - ref);
            l[n][e] = fmaf(l[n][e], alpha[n][e], x + y);
          }
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              *reinterpret_cast<float2*>(weights + (g + h * 8) * kPitch + n * 8 + c * 2) = make_float2(sc[n][2 * h], sc[n][2 * h + 1]);
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {   // keys g, then g + 8: rows of an 8 x 8 matrix, turned into columns
              const float x = sc[n][2 * h], y = sc[n][2 * h + 1];
              const uint32_t u = pack_bf16x2(x, y);
              hi[n][h] = transpose8(u);
              lo[n][h] = transpose8(pack_bf16x2(x - __uint_as_float(u << 16), y - __uint_as_float(u & 0xFFFF0000u)));
            }
          }
        }
        if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
          for (int d = 0; d < kD / 16; ++d)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[d][n][e] *= alpha[n][e & 1];
        }
        if constexpr (sizeof(T) == 2) {
          const int vr = (lane & 7) + (lane >> 4) * 8;              // ldmatrix rows: keys 0-7 (dims 0-7, 8-15), keys 8-15
#pragma unroll
          for (int d = 0; d < kD / 16; ++d) {
            uint32_t a[4];
            ldsm4_t(R::at(V, vr, d * 2 + (lane >> 3 & 1)), a);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_bf16(o[d][n], a, hi[n]);
              mma_bf16(o[d][n], a, lo[n]);
            }
          }
        } else {
          // The order of a step's eight keys is free: keys 2 c and 2 c + 1 serve as columns c
          // and c + 4, which reads V without bank conflicts.
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float* w = weights + (j * 8 + c * 2) * kPitch + n * 8 + g;
              const Split2 ws(w[0], w[kPitch]);
#pragma unroll
              for (int d = 0; d < kD / 16; ++d) {
                uint32_t a[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {   // (dim g, key 2c), (g + 8, 2c), (g, 2c + 1), (g + 8, 2c + 1)
                  const int dim = d * 16 + g + (e & 1) * 8;
                  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(a[e]) : "r"(R::at(V, j * 8 + c * 2 + (e >> 1), dim >> 2) + (dim & 3) * 4));
                }
                mma_3tf32(o[d][n], Split4(a), ws);
              }
            }
        }
        __syncwarp();                      // the stage has been read before it is filled again
      }
      if (--left == 0 || t + 1 == tiles) { // the chunk is done
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float sum = l[n][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            const int r = n * 8 + c * 2 + e;
            bool nan = false;
            if (r < it.nh) {
              if (it.chunks == 1) {
                T* dst = out_at<T>(p, it, r) + g;
#pragma unroll
                for (int d = 0; d < kD / 16; ++d)
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    const float y = some ? o[d][n][h * 2 + e] / sum : 0.f;
                    nan |= y != y;
                    if constexpr (sizeof(T) == 2) dst[d * 16 + h * 8] = f32_to_bf16_bits(y);
                    else dst[d * 16 + h * 8] = y;
                  }
              } else {
                float* dst = acc_at(p, part, it, r, chunk) + g;
#pragma unroll
                for (int d = 0; d < kD / 16; ++d)
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    nan |= o[d][n][h * 2 + e] != o[d][n][h * 2 + e];
                    dst[d * 16 + h * 8] = o[d][n][h * 2 + e];
                  }
                if (g == 0) *ml_at(p, part, it, r, chunk) = make_float2(m[n][e], some ? sum : kNothing);
              }
            }
            const unsigned again = __ballot_sync(0xffffffffu, nan);
            if (again) {
              __syncwarp();   // the row's first result is in place before the second
              for (int x = 0; x < 4; ++x)
                if (again & (0x11111111u << x)) redo_row<T>(p, it, part, n * 8 + x * 2 + e, chunk);
            }
          }
        reset();
        left = per_chunk;
        some = false;
        ++chunk;
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) there[i] = there[i + 1];
    }
  }
}

// Block (head, sequence): warp w takes chunks w, w + kJoinWarps, ..., four dims a lane; the
// warps' sums are added in order.
constexpr int kJoinWarps = 8;
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) join_chunks(const Dev p, const float* __restrict__ part) {
  __shared__ float4 accs[kJoinWarps][32];
  __shared__ float sums[kJoinWarps];
  __shared__ bool any[kJoinWarps];
  pdl_wait();
  pdl_trigger();
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int row;
  const int n = chunks_of(length_of(p, b, &row), p.es);
  if (n <= 1) return;   // written by the chunk's own warp
  const int64_t head = (static_cast<int64_t>(b) * p.H + h) * p.splits;
  const float4* acc = reinterpret_cast<const float4*>(part + head * kD) + lane;
  const float2* ml = reinterpret_cast<const float2*>(part + static_cast<int64_t>(p.B) * p.H * p.splits * kD) + head;
  float m = -INFINITY;
  for (int c = lane; c < n; c += 32) m = fmaxf(m, ml[c].x);
  m = warp_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  bool some = false;
#pragma unroll 4
  for (int c = warp; c < n; c += kJoinWarps) {
    const float2 x = ml[c];
    const float4 v = acc[c * (kD / 4)];
    const float f = fast_exp2(x.x - ref);   // 0 for a chunk with nothing in it
    some |= x.y != kNothing;
    a.x = fmaf(f, v.x, a.x);
    a.y = fmaf(f, v.y, a.y);
    a.z = fmaf(f, v.z, a.z);
    a.w = fmaf(f, v.w, a.w);
    l = fmaf(f, x.y, l);
  }
  accs[warp][lane] = a;
  if (lane == 0) {
    sums[warp] = l;
    any[warp] = some;
  }
  __syncthreads();
  if (warp > 0) return;
#pragma unroll
  for (int w = 1; w < kJoinWarps; ++w) {
    const float4 v = accs[w][lane];
    a.x += v.x;
    a.y += v.y;
    a.z += v.z;
    a.w += v.w;
    l += sums[w];
    some |= any[w];
  }
  const float4 y = some ? make_float4(a.x / l, a.y / l, a.z / l, a.w / l) : make_float4(0.f, 0.f, 0.f, 0.f);
  const int64_t at = b * p.sob + h * p.soh + lane * 4;
  if (sizeof(T) == 4) *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = y;
  else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
}

}  // namespace pg

static int paged_max_len(const rb_paged_args* a) {
  const int64_t cap = static_cast<int64_t>(a->width) * a->page_size;
  const int64_t want = a->max_length > 0 && a->max_length < cap ? a->max_length : cap;
  return static_cast<int>(want);
}

static int paged_validate(const rb_paged_args* a) {
  if (!a || a->B < 0 || a->H <= 0 || a->HK <= 0 || a->pages < 0 || a->page_size <= 0 || a->width < 0 || a->rows < 0 ||
      a->ahead < 0 || a->ld_table < a->width)
    return RB_ERR_INVALID_ARG;
  if ((a->dtype != RB_BF16 && a->dtype != RB_F32) || a->D != pg::kD || a->H % a->HK != 0) return RB_ERR_UNSUPPORTED;
  if (a->B > 65535 || a->H > 65535 || static_cast<int64_t>(a->width) * a->page_size > (INT64_C(1) << 30)) return RB_ERR_CAPACITY;
  if (a->B == 0) return RB_OK;
  if (!a->q || !a->out || (a->rows > 0 && (!a->lengths || (a->width > 0 && !a->table))) || (a->pages > 0 && (!a->k || !a->v)))
    return RB_ERR_INVALID_ARG;
  const int es = a->dtype == RB_BF16 ? 2 : 4;
  for (int64_t s : {a->sqb, a->sqh, a->skp, a->skh, a->sks, a->svp, a->svh, a->svs, a->sob, a->soh})
    if (s * es % 16 != 0) return RB_ERR_UNSUPPORTED;
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out)) return RB_ERR_UNSUPPORTED;
  if (!(a->sm_scale == a->sm_scale)) return RB_ERR_INVALID_ARG;
  return RB_OK;
}

// [pages, HK, page_size, 128] in boxes of 128 bytes of one tile's rows.
static int page_map(CUtensorMap* m, const void* base, const rb_paged_args* a, int64_t slot, int64_t head, int64_t page) {
  const uint32_t es = a->dtype == RB_BF16 ? 2 : 4;
  // a dimension of one entry may have any stride: give the map a plain one
  const uint64_t dims[4] = {pg::kD, static_cast<uint64_t>(a->page_size), static_cast<uint64_t>(a->HK), static_cast<uint64_t>(a->pages)};
  const uint64_t strides[3] = {static_cast<uint64_t>(slot) * es, static_cast<uint64_t>(a->HK > 1 ? head : 8) * es,
                               static_cast<uint64_t>(a->pages > 1 ? page : 8) * es};
  const uint32_t box[4] = {128 / es, pg::kKeys, 1, 1};
  return encode_tiled(m, es == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, base, dims, strides, box,
                      CU_TENSOR_MAP_SWIZZLE_128B);
}

size_t paged_workspace(const rb_paged_args* a) {
  if (paged_validate(a) != RB_OK || a->B == 0) return 0;
  const int splits = pg::max_chunks(paged_max_len(a), a->dtype == RB_BF16 ? 2 : 4);
  return splits > 1 ? static_cast<size_t>(a->B) * a->H * splits * (pg::kD + 2) * sizeof(float) : 0;
}

int paged_launch(const rb_paged_args* a, void* ws, size_t ws_bytes, cudaStream_t st) {
  using namespace pg;
  int r = paged_validate(a);
  if (r != RB_OK || a->B == 0) return r;
  const size_t need = paged_workspace(a);
  if (need > 0 && (!ws || ws_bytes < need || !aligned16(ws))) return RB_ERR_WORKSPACE;
  Dev p{};
  p.q = a->q; p.sqb = a->sqb; p.sqh = a->sqh;
  p.k = a->k; p.skp = a->skp; p.skh = a->skh; p.sks = a->sks;
  p.v = a->v; p.svp = a->svp; p.svh = a->svh; p.svs = a->svs;
  p.table = a->table; p.lengths = a->lengths; p.seqs = a->seqs; p.ld_table = a->ld_table;
  p.B = a->B; p.H = a->H; p.HK = a->HK; p.pages = a->pages; p.page_size = a->page_size; p.width = a->width;
  p.rows = a->rows; p.ahead = a->ahead; p.max_len = paged_max_len(a);
  p.es = a->dtype == RB_BF16 ? 2 : 4;
  p.splits = max_chunks(p.max_len, p.es);
  p.out = a->out; p.sob = a->sob; p.soh = a->soh;
  p.scale2 = a->sm_scale * 1.4426950408889634f;
  float* part = static_cast<float*>(ws);
  const int tiles = (a->H / a->HK + kRows - 1) / kRows;
  // A warp takes one chunk while that leaves no more than about four rounds of warps, and
  // up to eight so that the ring's start is paid less often. No result depends on it.
  const int64_t chunks = static_cast<int64_t>(p.splits) * a->HK * tiles * a->B;
  const int64_t rounds = chunks / (static_cast<int64_t>(device_sm_count()) * 8 * 4);
  p.per_warp = static_cast<int>(rounds < 1 ? 1 : rounds > 8 ? 8 : rounds);
  const dim3 grid((p.splits + p.per_warp - 1) / p.per_warp, a->HK * tiles, a->B);
  CUtensorMap tk{}, tv{};
  // rows are gathered one by one where a tile may cross pages or a map cannot say the layout
  const bool tma = a->page_size % kKeys == 0 && a->pages > 0 && page_map(&tk, a->k, a, a->sks, a->skh, a->skp) == RB_OK &&
                   page_map(&tv, a->v, a, a->svs, a->svh, a->svp) == RB_OK;
  auto go = [&](auto kern, int smem) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return static_cast<int>(RB_ERR_CUDA);
    return launch_k(kern, grid, dim3(kThreads), smem, st, true, tk, tv, p, part);
  };
  const bool bf = a->dtype == RB_BF16, one = a->H / a->HK <= 8;
  auto both = [&](auto zero, auto nt) {
    using T = decltype(zero);
    constexpr int NT = decltype(nt)::value;
    return tma ? go(paged_kernel<T, NT, true>, Ring<T, true>::smem(NT)) : go(paged_kernel<T, NT, false>, Ring<T, false>::smem(NT));
  };
  const std::integral_constant<int, 1> nt1{};
  const std::integral_constant<int, 2> nt2{};
  r = bf ? (one ? both(uint16_t(0), nt1) : both(uint16_t(0), nt2)) : (one ? both(0.f, nt1) : both(0.f, nt2));
  if (r != RB_OK || p.splits == 1) return r;
  return launch_k(bf ? join_chunks<uint16_t> : join_chunks<float>, dim3(a->H, a->B), dim3(32 * kJoinWarps), 0, st, true, p,
                  static_cast<const float*>(part));
}

}  // namespace rb
