// Attention of one new token per sequence over a paged KV cache.
//
//   out[b, h] = sum_t softmax_t(q[b, h] . k_t * scale) v_t,   t < length of sequence b
//
// Bound: every cached K and V row is read once from HBM for all heads of its group
// (4 D flops per 2 D elements and query head: far below the tensor ridge). So the
// work is cut along the length into chunks (one block each, a warp every kWarps-th
// tile of 16 keys), each warp keeps its own ring of asynchronous copies in flight,
// and a second kernel joins the chunks' (accumulator, max, sum) in chunk order.
// Chunks are at absolute positions and their size depends on the sequence's own
// length only, so a sequence gives the same bits alone or in any batch.
//
// bf16: S and P V on m16n8k16 tiles, 16 query heads of the group per tile; P enters
// P V as two bf16 parts (hi + lo), so a weight is good to 2^-16 and the result is
// rounded once, at the end. fp32: fp32 multiply-adds on the CUDA cores (they keep
// pace with HBM for a group of 16).
#include "common.cuh"
#include "host_util.h"

namespace rb {
namespace pg {

constexpr int kD = 128;
constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kKeys = 16;                  // keys of a tile
constexpr int kStages = 3;
constexpr int kRows = 16;                  // query heads of a block
constexpr int kMinChunk = 128, kMaxChunk = 2048, kSplits = 64;
constexpr int kPart = kD + 4;              // acc[128], max (log2 domain), sum, 2 pad

// Keys per chunk of a sequence of `len` tokens: a power of two that gives about
// kSplits chunks.
__host__ __device__ inline int chunk_of(int len) {
  int c = kMinChunk;
  while (c < kMaxChunk && c * kSplits < len) c *= 2;
  return c;
}
__host__ __device__ inline int chunks_of(int len) {
  const int c = chunk_of(len);
  return len / c + (len % c != 0);
}
// Upper bound of chunks_of over every length up to `len`.
__host__ inline int max_chunks(int len) {
  const int a = len / kMinChunk + (len % kMinChunk != 0), b = len / kMaxChunk + (len % kMaxChunk != 0);
  return a < kSplits ? (a > 0 ? a : 1) : (b > kSplits ? b : kSplits);
}

struct Dev {
  const void* q;
  int64_t sqb, sqh;
  const void *k, *v;
  int64_t skp, skh, sks, svp, svh, svs;   // strides of pages, heads, slots (elements)
  const int32_t *table, *lengths, *seqs;
  int64_t ld_table;
  int B, H, HK, pages, page_size, width, rows, ahead, max_len, splits;
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

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {   // bytes < 16: zero fill
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

// What every block starts with: its sequence, chunk and pages.
struct Item {
  int b, kvh, h0, nh;        // batch entry, kv head, first query head and how many
  int len, k0, k1, chunks;   // tokens read, this chunk's keys, chunks of the sequence
  int first;                 // first page of the chunk in the table row
};
__device__ __forceinline__ bool item_of(const Dev& p, int* pages, Item* it) {
  const int G = p.H / p.HK, tiles = (G + kRows - 1) / kRows;
  it->b = blockIdx.z;
  it->kvh = blockIdx.y / tiles;
  const int g0 = blockIdx.y % tiles * kRows;
  it->h0 = it->kvh * G + g0;
  it->nh = min(kRows, G - g0);
  int row;
  it->len = length_of(p, it->b, &row);
  const int C = chunk_of(it->len);
  it->chunks = chunks_of(it->len);
  it->k0 = blockIdx.x * C;
  it->k1 = min(it->len, it->k0 + C);
  if (it->k0 >= it->k1) return false;
  it->first = it->k0 / p.page_size;
  const int n = (it->k1 - 1) / p.page_size - it->first + 1;
  const int32_t* t = p.table + row * p.ld_table + it->first;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int x = t[i];
    pages[i] = x >= 0 && x < p.pages ? x : -1;   // no page: its keys are left out
  }
  return true;
}

// Tile t of the chunk: offsets of the row this lane looks after (lane & 15), and
// which of the tile's keys exist.
struct Rows { int64_t k, v; uint32_t valid; };
__device__ __forceinline__ Rows rows_of(const Dev& p, const Item& it, const int* pages, int t) {
  const int key = it.k0 + t * kKeys + (threadIdx.x & 15);
  Rows r{0, 0, 0};
  bool ok = key < it.k1;
  if (ok) {
    const int idx = key / p.page_size, page = pages[idx - it.first];
    const int slot = key - idx * p.page_size;
    ok = page >= 0;
    if (ok) {
      r.k = page * p.skp + slot * p.sks;
      r.v = page * p.svp + slot * p.svs;
    }
  }
  r.valid = __ballot_sync(0xffffffffu, ok) & 0xFFFFu;
  return r;
}

// Copies a tile's K and V rows (RB bytes each) into `dst` (K rows, then V rows; 16-byte
// pieces swizzled by row & 7). Rows that do not exist are zero.
template <int RB>
__device__ __forceinline__ void fetch(const Dev& p, const Item& it, const Rows& r, uint32_t dst, int es) {
  constexpr int P = RB / 16, R = 32 / P;   // pieces of a row, rows of one pass
  const int lane = threadIdx.x & 31, piece = lane % P;
  const uint8_t* k = static_cast<const uint8_t*>(p.k) + it.kvh * p.skh * es + piece * 16;
  const uint8_t* v = static_cast<const uint8_t*>(p.v) + it.kvh * p.svh * es + piece * 16;
#pragma unroll
  for (int i = 0; i < kKeys / R; ++i) {
    const int row = i * R + lane / P;
    const int64_t ko = __shfl_sync(0xffffffffu, r.k, row) * es, vo = __shfl_sync(0xffffffffu, r.v, row) * es;
    const uint32_t n = (r.valid >> row & 1) ? 16u : 0u;
    const uint32_t at = dst + row * RB + ((piece ^ (row & 7)) * 16);
    copy16(at, n ? k + ko : p.q, n);   // a row that does not exist reads nothing
    copy16(at + kKeys * RB, n ? v + vo : p.q, n);
  }
}

// Row r of the chunk again, by one warp and key by key, in place of the warps'
// accumulators (`w`, as finish() reads them). The second part of a weight is often
// zero, which times an infinity in V is a NaN that the product itself is not; a row
// that came out NaN is settled here.
__device__ __noinline__ void redo_bf16(const Dev& p, const Item& it, const int* pages, float* w, int r) {
  const int lane = threadIdx.x & 31, d = lane * 4;
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    q[e] = bf16_bits_to_f32(static_cast<const uint16_t*>(p.q)[it.b * p.sqb + (it.h0 + r) * p.sqh + d + e]);
  for (int key = it.k0; key < it.k1; ++key) {
    const int page = pages[key / p.page_size - it.first], slot = key % p.page_size;
    if (page < 0) continue;
    const uint16_t* k = static_cast<const uint16_t*>(p.k) + page * p.skp + it.kvh * p.skh + slot * p.sks + d;
    const uint16_t* v = static_cast<const uint16_t*>(p.v) + page * p.svp + it.kvh * p.svh + slot * p.svs + d;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fmaf(q[e], bf16_bits_to_f32(k[e]), s);
    s = warp_sum(s) * p.scale2;
    const float mx = fmaxf(m, s), ref = mx == -INFINITY ? 0.f : mx;
    const float a = fast_exp2(m - ref), x = fast_exp2(s - ref);
    m = mx;
    l = fmaf(l, a, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = a == 0.f ? x * bf16_bits_to_f32(v[e]) : fmaf(o[e], a, x * bf16_bits_to_f32(v[e]));
  }
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    float* row = w + (i * kRows + r) * kPart;
    *reinterpret_cast<float4*>(row + d) = i == 0 ? make_float4(o[0], o[1], o[2], o[3]) : make_float4(0.f, 0.f, 0.f, 0.f);
    if (lane == 0) *reinterpret_cast<float2*>(row + kD) = i == 0 ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
  }
}

// Joins the warps' accumulators (`w`: [kWarps][kRows][kPart] floats) of the block's
// heads in warp order and writes the chunk's partial, or the result when the
// sequence has one chunk.
template <typename T>
__device__ __forceinline__ void finish(const Dev& p, const Item& it, const float* w, float* part) {
  const int d = threadIdx.x;   // kThreads == kD
  for (int r = 0; r < it.nh; ++r) {
    float m = -INFINITY;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) m = fmaxf(m, w[(x * kRows + r) * kPart + kD]);
    float acc = 0.f, l = 0.f;
    if (m != -INFINITY) {
#pragma unroll
      for (int x = 0; x < kWarps; ++x) {
        const float* s = w + (x * kRows + r) * kPart;
        const float f = fast_exp2(s[kD] - m);
        acc = fmaf(f, s[d], acc);
        l = fmaf(f, s[kD + 1], l);
      }
    }
    const int h = it.h0 + r;
    if (it.chunks == 1) {
      const float o = l > 0.f || l != l ? acc / l : 0.f;
      const int64_t at = it.b * p.sob + h * p.soh + d;
      if (sizeof(T) == 4) static_cast<float*>(p.out)[at] = o;
      else static_cast<uint16_t*>(p.out)[at] = f32_to_bf16_bits(o);
    } else {
      float* dst = part + ((static_cast<int64_t>(it.b) * p.H + h) * p.splits + blockIdx.x) * kPart;
      dst[d] = acc;
      if (d == 0) *reinterpret_cast<float2*>(dst + kD) = make_float2(m, l);
    }
  }
}
template <typename T>
__device__ __forceinline__ void write_empty(const Dev& p, const Item& it) {
  if (blockIdx.x != 0) return;
  for (int r = 0; r < it.nh; ++r) {
    const int64_t at = it.b * p.sob + (it.h0 + r) * p.soh + threadIdx.x;
    if (sizeof(T) == 4) static_cast<float*>(p.out)[at] = 0.f;
    else static_cast<uint16_t*>(p.out)[at] = 0;
  }
}

constexpr int kTileBytes16 = 2 * kKeys * kD * 2, kTileBytes32 = 2 * kKeys * kD * 4;
// rings | page numbers of the chunk | (fp32: queries and weights)
constexpr int smem16() { return kWarps * kStages * kTileBytes16 + (kMaxChunk + 2) * 4; }
constexpr int smem32() { return kWarps * kStages * kTileBytes32 + (kMaxChunk + 2) * 4 + kRows * kD * 4 + kWarps * kKeys * kRows * 4 + 16; }
static_assert(kWarps * kStages * kTileBytes16 >= kWarps * kRows * kPart * 4 + 4, "the join reuses the rings");
static_assert(smem32() <= 232448, "shared memory budget");
static_assert(kThreads == kD, "finish() gives a thread one dim");

__global__ void __launch_bounds__(kThreads) paged_bf16(const Dev p, float* __restrict__ part) {
  extern __shared__ __align__(128) uint8_t sm[];
  int* pages = reinterpret_cast<int*>(sm + kWarps * kStages * kTileBytes16);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  pdl_wait();
  pdl_trigger();
  Item it;
  if (!item_of(p, pages, &it)) {
    if (it.len == 0) write_empty<uint16_t>(p, it);
    return;
  }
  __syncthreads();
  const int tiles = (it.k1 - it.k0 + kKeys - 1) / kKeys;
  const uint32_t ring = smem_u32(sm) + warp * kStages * kTileBytes16;
  uint32_t valid[kStages];
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    const int t = warp + s * kWarps;
    valid[s] = 0;
    if (t < tiles) {
      const Rows r = rows_of(p, it, pages, t);
      valid[s] = r.valid;
      fetch<kD * 2>(p, it, r, ring + s * kTileBytes16, 2);
    }
    copy_commit();
  }
  // queries as A fragments: rows g, g + 8 (heads past the group are zero)
  uint32_t qa[kD / 16][4];
  {
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + it.b * p.sqb + it.h0 * p.sqh;
#pragma unroll
    for (int kk = 0; kk < kD / 16; ++kk)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = g + (e & 1) * 8;
        qa[kk][e] = r < it.nh ? *reinterpret_cast<const uint32_t*>(q + r * p.sqh + kk * 16 + (e >> 1) * 8 + c * 2) : 0u;
      }
  }
  float o[kD / 8][4];
#pragma unroll
  for (int n = 0; n < kD / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  for (int t0 = warp; t0 < tiles; t0 += kWarps * kStages) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
      const int t = t0 + s * kWarps;
      if (t >= tiles) break;
      {   // the tile kStages - 1 steps ahead, into the stage read last
        constexpr int kAhead = kStages - 1;
        const int tn = t + kAhead * kWarps, sn = (s + kAhead) % kStages;
        valid[sn] = 0;
        if (tn < tiles) {
          const Rows r = rows_of(p, it, pages, tn);
          valid[sn] = r.valid;
          fetch<kD * 2>(p, it, r, ring + sn * kTileBytes16, 2);
        }
        copy_commit();
      }
      copy_wait<kStages - 1>();
      __syncwarp();
      const uint32_t K = ring + s * kTileBytes16, V = K + kKeys * kD * 2;
      // S: two 8-key tiles; ldmatrix matrices = (keys 0-7, 8-15) x (k halves)
      float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      const int kr = (lane & 7) + (lane >> 4) * 8;
#pragma unroll
      for (int kk = 0; kk < kD / 16; ++kk) {
        uint32_t kb[4];
        ldsm4(K + kr * (kD * 2) + (((kk * 2 + (lane >> 3 & 1)) ^ (kr & 7)) * 16), kb);
        mma_bf16_16816(sc[0], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], kb[0], kb[1]);
        mma_bf16_16816(sc[1], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], kb[2], kb[3]);
      }
      float alpha[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {   // rows g and g + 8
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = sc[j][h * 2 + e];
            x = (valid[s] >> (j * 8 + c * 2 + e) & 1) ? x * p.scale2 : -INFINITY;
            mx = fmaxf(mx, x);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        mx = fmaxf(mx, m[h]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        alpha[h] = fast_exp2(m[h] - ref);
        m[h] = mx;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = sc[j][h * 2 + e];
            x = fast_exp2(x - ref);
            sum += x;
          }
        l[h] = fmaf(l[h], alpha[h], sum);
      }
      if (!__all_sync(0xffffffffu, alpha[0] == 1.f && alpha[1] == 1.f)) {
#pragma unroll
        for (int n = 0; n < kD / 8; ++n) {
          o[n][0] *= alpha[0];
          o[n][1] *= alpha[0];
          o[n][2] *= alpha[1];
          o[n][3] *= alpha[1];
        }
      }
      // P as A fragments, in two parts
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = sc[e >> 1][(e & 1) * 2], b = sc[e >> 1][(e & 1) * 2 + 1];
        hi[e] = pack_bf16x2(a, b);
        lo[e] = pack_bf16x2(a - __uint_as_float(hi[e] << 16), b - __uint_as_float(hi[e] & 0xFFFF0000u));
      }
      const int vr = lane & 15;
#pragma unroll
      for (int n = 0; n < kD / 16; ++n) {
        uint32_t vb[4];
        ldsm4_t(V + vr * (kD * 2) + (((n * 2 + (lane >> 4)) ^ (vr & 7)) * 16), vb);
        mma_bf16_16816(o[2 * n], hi[0], hi[1], hi[2], hi[3], vb[0], vb[1]);
        mma_bf16_16816(o[2 * n], lo[0], lo[1], lo[2], lo[3], vb[0], vb[1]);
        mma_bf16_16816(o[2 * n + 1], hi[0], hi[1], hi[2], hi[3], vb[2], vb[3]);
        mma_bf16_16816(o[2 * n + 1], lo[0], lo[1], lo[2], lo[3], vb[2], vb[3]);
      }
      __syncwarp();   // the stage has been read before it is filled again
    }
  }
  copy_wait<0>();
  __syncthreads();    // every warp is done with its ring
  uint32_t nan = 0;   // rows with a NaN
  float* w = reinterpret_cast<float*>(sm) + warp * kRows * kPart;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float s = l[h];
    s += __shfl_xor_sync(0xffffffffu, s, 1);
    s += __shfl_xor_sync(0xffffffffu, s, 2);
    float* row = w + (g + h * 8) * kPart;
    if (c == 0) *reinterpret_cast<float2*>(row + kD) = make_float2(m[h], s);
#pragma unroll
    for (int n = 0; n < kD / 8; ++n) {
      *reinterpret_cast<float2*>(row + n * 8 + c * 2) = make_float2(o[n][h * 2], o[n][h * 2 + 1]);
      if (o[n][h * 2] != o[n][h * 2] || o[n][h * 2 + 1] != o[n][h * 2 + 1]) nan |= 1u << (g + h * 8);
    }
  }
  if (__syncthreads_or(nan & ((1u << it.nh) - 1u))) {   // kRows <= 16 heads
    uint32_t* again = reinterpret_cast<uint32_t*>(sm) + kWarps * kRows * kPart;
    if (threadIdx.x == 0) *again = 0;
    __syncthreads();
    if (nan) atomicOr(again, nan);
    __syncthreads();
    const uint32_t rows = *again;
    for (int r = warp; r < it.nh; r += kWarps)
      if (rows >> r & 1) redo_bf16(p, it, pages, reinterpret_cast<float*>(sm), r);
  }
  __syncthreads();
  finish<uint16_t>(p, it, reinterpret_cast<const float*>(sm), part);
}

// fp32: a lane holds one key (lane & 15) and half of the dims while scores are made,
// four dims of every head while P V is.
__global__ void __launch_bounds__(kThreads) paged_f32(const Dev p, float* __restrict__ part) {
  extern __shared__ __align__(128) uint8_t sm[];
  int* pages = reinterpret_cast<int*>(sm + kWarps * kStages * kTileBytes32);
  float* qs = reinterpret_cast<float*>(sm + kWarps * kStages * kTileBytes32 + ((kMaxChunk + 2) * 4 + 15) / 16 * 16);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* ps = qs + kRows * kD + warp * kKeys * kRows;   // weights of a tile, [key][head]
  pdl_wait();
  pdl_trigger();
  Item it;
  if (!item_of(p, pages, &it)) {
    if (it.len == 0) write_empty<float>(p, it);
    return;
  }
  const float* q = static_cast<const float*>(p.q) + it.b * p.sqb + it.h0 * p.sqh;
  for (int r = 0; r < kRows; ++r) qs[r * kD + threadIdx.x] = r < it.nh ? q[r * p.sqh + threadIdx.x] : 0.f;
  __syncthreads();
  const int tiles = (it.k1 - it.k0 + kKeys - 1) / kKeys;
  const uint32_t ring = smem_u32(sm) + warp * kStages * kTileBytes32;
  const uint8_t* ring_p = sm + warp * kStages * kTileBytes32;
  uint32_t valid[kStages];
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    const int t = warp + s * kWarps;
    valid[s] = 0;
    if (t < tiles) {
      const Rows r = rows_of(p, it, pages, t);
      valid[s] = r.valid;
      fetch<kD * 4>(p, it, r, ring + s * kTileBytes32, 4);
    }
    copy_commit();
  }
  float o[kRows][4], m[kRows], l[kRows];   // l: this lane's keys only
#pragma unroll
  for (int h = 0; h < kRows; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[h][e] = 0.f;
  }
  const int key = lane & 15, half = lane >> 4;
  for (int t0 = warp; t0 < tiles; t0 += kWarps * kStages) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
      const int t = t0 + s * kWarps;
      if (t >= tiles) break;
      {
        constexpr int kAhead = kStages - 1;
        const int tn = t + kAhead * kWarps, sn = (s + kAhead) % kStages;
        valid[sn] = 0;
        if (tn < tiles) {
          const Rows r = rows_of(p, it, pages, tn);
          valid[sn] = r.valid;
          fetch<kD * 4>(p, it, r, ring + sn * kTileBytes32, 4);
        }
        copy_commit();
      }
      copy_wait<kStages - 1>();
      __syncwarp();
      const uint8_t* K = ring_p + s * kTileBytes32;
      const uint8_t* V = K + kKeys * kD * 4;
      float sc[kRows];
#pragma unroll
      for (int h = 0; h < kRows; ++h) sc[h] = 0.f;
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {   // this half's 64 dims
        const int piece = half * 16 + i;
        const float4 k = *reinterpret_cast<const float4*>(K + key * (kD * 4) + ((piece ^ (key & 7)) * 16));
#pragma unroll
        for (int h = 0; h < kRows; ++h) {
          if (h >= it.nh) break;
          const float4 x = *reinterpret_cast<const float4*>(qs + h * kD + piece * 4);
          sc[h] = fmaf(x.x, k.x, fmaf(x.y, k.y, fmaf(x.z, k.z, fmaf(x.w, k.w, sc[h]))));
        }
      }
      const bool ok = valid[s] >> key & 1;
#pragma unroll
      for (int h = 0; h < kRows; ++h) {
        if (h >= it.nh) break;
        float x = (sc[h] + __shfl_xor_sync(0xffffffffu, sc[h], 16)) * p.scale2;
        x = ok ? x : -INFINITY;
        float mx = x;
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        mx = fmaxf(mx, m[h]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        const float a = fast_exp2(m[h] - ref), w = fast_exp2(x - ref);
        m[h] = mx;
        l[h] = fmaf(l[h], a, w);
        if (half == 0) ps[key * kRows + h] = w;
        if (a != 1.f) {   // the same in every lane
#pragma unroll
          for (int e = 0; e < 4; ++e) o[h][e] *= a;
        }
      }
      __syncwarp();
#pragma unroll 4
      for (int j = 0; j < kKeys; ++j) {
        const float4 v = *reinterpret_cast<const float4*>(V + j * (kD * 4) + ((lane ^ (j & 7)) * 16));
#pragma unroll
        for (int h = 0; h < kRows; ++h) {
          if (h >= it.nh) break;
          const float w = ps[j * kRows + h];
          o[h][0] = fmaf(w, v.x, o[h][0]);
          o[h][1] = fmaf(w, v.y, o[h][1]);
          o[h][2] = fmaf(w, v.z, o[h][2]);
          o[h][3] = fmaf(w, v.w, o[h][3]);
        }
      }
      __syncwarp();
    }
  }
  copy_wait<0>();
  __syncthreads();
  float* w = reinterpret_cast<float*>(sm) + warp * kRows * kPart;
#pragma unroll
  for (int h = 0; h < kRows; ++h) {
    if (h >= it.nh) break;
    float s = l[h];   // both halves hold the same 16 keys
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    *reinterpret_cast<float4*>(w + h * kPart + lane * 4) = make_float4(o[h][0], o[h][1], o[h][2], o[h][3]);
    if (lane == 0) *reinterpret_cast<float2*>(w + h * kPart + kD) = make_float2(m[h], s);
  }
  __syncthreads();
  finish<float>(p, it, reinterpret_cast<const float*>(sm), part);
}

// Block (head, sequence), thread = dim: the chunks' partials in chunk order.
template <typename T>
__global__ void __launch_bounds__(kD) join_chunks(const Dev p, const float* __restrict__ part) {
  __shared__ float wsum[kD / 32];
  pdl_wait();
  pdl_trigger();
  const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  int row;
  const int n = chunks_of(length_of(p, b, &row));
  if (n <= 1) return;   // written by the chunk's own block
  const float* src = part + (static_cast<int64_t>(b) * p.H + h) * p.splits * kPart;
  float m = -INFINITY;
  for (int c = d; c < n; c += kD) m = fmaxf(m, src[c * kPart + kD]);
  m = warp_max(m);
  if ((d & 31) == 0) wsum[d >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kD / 32; ++w) m = fmaxf(m, wsum[w]);
  float acc = 0.f, l = 0.f;
  if (m != -INFINITY) {
#pragma unroll 8
    for (int c = 0; c < n; ++c) {
      const float2 ml = *reinterpret_cast<const float2*>(src + c * kPart + kD);
      const float f = fast_exp2(ml.x - m);
      acc = fmaf(f, src[c * kPart + d], acc);
      l = fmaf(f, ml.y, l);
    }
  }
  const float o = l > 0.f || l != l ? acc / l : 0.f;
  const int64_t at = b * p.sob + h * p.soh + d;
  if (sizeof(T) == 4) static_cast<float*>(p.out)[at] = o;
  else static_cast<uint16_t*>(p.out)[at] = f32_to_bf16_bits(o);
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
  if (!a->q || !a->out || !a->lengths || (a->width > 0 && !a->table) || (a->pages > 0 && (!a->k || !a->v)))
    return RB_ERR_INVALID_ARG;
  const int es = a->dtype == RB_BF16 ? 2 : 4;
  for (int64_t s : {a->sqb, a->sqh, a->skp, a->skh, a->sks, a->svp, a->svh, a->svs, a->sob, a->soh})
    if (s * es % 16 != 0) return RB_ERR_UNSUPPORTED;
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out)) return RB_ERR_UNSUPPORTED;
  if (!(a->sm_scale == a->sm_scale)) return RB_ERR_INVALID_ARG;
  return RB_OK;
}

size_t paged_workspace(const rb_paged_args* a) {
  if (paged_validate(a) != RB_OK || a->B == 0) return 0;
  const int splits = pg::max_chunks(paged_max_len(a));
  return splits > 1 ? static_cast<size_t>(a->B) * a->H * splits * pg::kPart * sizeof(float) : 0;
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
  p.rows = a->rows; p.ahead = a->ahead; p.max_len = paged_max_len(a); p.splits = max_chunks(p.max_len);
  p.out = a->out; p.sob = a->sob; p.soh = a->soh;
  p.scale2 = a->sm_scale * 1.4426950408889634f;
  float* part = static_cast<float*>(ws);
  const int tiles = (a->H / a->HK + kRows - 1) / kRows;
  const dim3 grid(p.splits, a->HK * tiles, a->B);
  const bool bf = a->dtype == RB_BF16;
  const int smem = bf ? smem16() : smem32();
  if (cudaFuncSetAttribute(bf ? paged_bf16 : paged_f32, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return RB_ERR_CUDA;
  r = launch_k(bf ? paged_bf16 : paged_f32, grid, dim3(kThreads), smem, st, true, p, part);
  if (r != RB_OK || p.splits == 1) return r;
  return launch_k(bf ? join_chunks<uint16_t> : join_chunks<float>, dim3(a->H, a->B), dim3(kD), 0, st, true, p,
                  static_cast<const float*>(part));
}

}  // namespace rb
