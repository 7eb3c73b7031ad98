// Causal grouped-query attention over whole packed prompts.
//
//   out_i = sum_{j <= i} softmax_j(q_i . k_j * scale) v_j   within each sequence
//
// A tile is TP = rows / G tokens x the G query heads of one kv head (row r = token
// r / G, head r % G), so a group's heads share every K / V tile and short prompts
// fill the rows. Keys are taken in tiles at absolute positions of the sequence, in
// ascending order; a tile that lies wholly after a row's token changes nothing of
// that row. A row's bits therefore depend on its own sequence alone, not on the
// packing or on which tile it falls into.
#include "common.cuh"
#include "host_util.h"

namespace rb {
namespace pr {

constexpr int kD = 128;

struct Dev {
  const void *q, *k, *v;
  int64_t sqt, sqh, skt, skh, svt, svh;   // strides of tokens and heads (elements)
  const int32_t* cu;
  int B, T, H, HK;
  void* out;
  int64_t sot, soh;
  float scale2;                            // sm_scale * log2 e
  int wide;                                // tiles of a band: about as many as run at a time
  int zero_rest;                           // rows of no sequence: zeros (else left alone)
};

__device__ __forceinline__ int start_of(const Dev& p, int i) { return min(max(p.cu[i], 0), p.T); }
__device__ __forceinline__ int length_of(const Dev& p, int i) { return max(start_of(p, i + 1) - start_of(p, i), 0); }

// The rank-th tile of tp tokens. Tiles are ordered by the band of `wide` tiles they lie
// in, the later band first, then by sequence, then the later tile first: work falls
// from the first rank to the last, and tiles that run at the same time read the same
// K / V. Warp-wide, the same in every lane; false when there are fewer tiles.
__device__ __forceinline__ bool find_tile(const Dev& p, int tp, int wide, int rank, int* seq, int* tile) {
  const int lane = threadIdx.x & 31;
  int tiles0 = 0, most = 0;   // this lane's first sequence is looked at often
  if (lane < p.B) tiles0 = (length_of(p, lane) + tp - 1) / tp;
  for (int i = lane; i < p.B; i += 32) most = max(most, i == lane ? tiles0 : (length_of(p, i) + tp - 1) / tp);
  most = (__reduce_max_sync(0xffffffffu, most) + wide - 1) / wide;   // bands
  auto from = [&](int band) {                                        // tiles in it and in later ones
    int n = max(tiles0 - band * wide, 0);
    for (int i = lane + 32; i < p.B; i += 32) n += max((length_of(p, i) + tp - 1) / tp - band * wide, 0);
    return __reduce_add_sync(0xffffffffu, n);
  };
  if (from(0) <= rank) return false;
  int lo = 0, hi = most;      // from(lo) > rank >= from(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (from(mid) > rank) lo = mid; else hi = mid;
  }
  int left = rank - from(lo + 1);   // within the band
  for (int base = 0; base < p.B; base += 32) {
    const int i = base + lane;
    const int n = base == 0 ? tiles0 : i < p.B ? (length_of(p, i) + tp - 1) / tp : 0;
    const int here = min(max(n - lo * wide, 0), wide);
    int sum = here;           // inclusive prefix sum
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, sum > left);
    if (past) {
      const int l = __ffs(past) - 1;
      *seq = base + l;
      *tile = lo * wide + __shfl_sync(0xffffffffu, sum, l) - 1 - left;
      return true;
    }
    left -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}

// Rows before cu[0] and from cu[B] on belong to no sequence.
template <typename T>
__device__ __forceinline__ void zero_rest(const Dev& p, int threads) {   // the block's first `threads` threads
  const int a = start_of(p, 0), b = max(start_of(p, p.B), a);
  const int64_t n = static_cast<int64_t>(a + (p.T - b)) * p.H * kD;
  for (int64_t x = static_cast<int64_t>(blockIdx.x) * threads + threadIdx.x; x < n;
       x += static_cast<int64_t>(gridDim.x) * threads) {
    int64_t t = x / (p.H * kD);
    if (t >= a) t += b - a;
    const int h = static_cast<int>(x / kD % p.H), d = static_cast<int>(x % kD);
    static_cast<T*>(p.out)[t * p.sot + h * p.soh + d] = T(0);
  }
}

// ---------------------------------------------------------------- fp32
// Tensor cores with every operand in two tf32 parts (hi hi + hi lo + lo hi: good to
// about 2^-22 of a product). Four warps of 16 rows; K / V tiles of 32 keys arrive by
// cp.async one tile ahead. Each step of eight starts from zero and is added to the
// running sum in fp32, so that sum rounds to nearest however long it gets.
//
// A row that comes out NaN is looked at again at the end (settle_rows).
//
// Bound: mma.sync, whose pipe is half busy (as are the issue slots: about eight instructions
// an MMA, two warps a scheduler). Measured: 2,570 tokens of five prompts, 28 / 4 heads, 504 us
// = 42 TFLOP/s, three tf32 products each (with the conversion instruction in split() 597).
namespace f32 {
constexpr int kWarps = 4, kThreads = 32 * kWarps, kRows = 16 * kWarps, kKeys = 32;
constexpr int kPitch = kD + 4;   // floats per staged row: fragment reads without bank conflicts
constexpr int kTile = kKeys * kPitch;
constexpr int kSmem = (kRows * kPitch + 4 * kTile) * 4;

// x = hi + lo: hi rounded to tf32's 11 bits by integer arithmetic (the conversion
// instruction is several times slower), lo what is left, which the tensor core cuts to 11
// bits: good to 2^-22 of x. A NaN survives in lo; an infinity gives one.
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(   // not volatile: independent products may pass one another
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {   // from zero
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma3(float (&d)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], float b0, float b1) {
  uint32_t h0, l0, h1, l1;
  split(b0, h0, l0);
  split(b1, h1, l1);
  float t[4];                          // from zero: the tensor core's own additions truncate, so they are kept short
  mma8_zero(t, al, h0, h1);
  mma8(t, ah, l0, l1);
  mma8(t, ah, h0, h1);
#pragma unroll
  for (int e = 0; e < 4; ++e) d[e] += t[e];
}
__device__ __forceinline__ void copy16(float* dst, const float* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}

// The rows of `bad` (bit r: row r came out NaN) again without tensor cores, by the whole block. The
// tiles give a NaN that the definition does not where a masked V row, multiplied by zero, is not
// finite, and where an operand is infinite (in two parts, infinity + NaN) or a score's terms
// overflow. If there is nothing of the kind among what the block's rows read, their NaNs are real.
// Else a row is taken by two threads, 64 dims each, in the order of its keys. Measured (8,000 tokens,
// 4 / 1 heads): 1.38 ms; with a NaN that every row attends to 1.65, with an infinity 4.4.
// Q: the block's queries (staged, with the scale's sign), KV: room for two tiles.
__device__ __noinline__ void settle_rows(const Dev& p, const float* Q, float* KV, int s0, int len, int tok0, int toks, int kvh,
                                         uint64_t bad) {
  const int G = p.H / p.HK, end = tok0 + toks, lane = threadIdx.x & 31;
  const float* kg = static_cast<const float*>(p.k) + static_cast<int64_t>(s0) * p.skt + kvh * p.skh;
  const float* vg = static_cast<const float*>(p.v) + static_cast<int64_t>(s0) * p.svt + kvh * p.svh;
  auto large = [](float4 x) {      // products of two smaller ones cannot overflow in a sum of 128; not NaN
    return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))) >= 1.152921504606846976e18f;
  };
  auto tops = [](float4 x) {       // infinite, or so as its first part
    return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))) >= 3.4e38f;
  };
  bool look = false;
  for (int x = threadIdx.x; x < kRows * 32; x += kThreads) look |= large(*reinterpret_cast<const float4*>(Q + (x >> 5) * kPitch + (x & 31) * 4));
  const int rows = min(static_cast<int64_t>(len), (static_cast<int64_t>(end) + kKeys - 1) / kKeys * kKeys);   // whose V the tiles read
#pragma unroll 4
  for (int r = threadIdx.x >> 5; r < rows; r += kWarps) {
    const float4 v = *reinterpret_cast<const float4*>(vg + r * p.svt + lane * 4);
    look |= tops(v) || (r > tok0 && (v.x != v.x || v.y != v.y || v.z != v.z || v.w != v.w));
    if (r < end) look |= large(*reinterpret_cast<const float4*>(kg + r * p.skt + lane * 4));
  }
  if (!__syncthreads_or(look)) return;
  const int r = threadIdx.x >> 1, half = threadIdx.x & 1, tok = tok0 + r / G;
  const bool mine = bad >> r & 1;
  const float scale2 = fabsf(p.scale2);
  float4 q[kD / 8], o[kD / 8];     // dims 8 i + 4 half
#pragma unroll
  for (int i = 0; i < kD / 8; ++i) {
    q[i] = *reinterpret_cast<const float4*>(Q + r * kPitch + i * 8 + half * 4);
    o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float m = -INFINITY, l = 0.f;
  auto fetch = [&](int t) {
    float* K = KV + (t & 1) * 2 * kTile;
    for (int x = threadIdx.x; x < kKeys * 32; x += kThreads) {
      const int key = t * kKeys + (x >> 5), to = (x >> 5) * kPitch + (x & 31) * 4;
      if (key >= end) break;       // read by nobody
      copy16(K + to, kg + key * p.skt + (x & 31) * 4, 16u);
      copy16(K + kTile + to, vg + key * p.svt + (x & 31) * 4, 16u);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(0);
  for (int t = 0; t * kKeys < end; ++t) {
    __syncthreads();               // the other stage has been read
    fetch(t + 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    // the same keys in every lane of a warp, up to its last row's
    const int keys = __any_sync(0xffffffffu, mine) ? min(kKeys, __shfl_sync(0xffffffffu, tok, 31) + 1 - t * kKeys) : 0;
#pragma unroll 1
    for (int j = 0; j < keys; ++j) {
      const float* k = KV + (t & 1) * 2 * kTile + j * kPitch + half * 4;
      const float* v = k + kTile;
      float4 d = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kD / 8; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(k + i * 8);
        d = make_float4(fmaf(q[i].x, x.x, d.x), fmaf(q[i].y, x.y, d.y), fmaf(q[i].z, x.z, d.z), fmaf(q[i].w, x.w, d.w));
      }
      float s = (d.x + d.y) + (d.z + d.w);
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      if (!mine || t * kKeys + j > tok) continue;
      const float mx = fmaxf(m, s), ref = mx == -INFINITY ? 0.f : mx;
      if (mx != m) {
        const float a = fast_exp2((m - ref) * scale2);
        l *= a;
#pragma unroll
        for (int i = 0; i < kD / 8; ++i) o[i] = make_float4(o[i].x * a, o[i].y * a, o[i].z * a, o[i].w * a);
        m = mx;
      }
      const float w = fast_exp2((s - ref) * scale2);
      l += w;
#pragma unroll
      for (int i = 0; i < kD / 8; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(v + i * 8);
        o[i] = make_float4(fmaf(w, x.x, o[i].x), fmaf(w, x.y, o[i].y), fmaf(w, x.z, o[i].z), fmaf(w, x.w, o[i].w));
      }
    }
  }
  if (!mine) return;
  float* out = static_cast<float*>(p.out) + static_cast<int64_t>(s0 + tok) * p.sot + (kvh * G + r % G) * p.soh + half * 4;
#pragma unroll
  for (int i = 0; i < kD / 8; ++i) *reinterpret_cast<float4*>(out + i * 8) = make_float4(o[i].x / l, o[i].y / l, o[i].z / l, o[i].w / l);
}
}  // namespace f32

__global__ void __launch_bounds__(f32::kThreads, 2) prompt_f32(const Dev p) {
  using namespace f32;
  extern __shared__ __align__(16) float fsm[];
  float* Q = fsm;
  float* KV = fsm + kRows * kPitch;   // two stages of K, V
  __shared__ uint32_t bad[kRows / 32];   // rows that came out NaN
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  pdl_wait();
  pdl_trigger();
  if (p.zero_rest) zero_rest<float>(p, kThreads);
  const int G = p.H / p.HK, TP = kRows / G;
  const int kvh = blockIdx.x % p.HK;
  int seq, tile;
  if (!find_tile(p, TP, p.wide, blockIdx.x / p.HK, &seq, &tile)) return;
  const int s0 = start_of(p, seq), len = length_of(p, seq);
  const int tok0 = tile * TP, toks = min(TP, len - tok0), rows = toks * G;
  const int tiles = (tok0 + toks + kKeys - 1) / kKeys;
  const float* kg = static_cast<const float*>(p.k) + static_cast<int64_t>(s0) * p.skt + kvh * p.skh;
  const float* vg = static_cast<const float*>(p.v) + static_cast<int64_t>(s0) * p.svt + kvh * p.svh;
  auto fetch = [&](int t) {   // rows past the sequence are zero
    float* K = KV + (t & 1) * 2 * kTile;
    for (int x = threadIdx.x; x < kKeys * 32; x += kThreads) {
      const int r = x >> 5, piece = (x & 31) * 4, key = t * kKeys + r;
      const bool ok = key < len;
      copy16(K + r * kPitch + piece, ok ? kg + key * p.skt + piece : kg, ok ? 16u : 0u);
      copy16(K + kTile + r * kPitch + piece, ok ? vg + key * p.svt + piece : vg, ok ? 16u : 0u);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(0);
  if (threadIdx.x < kRows / 32) bad[threadIdx.x] = 0;
  const float* qg = static_cast<const float*>(p.q) + static_cast<int64_t>(s0 + tok0) * p.sqt + kvh * G * p.sqh;
  // a negative scale's sign goes into Q, so that the largest score has the largest weight
  const float scale2 = fabsf(p.scale2), sign = p.scale2 < 0.f ? -1.f : 1.f;
  for (int x = threadIdx.x; x < kRows * 32; x += kThreads) {
    const int r = x >> 5, piece = (x & 31) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < rows) v = *reinterpret_cast<const float4*>(qg + r / G * p.sqt + r % G * p.sqh + piece);
    *reinterpret_cast<float4*>(Q + r * kPitch + piece) = make_float4(v.x * sign, v.y * sign, v.z * sign, v.w * sign);
  }
  float o[kD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < kD / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  const int row0 = warp * 16 + g;
  const int tok[2] = {tok0 + row0 / G, tok0 + (row0 + 8) / G};   // keys <= tok are attended
  for (int t = 0; t < tiles; ++t) {
    __syncthreads();   // the other stage has been read
    if (t + 1 < tiles) fetch(t + 1);
    else asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    const float* K = KV + (t & 1) * 2 * kTile;
    const float* V = K + kTile;
    float sc[kKeys / 8][4];
#pragma unroll
    for (int j = 0; j < kKeys / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[j][e] = 0.f;
#pragma unroll 4
    for (int kk = 0; kk < kD / 8; ++kk) {
      uint32_t ah[4], al[4];
      const float* qr = Q + row0 * kPitch + kk * 8 + c;
      split(qr[0], ah[0], al[0]);
      split(qr[8 * kPitch], ah[1], al[1]);
      split(qr[4], ah[2], al[2]);
      split(qr[8 * kPitch + 4], ah[3], al[3]);
#pragma unroll
      for (int j = 0; j < kKeys / 8; ++j) {
        const float* kr = K + (j * 8 + g) * kPitch + kk * 8 + c;
        mma3(sc[j], ah, al, kr[0], kr[4]);
      }
    }
    float alpha[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < kKeys / 8; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = sc[j][h * 2 + e];
          if (t * kKeys + j * 8 + c * 2 + e > tok[h]) x = -INFINITY;
          mx = fmaxf(mx, x);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      mx = fmaxf(mx, m[h]);
      const float ref = mx == -INFINITY ? 0.f : mx;
      alpha[h] = fast_exp2((m[h] - ref) * scale2);
      m[h] = mx;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < kKeys / 8; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = sc[j][h * 2 + e];
          x = fast_exp2((x - ref) * scale2);   // the difference first: large scores cost no accuracy
          sum += x;
        }
      l[h] = fmaf(l[h], alpha[h], sum);
    }
    // P V: the order of the eight keys of a step is free, so the accumulator's columns
    // (2c, 2c + 1) serve as the A fragment's (c, c + 4), and V's rows follow.
    uint32_t ph[kKeys / 8][4], pl[kKeys / 8][4];
#pragma unroll
    for (int j = 0; j < kKeys / 8; ++j) {
      split(sc[j][0], ph[j][0], pl[j][0]);
      split(sc[j][2], ph[j][1], pl[j][1]);
      split(sc[j][1], ph[j][2], pl[j][2]);
      split(sc[j][3], ph[j][3], pl[j][3]);
    }
#pragma unroll
    for (int n = 0; n < kD / 8; ++n) {
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kKeys / 8; ++j) {
        const float* vr = V + (j * 8 + c * 2) * kPitch + n * 8 + g;
        mma3(acc, ph[j], pl[j], vr[0], vr[kPitch]);
      }
      o[n][0] = fmaf(o[n][0], alpha[0], acc[0]);
      o[n][1] = fmaf(o[n][1], alpha[0], acc[1]);
      o[n][2] = fmaf(o[n][2], alpha[1], acc[2]);
      o[n][3] = fmaf(o[n][3], alpha[1], acc[3]);
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float s = l[h];
    s += __shfl_xor_sync(0xffffffffu, s, 1);
    s += __shfl_xor_sync(0xffffffffu, s, 2);
    const int r = row0 + h * 8;
    if (r < rows) {   // every row attends to itself: s >= 1, or NaN
      bool nan = false;
      float* out = static_cast<float*>(p.out) + static_cast<int64_t>(s0 + tok0 + r / G) * p.sot + (kvh * G + r % G) * p.soh;
#pragma unroll
      for (int n = 0; n < kD / 8; ++n) {
        const float2 y = make_float2(o[n][h * 2] / s, o[n][h * 2 + 1] / s);
        nan |= y.x != y.x || y.y != y.y;
        *reinterpret_cast<float2*>(out + n * 8 + c * 2) = y;
      }
      if (nan) atomicOr(&bad[r >> 5], 1u << (r & 31));
    }
  }
  __syncthreads();
  if (bad[0] | bad[1]) settle_rows(p, Q, KV, s0, len, tok0, toks, kvh, bad[0] | static_cast<uint64_t>(bad[1]) << 32);
}

// ---------------------------------------------------------------- bf16
// tcgen05. A block works on two tiles (A, B) of 128 rows, consecutive in the same
// sequence and kv head, against K / V tiles of 128 keys: while the tensor core runs one
// tile's products, the other tile's softmax runs, one thread per row.
//
//   S_t = Q_t K^T           tcgen05.mma 128 x 128 x 128 -> TMEM
//   p = 2^(S scale2 - m)    m moves (and O, l are rescaled) only when the tile's maximum
//                           exceeds it by more than 2^8: exact, and rare after the first tiles
//   O_t += bf16(p) V        tcgen05.mma, A = P in tensor memory (over S_t), O stays in TMEM
//
// A weight enters P V as one bf16 part, good to 2^-8, as in the trie kernel's prefix: a second part
// would make the products of a step half as long again. On 96 random tokens the result
// is off by 1.84e-3 (2-norm), where one rounded once from nearly exact sums is by 1.59e-3. Scores,
// maxima, weights before that rounding and their sums are fp32.
//
// Warps 0-3 / 4-7: softmax of tile A / B, one row a thread (no exchange between
// threads); warp 8: TMA (Q of the block, a ring of K and V tiles); warp 9: issues the
// MMAs; warp 10: says which tiles are next; warp 11: cleans V. The block is persistent: K / V and Q of its
// next work item arrive, and S of it is computed, while the results of the last one are
// written out.
//
// A weight of zero does not silence a masked V row that holds an infinity or a NaN. So warp 11
// looks at the V rows after the item's first token (every row of the item attends to those up to
// it) while their softmax runs, and clears what is not finite, and rows past the sequence, before
// their P V. What rows attend to of it is added to the results at the end (restore_rows): at most
// 2 TP - 1 keys a row, whatever the length, and nothing where V is finite. It costs 16 / 16 heads (255
// V rows an item) 2%, groups of 4 and 7 nothing that shows.
//
// Bound: the chain S -> softmax -> P V -> next S of a tile (S and P share tensor memory).
// A step of 128 keys takes about 3,100 cycles, of which the two tiles' four products need
// 2,048: 1,880 of softmax (1,024 of them the exponentials of a thread's 128 scores), 770 of
// MMA that the other tile's softmax covers, the rest hand-overs. Measured: 32,768 tokens,
// 32 / 8 heads 7.5 ms (1,170 TFLOP/s; a matrix product of the library holds 1,390 for that
// long); 16 prompts of about 4,096, 28 / 4 heads 2.0 ms (950). Two threads a row
// (16 softmax warps) measured slower (1,020), as did more of the exponentials on the FMA
// pipe (a half: 1,050) and P in four parts (1,090).
namespace tcp {
constexpr int kRows = 128, kKeys = 128;
constexpr int kHalf = 128 * 64 * 2;              // 64 dims of 128 rows: 16 KB, 128-byte swizzle
constexpr int kTile = 2 * kHalf;
constexpr int kRing = 4;                         // K / V buffers
constexpr int kKVOff = 2 * kTile;                // after Q_A, Q_B
constexpr int kStageOff = kKVOff + kRing * kTile;  // results on their way out: 32 rows of 64 dims a softmax warp
constexpr int kBarOff = kStageOff + 8 * 4096;
constexpr int kItemOff = kBarOff + 256;          // announced items, 32 bytes each
constexpr int kRefOff = kItemOff + 64;           // references of the rows' weights, for restore_rows
constexpr int kSmem = 1024 + kRefOff + 2 * kRows * 4;
static_assert(kSmem <= 232448, "shared memory budget");
constexpr int kTileThreads = 128, kThreads = 3 * kTileThreads;   // the last warpgroup: TMA, MMA, the work items, V
// registers a thread: 168 at launch (3 x 128 of them); the softmax warps take what the others leave
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;
static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * 168, "register split");
constexpr int kProducerWarp = 8, kMmaWarp = 9, kItemWarp = 10, kCleanWarp = 11;
constexpr int kParts = 2;                        // P is handed over in parts of 128 / kParts keys
constexpr int kItems = 2;                        // work items announced ahead
enum { Q_FULL = 0, Q_EMPTY = 1, KV_FULL = 2, KV_EMPTY = KV_FULL + kRing, S_FULL = KV_EMPTY + kRing, P_FULL = S_FULL + 2,
       O_FULL = P_FULL + 2 * kParts, ITEM_FULL = O_FULL + 2, ITEM_EMPTY = ITEM_FULL + kItems, V_ASK = ITEM_EMPTY + kItems,
       V_CLEAN = V_ASK + 2, NBAR = V_CLEAN + 2 };
static_assert(kRing == 4, "K in the even buffers, V in the odd ones: V_ASK and V_CLEAN of buffer b are number b / 2");
// Items whose V held something not finite: word i % kOddItems is i + 1 where item i is one. A warp
// still at item i keeps the others from going past item i + kItems.
constexpr int kOddItems = 4;
static_assert(kOddItems > kItems, "a word is not written again before it has been read");
static_assert(NBAR * 8 + 4 + kOddItems * 4 <= kItemOff - kBarOff, "barriers, TMEM address and flags");
constexpr uint32_t kSCol = 0, kOCol = 256;       // S_t (and P_t) at 128 t, O_t at 256 + 128 t
constexpr uint32_t kIdescQK = idesc_bf16_f32(128, 128, 0, 0);
constexpr uint32_t kIdescPV = idesc_bf16_f32(128, 128, 0, 1);
constexpr float kSlack = 8.0f;

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_plain(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
// 32 consecutive columns per thread, without the wait.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void mbar_arrive_if(uint32_t bar, bool go) {   // without a branch
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar),
               "r"(static_cast<uint32_t>(go))
               : "memory");
}
__device__ __forceinline__ bool elect_one() {   // true in one lane of a converged warp
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// Bits 15 and 31: the half is an infinity or a NaN.
__device__ __forceinline__ uint32_t not_finite(uint32_t x) { return ((x & 0x7F807F80u) + 0x00800080u) & 0x80008000u; }
__device__ __forceinline__ void max_abs(uint32_t& m, uint4 x) {   // of bf16 pairs; the signs mean nothing
  for (const uint32_t w : {x.x, x.y, x.z, x.w}) asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The i-th work item of a block: the blocks take turns forwards and backwards, so that
// a round's heavy end does not always fall to the same block.
__device__ __forceinline__ int unit_of(int i) {
  return i * gridDim.x + ((i & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

// 2^x for a pair on the FMA pipe: x = n + f with n = round(x), |f| <= 1/2, times a cubic
// for 2^f (least relative error with the constant fixed at 1, found numerically: 2^-13.3,
// against the 2^-9 of the bf16 weight it becomes). x is at most kSlack; below -127, and
// for a masked -inf, the result is exactly 0; a NaN stays one.
__device__ __forceinline__ uint64_t exp2_pair(uint64_t x) {
  float a, b;
  unpair(x, a, b);
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(a), "f"(-127.f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(b), "f"(-127.f));
  x = pair(a, b);
  constexpr float kShift = 12582912.f + 127.f;   // 1.5 * 2^23: the low bits of x + kShift are n + 127
  const uint64_t t = add2(x, pair(kShift, kShift));
  const uint64_t f = sub2(x, sub2(t, pair(kShift, kShift)));
  uint64_t y = fma2(f, pair(0.05500892f, 0.05500892f), pair(0.24221096f, 0.24221096f));
  y = fma2(y, f, pair(0.69328293f, 0.69328293f));
  y = fma2(y, f, pair(1.f, 1.f));
  unpair(t, a, b);
  return mul2(y, pair(__uint_as_float(__float_as_uint(a) << 23), __uint_as_float(__float_as_uint(b) << 23)));
}

// One work item: two tiles of one sequence and kv head.
struct Item {
  int s0, len, tok0, kvh;   // sequence start, its length, first token of tile A
  int n[2];                 // K / V tiles of A and B (0: the tile has no token; A has one, or there is no item)
  int pad[2];
};
__device__ __forceinline__ void item_of(const Dev& p, int unit, Item* it) {
  const int TP = kRows / (p.H / p.HK);
  int seq, tile;
  it->n[0] = 0;
  if (!find_tile(p, 2 * TP, p.wide, unit / p.HK, &seq, &tile)) return;
  it->kvh = unit % p.HK;
  it->s0 = start_of(p, seq);
  it->len = length_of(p, seq);
  it->tok0 = tile * 2 * TP;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int first = it->tok0 + t * TP, last = min(first + TP, it->len);   // one past the tile's last token
    it->n[t] = first < it->len ? (last + kKeys - 1) / kKeys : 0;
  }
}
// First K / V tile with a key after the item's first token.
__device__ __forceinline__ int first_masked(const Item& it) { return (it.tok0 + 1) / kKeys; }

// What a softmax warp's rows attend to of the V entries that the clean warp took out (keys after
// the item's first token): such an entry makes its dim infinite or NaN. refs: the references of
// the rows' weights.
__device__ __noinline__ void restore_rows(const Dev& p, int s0, int len, int tok0, int kvh, const float* refs) {
  const int G = p.H / p.HK, TP = kRows / G, d = (threadIdx.x & 31) * 4;
  const int first = tok0 + (threadIdx.x / kRows) * TP, r0 = threadIdx.x / 32 % 4 * 32;   // of the tile: first token; of the warp: first row
  const int rows = min(TP, len - first) * G;
  auto load = [&](const void* base, int64_t at) {
    return *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + at + d);
  };
  auto value = [](uint2 x, int e) {
    const uint32_t w = e < 2 ? x.x : x.y;
    return __uint_as_float((e & 1) ? (w & 0xFFFF0000u) : (w << 16));
  };
  for (int r = r0; r < min(rows, r0 + 32); ++r) {
    const int tok = first + r / G, h = kvh * G + r % G;
    const float ref = refs[r - r0] == -INFINITY ? 0.f : refs[r - r0];
    const uint2 q = load(p.q, static_cast<int64_t>(s0 + tok) * p.sqt + h * p.sqh);
    float add[4] = {0.f, 0.f, 0.f, 0.f};
    uint32_t touched = 0;
#pragma unroll 4
    for (int key = tok0 + 1; key <= tok; ++key) {
      const uint2 v = load(p.v, static_cast<int64_t>(s0 + key) * p.svt + kvh * p.svh);
      const uint32_t lo = not_finite(v.x), hi = not_finite(v.y);
      if (!__any_sync(0xffffffffu, lo | hi)) continue;
      const uint2 k = load(p.k, static_cast<int64_t>(s0 + key) * p.skt + kvh * p.skh);
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) dot = fmaf(value(q, e), value(k, e), dot);
      const float w = fast_exp2(fmaf(warp_sum(dot), p.scale2, -ref));
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((e < 2 ? lo : hi) >> ((e & 1) * 16 + 15) & 1) {
          add[e] += w * value(v, e);
          touched |= 1u << e;
        }
    }
    uint16_t* out = static_cast<uint16_t*>(p.out) + static_cast<int64_t>(s0 + tok) * p.sot + h * p.soh + d;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (touched >> e & 1) out[e] = f32_to_bf16_bits(add[e] + bf16_bits_to_f32(out[e]));
  }
}
}  // namespace tcp

// kFlip: a negative scale, with which the largest weight is at the smallest S.
template <bool kFlip>
__global__ void __launch_bounds__(tcp::kThreads, 1)
    prompt_tc(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
              const __grid_constant__ CUtensorMap tv, const Dev p) {
  using namespace tcp;
  extern __shared__ uint8_t psm[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(psm) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kBarOff);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + NBAR);
  volatile int* odd_items = reinterpret_cast<int*>(tmem_slot + 1);
  auto bar = [&](int i) { return smem_u32(bars + i); };
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int G = p.H / p.HK, TP = kRows / G;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tq);
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
    mbar_init(bar(Q_FULL), 1);
    mbar_init(bar(Q_EMPTY), 1);
    for (int i = 0; i < kRing; ++i) {
      mbar_init(bar(KV_FULL + i), 1);
      mbar_init(bar(KV_EMPTY + i), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar(S_FULL + t), 1);
      for (int x = 0; x < kParts; ++x) mbar_init(bar(P_FULL + t * kParts + x), kTileThreads / 32);
      mbar_init(bar(O_FULL + t), 1);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(bar(ITEM_FULL + i), 1);
      mbar_init(bar(ITEM_EMPTY + i), 11);   // eight softmax warps, TMA, MMA, V
    }
    for (int i = 0; i < kOddItems; ++i) odd_items[i] = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(V_ASK + i), 1);
      mbar_init(bar(V_CLEAN + i), 1);
    }
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  pdl_wait();
  pdl_trigger();
  const uint32_t sQ = smem_u32(smem), sKV = smem_u32(smem + kKVOff);
  Item* items = reinterpret_cast<Item*>(smem + kItemOff);
  float* refs = reinterpret_cast<float*>(smem + kRefOff);
  Item it;
  // The i-th item, as announced; false after the last one (or after a wait gave up).
  auto next_item = [&](int i) {
    const int x = i % kItems;
    if (!__all_sync(0xffffffffu, mbar_wait_spin(bar(ITEM_FULL + x), (i / kItems) & 1, 0x31a))) return false;
    it = items[x];
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(ITEM_EMPTY + x));
    return it.n[0] > 0;
  };

  if (warp >= kProducerWarp) {   // one setmaxnreg for the whole warpgroup
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kProducerWarp) {
      uint32_t ring = 0, q_loads = 0;   // K / V tiles, Q pairs loaded so far
      bool ok = true;
      for (int i = 0; ok && next_item(i); ++i) {
        if (lane == 0) {
          if (i > 0) ok = mbar_wait_spin(bar(Q_EMPTY), (i - 1) & 1, 0x311);
          if (ok) {
            const int tiles = it.n[1] > 0 ? 2 : 1;
            mbar_arrive_expect_tx(bar(Q_FULL), tiles * 2 * TP * G * 128);
            ++q_loads;
            for (int t = 0; t < tiles; ++t)
              for (int h = 0; h < 2; ++h)
                tma_load_4d(sQ + t * kTile + h * kHalf, &tq, bar(Q_FULL), h * 64, 0, it.kvh, it.s0 + it.tok0 + t * TP);
          }
          const int n = max(it.n[0], it.n[1]);
          for (int x = 0; ok && x < 2 * n; ++x, ++ring) {   // K0, V0, K1, V1, ...
            const int b = ring % kRing;
            const uint32_t use = ring / kRing;
            if (use > 0) ok = mbar_wait_spin(bar(KV_EMPTY + b), (use - 1) & 1, 0x312);
            if (!ok) break;
            mbar_arrive_expect_tx(bar(KV_FULL + b), kTile);
            const CUtensorMap* m = (x & 1) ? &tv : &tk;
            for (int h = 0; h < 2; ++h)
              tma_load_3d_plain(sKV + b * kTile + h * kHalf, m, bar(KV_FULL + b), h * 64, it.s0 + (x >> 1) * kKeys, it.kvh);
            if ((x & 1) && (x >> 1) >= first_masked(it)) mbar_arrive(bar(V_ASK + b / 2));
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
      }
      if (!ok && lane == 0) {   // an error flag is up: see the copies in flight out
        if (q_loads > 0) mbar_wait(bar(Q_FULL), (q_loads - 1) & 1, 0x31d);
        for (uint32_t x = ring > kRing ? ring - kRing : 0; x < ring; ++x) mbar_wait(bar(KV_FULL + x % kRing), (x / kRing) & 1, 0x31d);
      }
    } else if (warp == kMmaWarp) {
      // The whole warp keeps the books, one lane issues: its loop is nothing but MMAs with
      // descriptors a constant apart (a branch or an address computation between them costs
      // more than the 64 cycles an MMA takes). Descriptors count addresses in 16-byte units
      // from bit 0, so steps are plain additions.
      const bool leader = elect_one();
      const uint64_t dq = sdesc_kmajor_sw128(sQ), dk = sdesc_kmajor_sw128(sKV), dv = sdesc_mnmajor_sw128(sKV, kHalf);
      uint32_t buf = 0, phase = 0;        // of the next K / V tile
      uint32_t steps[2] = {0, 0};         // P tiles of A and B consumed so far
      uint32_t clean = 0;                 // bit x: parity of V_CLEAN x
      auto advance = [&] {
        if (++buf == kRing) {
          buf = 0;
          phase ^= 1;
        }
      };
      auto issue_s = [&](int t, uint32_t kbuf) {
        if (leader) {
          const uint64_t q = dq + t * (kTile >> 4), k = dk + kbuf * (kTile >> 4);
#pragma unroll
          for (int kk = 0; kk < kD / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * kHalf + (kk & 3) * 32) >> 4;
            umma_bf16(tmem + kSCol + t * 128, q + off, k + off, kIdescQK, kk ? 1u : 0u);
          }
          umma_commit(bar(S_FULL + t));
        }
      };
      auto issue_o = [&](int t, uint32_t vbuf, int part, uint32_t add) {
        if (leader) {
          const uint64_t v = dv + vbuf * (kTile >> 4) + part * (kKeys / 16 / kParts * (2048 >> 4));
#pragma unroll
          for (int kk = 0; kk < kKeys / 16 / kParts; ++kk)
            umma_bf16_ta(tmem + kOCol + t * 128, tmem + kSCol + t * 128 + part * (64 / kParts) + kk * 8, v + kk * (2048 >> 4),
                         kIdescPV, kk ? 1u : add);
        }
      };
      auto commit = [&](int b) {
        if (leader) umma_commit(bar(b));
      };
      bool ok = true;
      for (int i = 0; ok && next_item(i); ++i) {
        const int n = max(it.n[0], it.n[1]), masked = first_masked(it);
        ok = mbar_wait_spin(bar(Q_FULL), i & 1, 0x314) && mbar_wait_spin(bar(KV_FULL + buf), phase, 0x313);
        if (!ok) break;
        tc_fence_after();
        issue_s(0, buf);
        if (it.n[1] > 0) issue_s(1, buf);
        commit(KV_EMPTY + buf);
        if (n == 1) commit(Q_EMPTY);
        advance();
        for (int j = 0; ok && j < n; ++j) {
          const uint32_t vbuf = buf, vphase = phase;
          advance();                      // buf, phase: K of the next tile, if there is one
          const bool more = j + 1 < n;
          bool v_in = false, k_in = false;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || j >= it.n[t]) continue;
            if (!v_in) {
              ok = v_in = mbar_wait_spin(bar(KV_FULL + vbuf), vphase, 0x313);
              if (ok && j >= masked) {
                const uint32_t x = vbuf >> 1;
                ok = mbar_wait_spin(bar(V_CLEAN + x), clean >> x & 1u, 0x318);
                clean ^= 1u << x;
              }
            }
#pragma unroll
            for (int x = 0; x < kParts; ++x) {
              ok = ok && mbar_wait_spin(bar(P_FULL + t * kParts + x), steps[t] & 1, 0x315);
              if (!ok) break;
              tc_fence_after();
              issue_o(t, vbuf, x, (j | x) ? 1u : 0u);
            }
            if (!ok) continue;
            ++steps[t];
            commit(O_FULL + t);
            if (t == 1 || j >= it.n[1]) commit(KV_EMPTY + vbuf);
            if (j + 1 < it.n[t]) {
              if (!k_in) ok = k_in = mbar_wait_spin(bar(KV_FULL + buf), phase, 0x31b);
              if (!ok) continue;
              tc_fence_after();
              issue_s(t, buf);
            }
          }
          if (ok && more) {
            commit(KV_EMPTY + buf);
            if (j + 2 == n) commit(Q_EMPTY);
            advance();
          }
        }
        ok = __all_sync(0xffffffffu, ok);
      }
    } else if (warp == kItemWarp) {
      bool ok = true;
      for (int i = 0; ok; ++i) {
        item_of(p, unit_of(i), &it);
        const int x = i % kItems;
        if (i >= kItems) ok = __all_sync(0xffffffffu, mbar_wait_spin(bar(ITEM_EMPTY + x), ((i / kItems) - 1) & 1, 0x31c));
        if (!ok) break;
        if (lane == 0) {
          items[x] = it;
          mbar_arrive(bar(ITEM_FULL + x));
        }
        if (it.n[0] == 0) break;
      }
    } else {
      // Of a V tile it is to clean it hears from the TMA warp (V_ASK): a wait on KV_FULL before the
      // tile's load has begun could take an earlier load's phase for it.
      uint32_t ring = 0;                  // of the item's K_0
      uint32_t asked = 0;                 // bit x: parity of V_ASK x
      bool ok = true;
      for (int i = 0; ok && next_item(i); ++i) {
        const int n = max(it.n[0], it.n[1]);
        bool odd = false;
        for (int j = first_masked(it); j < n; ++j) {
          const uint32_t at = ring + 2 * j + 1, b = at % kRing, y = b / 2;
          ok = __all_sync(0xffffffffu, mbar_wait_spin(bar(V_ASK + y), asked >> y & 1u, 0x31e) &&
                                           mbar_wait_spin(bar(KV_FULL + b), (at / kRing) & 1, 0x31f));
          if (!ok) break;
          asked ^= 1u << y;
          // half a row a quarter-warp: 16-byte pieces, whose order within a row does not matter
          uint8_t* v = smem + kKVOff + b * kTile + (lane >> 3 & 1) * kHalf + (lane & 7) * 16;
          const int from = max(it.tok0 + 1 - j * kKeys, 0) + (lane >> 4), end = min(it.len - j * kKeys, kKeys);
          uint32_t top = 0;               // largest magnitudes (a NaN if there is one)
          int r = from;
          for (; r + 14 < end; r += 16) {
#pragma unroll
            for (int e = 0; e < 8; ++e) max_abs(top, *reinterpret_cast<const uint4*>(v + (r + 2 * e) * 128));
          }
          for (; r < end; r += 2) max_abs(top, *reinterpret_cast<const uint4*>(v + r * 128));
#pragma unroll 4
          for (r = end + (lane >> 4); r < kKeys; r += 2) *reinterpret_cast<uint4*>(v + r * 128) = make_uint4(0, 0, 0, 0);
          if (not_finite(top)) {
            odd = true;
#pragma unroll 1
            for (r = from; r < end; r += 2) {
              uint4 x = *reinterpret_cast<const uint4*>(v + r * 128);
              x.x &= ~((not_finite(x.x) >> 15) * 0xFFFFu);
              x.y &= ~((not_finite(x.y) >> 15) * 0xFFFFu);
              x.z &= ~((not_finite(x.z) >> 15) * 0xFFFFu);
              x.w &= ~((not_finite(x.w) >> 15) * 0xFFFFu);
              *reinterpret_cast<uint4*>(v + r * 128) = x;
            }
          }
          if (odd) odd_items[i % kOddItems] = i + 1;
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(V_CLEAN + y));
        }
        ring += 2 * n;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int t = warp >> 2, q4 = warp & 3;
    const int r = q4 * 32 + lane;                      // row of the tile
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(q4 * 32) << 16);
    const uint32_t st = lane_base + kSCol + t * 128, ot = lane_base + kOCol + t * 128;
    const float masked = kFlip ? INFINITY : -INFINITY;
    const uint64_t scale_pair = pair(p.scale2, p.scale2);
    uint32_t step = 0;                                 // S tiles consumed so far
    bool ok = true;
    for (int i = 0; ok && next_item(i); ++i) {
      const int n = it.n[t];
      const int tok = it.tok0 + t * TP + r / G;        // keys <= tok are attended
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j, ++step) {
        ok = ok && __all_sync(0xffffffffu, mbar_wait_spin(bar(S_FULL + t), step & 1, 0x316));
        if (!ok) break;
        tc_fence_after();
        uint32_t s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(st + c * 32, s + c * 32);
        tmem_wait_ld();
        const int last = tok - j * kKeys;              // the last key of this tile that the row attends to
        if (__any_sync(0xffffffffu, last < kKeys - 1)) {
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c > last) s[c] = __float_as_uint(masked);
        }
        float top;
        if (!kFlip) {
          float a = __uint_as_float(s[0]), b = __uint_as_float(s[1]), c = __uint_as_float(s[2]), d = __uint_as_float(s[3]);
#pragma unroll
          for (int x = 4; x < 124; x += 8) {
            a = max3(a, __uint_as_float(s[x]), __uint_as_float(s[x + 1]));
            b = max3(b, __uint_as_float(s[x + 2]), __uint_as_float(s[x + 3]));
            c = max3(c, __uint_as_float(s[x + 4]), __uint_as_float(s[x + 5]));
            d = max3(d, __uint_as_float(s[x + 6]), __uint_as_float(s[x + 7]));
          }
          a = max3(a, __uint_as_float(s[124]), __uint_as_float(s[125]));
          b = max3(b, __uint_as_float(s[126]), __uint_as_float(s[127]));
          top = fmaxf(fmaxf(a, b), fmaxf(c, d));
        } else {
          top = __uint_as_float(s[0]);
#pragma unroll
          for (int x = 1; x < 128; ++x) top = fminf(top, __uint_as_float(s[x]));
        }
        top *= p.scale2;
        const float m_new = top > m + kSlack ? top : m;
        const float neg = m_new == -INFINITY ? 0.f : -m_new;
        if (j > 0 && __any_sync(0xffffffffu, m_new != m)) {   // O of this warp's rows, once P V of the last tile is in
          const float alpha = fast_exp2(m + neg);             // 1 for a row whose maximum stays
          l *= alpha;
          ok = __all_sync(0xffffffffu, mbar_wait_spin(bar(O_FULL + t), (step - 1) & 1, 0x317));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            uint32_t o[16];
            tmem_ld16_nowait(ot + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st16(ot + c * 16, o);
          }
        }
        m = m_new;
        // One straight run of code, so that the exponentials (8 cycles each on their pipe) of one
        // group of 16 overlap the sums, conversions and stores of the group before.
        const uint64_t neg_pair = pair(neg, neg);
        uint64_t sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)}, y[2][8];
        uint32_t w[2][8];
#pragma unroll
        for (int c = 0; c <= 8; ++c) {
          if (c < 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint64_t x = fma2(pair(__uint_as_float(s[c * 16 + 2 * e]), __uint_as_float(s[c * 16 + 2 * e + 1])), scale_pair, neg_pair);
              if (e == 7) {   // one pair of eight on the FMA pipe: the exponential's own is the longer queue
                y[c & 1][e] = exp2_pair(x);
              } else {
                float a, b;
                unpair(x, a, b);
                y[c & 1][e] = pair(fast_exp2(a), fast_exp2(b));
              }
            }
          }
          if (c > 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float a, b;
              unpair(y[(c - 1) & 1][e], a, b);
              sum[e & 1] = add2(sum[e & 1], y[(c - 1) & 1][e]);
              w[(c - 1) & 1][e] = pack_bf16x2(a, b);
            }
            tmem_st8(st + (c - 1) * 8, w[(c - 1) & 1]);
            if (c % (8 / kParts) == 0) {
              tmem_wait_st();     // the warp's own stores, all lanes
              tc_fence_before();
              mbar_arrive_if(bar(P_FULL + t * kParts + (c - 1) / (8 / kParts)), lane == 0);   // one per warp: arrivals queue up
            }
          }
        }
        float a, b;
        unpair(add2(sum[0], sum[1]), a, b);
        l += a + b;
      }
      const int tok_end = min(it.tok0 + (t + 1) * TP, it.len);
      if (n > 0 && ok) {
        ok = __all_sync(0xffffffffu, mbar_wait_spin(bar(O_FULL + t), (step - 1) & 1, 0x319));
        if (!ok) break;
        tc_fence_after();
        // Rows lie apart in memory (256 bytes each): a warp's 64 dims of 32 rows pass through
        // shared memory (16-byte pieces swizzled by row), so that a store covers 4 lines, not 32.
        const bool live = r < TP * G && tok < tok_end;
        const int64_t at = live ? static_cast<int64_t>(it.s0 + tok) * p.sot + (it.kvh * G + r % G) * p.soh : -1;
        const float inv = 1.f / l;
        refs[warp * 32 + lane] = m;
        uint8_t* stage = smem + kStageOff + warp * 4096;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t o[32];
            tmem_ld32(ot + half * 64 + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t w[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float a = __uint_as_float(o[e * 8 + 2 * x]) * inv, b = __uint_as_float(o[e * 8 + 2 * x + 1]) * inv;
                w[x] = pack_bf16x2(a, b);
              }
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((c * 4 + e) ^ (lane & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          __syncwarp();
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const int row = x * 4 + (lane >> 3), piece = lane & 7;
            const int64_t to = __shfl_sync(0xffffffffu, at, row);
            const uint4 v = *reinterpret_cast<const uint4*>(stage + row * 128 + ((piece ^ (row & 7)) * 16));
            if (to >= 0) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + to + half * 64 + piece * 8) = v;
          }
          __syncwarp();
        }
        tc_fence_before();   // O read before the next item's P (and so its P V) is announced
        if (__any_sync(0xffffffffu, odd_items[i % kOddItems] == i + 1))
          restore_rows(p, it.s0, it.len, it.tok0, it.kvh, refs + warp * 32);
      }
    }
    if (p.zero_rest) zero_rest<uint16_t>(p, 2 * kTileThreads);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace pr

static int prompt_validate(const rb_prompt_args* a) {
  if (!a || a->B < 0 || a->T < 0 || a->H <= 0 || a->HK <= 0) return RB_ERR_INVALID_ARG;
  if ((a->dtype != RB_BF16 && a->dtype != RB_F32) || a->D != pr::kD || a->H % a->HK != 0 || a->H / a->HK > 64)
    return RB_ERR_UNSUPPORTED;
  if (a->T == 0) return RB_OK;
  if (!a->q || !a->k || !a->v || !a->out || !a->cu) return RB_ERR_INVALID_ARG;
  const int es = a->dtype == RB_BF16 ? 2 : 4;
  for (int64_t s : {a->sqt, a->sqh, a->skt, a->skh, a->svt, a->svh, a->sot, a->soh})
    if (s < 0 || s * es % 16 != 0) return RB_ERR_UNSUPPORTED;
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out)) return RB_ERR_UNSUPPORTED;
  if (!(a->sm_scale == a->sm_scale)) return RB_ERR_INVALID_ARG;
  return RB_OK;
}

int prompt_launch(const rb_prompt_args* a, cudaStream_t st) {
  using namespace pr;
  int r = prompt_validate(a);
  if (r != RB_OK || a->T == 0) return r;
  Dev p{a->q, a->k, a->v, a->sqt, a->sqh, a->skt, a->skh, a->svt, a->svh, a->cu, a->B, a->T, a->H, a->HK,
        a->out, a->sot, a->soh, a->sm_scale * 1.4426950408889634f, (device_sm_count() + a->HK - 1) / a->HK, a->zero_rest};
  const int G = a->H / a->HK;
  if (a->sm_scale == 0.f) p.scale2 = 1e-37f;   // equal weights; a factor of zero would turn the mask's infinity into a NaN
  if (a->dtype == RB_BF16) {
    const int TP = tcp::kRows / G;
    const int64_t units = (static_cast<int64_t>(a->T) / (2 * TP) + a->B + 1) * a->HK;   // at most
    if (units > INT32_MAX / 2) return RB_ERR_CAPACITY;
    // a dimension of one entry may have any stride: give the map a plain one
    const int64_t sqt = a->T > 1 ? a->sqt : 8, sqh = G > 1 ? a->sqh : 8, sqg = a->HK > 1 ? G * a->sqh : 8;
    const int64_t skt = a->T > 1 ? a->skt : 8, skh = a->HK > 1 ? a->skh : 8, svt = a->T > 1 ? a->svt : 8, svh = a->HK > 1 ? a->svh : 8;
    CUtensorMap tq, tk, tv;
    const uint64_t dims[4] = {kD, static_cast<uint64_t>(G), static_cast<uint64_t>(a->HK), static_cast<uint64_t>(a->T)};
    const uint64_t strides[3] = {static_cast<uint64_t>(sqh) * 2, static_cast<uint64_t>(sqg) * 2, static_cast<uint64_t>(sqt) * 2};
    const uint32_t box[4] = {64, static_cast<uint32_t>(G), 1, static_cast<uint32_t>(TP)};
    r = encode_tiled(&tq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, a->q, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (r == RB_OK) r = encode_heads_3d(&tk, a->k, a->T, a->HK, skt, skh);
    if (r == RB_OK) r = encode_heads_3d(&tv, a->v, a->T, a->HK, svt, svh);
    if (r != RB_OK) return r;
    const auto kern = p.scale2 < 0.f ? prompt_tc<true> : prompt_tc<false>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, tcp::kSmem) != cudaSuccess)
      return RB_ERR_CUDA;
    const int64_t grid = units < device_sm_count() ? units : device_sm_count();
    return launch_k(kern, dim3(static_cast<unsigned>(grid)), dim3(tcp::kThreads), tcp::kSmem, st, true, tq, tk, tv, p);
  }
  const int TP = f32::kRows / G;
  const int64_t grid = (static_cast<int64_t>(a->T) / TP + a->B + 1) * a->HK;   // tiles at most
  if (grid > INT32_MAX) return RB_ERR_CAPACITY;
  if (cudaFuncSetAttribute(prompt_f32, cudaFuncAttributeMaxDynamicSharedMemorySize, f32::kSmem) != cudaSuccess)
    return RB_ERR_CUDA;
  return launch_k(prompt_f32, dim3(static_cast<unsigned>(grid)), dim3(f32::kThreads), f32::kSmem, st, true, p);
}

}  // namespace rb
