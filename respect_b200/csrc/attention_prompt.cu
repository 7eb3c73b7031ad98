// Causal grouped-query attention over whole packed prompts.
//
//   out_i = sum_{j <= i} softmax_j(q_i . k_j * scale) v_j   within each sequence
//
// A tile is TP = rows / G tokens x the G query heads of one kv head (row r = token
// r / G, head r % G), so a group's heads share every K / V tile and short prompts
// fill the rows. Keys are taken in tiles at absolute positions of the sequence, in
// ascending order; a tile that lies wholly after a row's token changes nothing of
// that row. A row's bits therefore depend on its own sequence alone, not on the
// packing or on which tile it falls into. Tiles are handed out heaviest first (by
// their number within the sequence), so that the last blocks to run are short.
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
  int zero_rest;                           // rows of no sequence: zeros (else left alone)
};

__device__ __forceinline__ int start_of(const Dev& p, int i) { return min(max(p.cu[i], 0), p.T); }
__device__ __forceinline__ int length_of(const Dev& p, int i) { return max(start_of(p, i + 1) - start_of(p, i), 0); }

// The rank-th tile of tp tokens in descending order of its number within its
// sequence (the earlier sequence first among equals). Warp-wide, the same in every
// lane; false when there are fewer tiles. `above(L)` counts the tiles numbered >= L.
__device__ __forceinline__ bool find_tile(const Dev& p, int tp, int rank, int* seq, int* tile) {
  const int lane = threadIdx.x & 31;
  int tiles0 = 0, most = 0;   // this lane's first sequence is looked at often
  if (lane < p.B) tiles0 = (length_of(p, lane) + tp - 1) / tp;
  for (int i = lane; i < p.B; i += 32) most = max(most, i == lane ? tiles0 : (length_of(p, i) + tp - 1) / tp);
  most = __reduce_max_sync(0xffffffffu, most);
  auto above = [&](int L) {
    int n = max(tiles0 - L, 0);
    for (int i = lane + 32; i < p.B; i += 32) n += max((length_of(p, i) + tp - 1) / tp - L, 0);
    return __reduce_add_sync(0xffffffffu, n);
  };
  if (above(0) <= rank) return false;
  int lo = 0, hi = most;      // above(lo) > rank >= above(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (above(mid) > rank) lo = mid; else hi = mid;
  }
  int left = rank - above(lo + 1);   // among the sequences with more than lo tiles
  for (int base = 0; base < p.B; base += 32) {
    const int i = base + lane;
    const int n = base == 0 ? tiles0 : i < p.B ? (length_of(p, i) + tp - 1) / tp : 0;
    const unsigned has = __ballot_sync(0xffffffffu, n > lo);
    const int c = __popc(has);
    if (left < c) {
      *seq = base + __fns(has, 0, left + 1);
      *tile = lo;
      return true;
    }
    left -= c;
  }
  return false;
}

// Rows before cu[0] and from cu[B] on belong to no sequence.
template <typename T>
__device__ __forceinline__ void zero_rest(const Dev& p) {
  const int a = start_of(p, 0), b = max(start_of(p, p.B), a);
  const int64_t n = static_cast<int64_t>(a + (p.T - b)) * p.H * kD;
  for (int64_t x = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; x < n;
       x += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    int64_t t = x / (p.H * kD);
    if (t >= a) t += b - a;
    const int h = static_cast<int>(x / kD % p.H), d = static_cast<int>(x % kD);
    static_cast<T*>(p.out)[t * p.sot + h * p.soh + d] = T(0);
  }
}

// Row `tok` of query head h again, by one warp and key by key. The tiles multiply V
// rows after the row's own token by a weight of zero, which is not nothing when such
// a row holds an infinity or a NaN; a row that came out NaN is settled here.
template <typename T>
__device__ __noinline__ void redo_row(const Dev& p, int s0, int tok, int h) {
  const int lane = threadIdx.x & 31, d = lane * 4, kvh = h / (p.H / p.HK);
  auto load = [&](const void* base, int64_t at, float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      x[e] = sizeof(T) == 4 ? static_cast<const float*>(base)[at + d + e]
                            : bf16_bits_to_f32(static_cast<const uint16_t*>(base)[at + d + e]);
  };
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  load(p.q, static_cast<int64_t>(s0 + tok) * p.sqt + h * p.sqh, q);
  for (int j = 0; j <= tok; ++j) {
    float k[4], v[4];
    load(p.k, static_cast<int64_t>(s0 + j) * p.skt + kvh * p.skh, k);
    load(p.v, static_cast<int64_t>(s0 + j) * p.svt + kvh * p.svh, v);
    const float s = warp_sum(fmaf(q[0], k[0], fmaf(q[1], k[1], fmaf(q[2], k[2], q[3] * k[3])))) * p.scale2;
    const float mx = fmaxf(m, s), ref = mx == -INFINITY ? 0.f : mx;
    const float a = fast_exp2(m - ref), w = fast_exp2(s - ref);
    m = mx;
    l = fmaf(l, a, w);
    bool nan = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = a == 0.f ? w * v[e] : fmaf(o[e], a, w * v[e]);
      nan &= o[e] != o[e];
    }
    if (__all_sync(0xffffffffu, nan || l != l)) break;   // nothing changes any more
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t at = static_cast<int64_t>(s0 + tok) * p.sot + h * p.soh + d + e;
    if (sizeof(T) == 4) static_cast<float*>(p.out)[at] = o[e] / l;
    else static_cast<uint16_t*>(p.out)[at] = f32_to_bf16_bits(o[e] / l);
  }
}

// ---------------------------------------------------------------- fp32
// Tensor cores with every operand in two tf32 parts (hi hi + hi lo + lo hi: good to
// about 2^-22 of a product). Four warps of 16 rows; K / V tiles of 32 keys arrive by
// cp.async one tile ahead. Each step of eight starts from zero and is added to the
// running sum in fp32, so that sum rounds to nearest however long it gets.
namespace f32 {
constexpr int kWarps = 4, kThreads = 32 * kWarps, kRows = 16 * kWarps, kKeys = 32;
constexpr int kPitch = kD + 4;   // floats per staged row: fragment reads without bank conflicts
constexpr int kTile = kKeys * kPitch;
constexpr int kSmem = (kRows * kPitch + 4 * kTile) * 4;

__device__ __forceinline__ uint32_t tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
  hi = tf32(x);
  lo = tf32(x - __uint_as_float(hi));
}
__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma3(float (&d)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], float b0, float b1) {
  uint32_t h0, l0, h1, l1;
  split(b0, h0, l0);
  split(b1, h1, l1);
  float t[4] = {0.f, 0.f, 0.f, 0.f};   // the tensor core's own additions truncate: keep them short
  mma8(t, al, h0, h1);
  mma8(t, ah, l0, l1);
  mma8(t, ah, h0, h1);
#pragma unroll
  for (int e = 0; e < 4; ++e) d[e] += t[e];
}
__device__ __forceinline__ float4 widen(const uint16_t* x) {
  const uint2 u = *reinterpret_cast<const uint2*>(x);
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xFFFF0000u));
}
__device__ __forceinline__ float4 widen(const float* x) { return *reinterpret_cast<const float4*>(x); }
__device__ __forceinline__ void copy16(float* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
}  // namespace f32

template <typename T>
__global__ void __launch_bounds__(f32::kThreads) prompt_mma(const Dev p) {
  using namespace f32;
  extern __shared__ __align__(16) float fsm[];
  float* Q = fsm;
  float* KV = fsm + kRows * kPitch;   // two stages of K, V
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  pdl_wait();
  pdl_trigger();
  if (p.zero_rest) zero_rest<T>(p);
  const int G = p.H / p.HK, TP = kRows / G;
  const int kvh = blockIdx.x % p.HK;
  int seq, tile;
  if (!find_tile(p, TP, blockIdx.x / p.HK, &seq, &tile)) return;
  const int s0 = start_of(p, seq), len = length_of(p, seq);
  const int tok0 = tile * TP, toks = min(TP, len - tok0), rows = toks * G;
  const int tiles = (tok0 + toks + kKeys - 1) / kKeys;
  const T* kg = static_cast<const T*>(p.k) + static_cast<int64_t>(s0) * p.skt + kvh * p.skh;
  const T* vg = static_cast<const T*>(p.v) + static_cast<int64_t>(s0) * p.svt + kvh * p.svh;
  auto fetch = [&](int t) {   // rows past the sequence are zero
    float* K = KV + (t & 1) * 2 * kTile;
    for (int x = threadIdx.x; x < kKeys * 32; x += kThreads) {
      const int r = x >> 5, piece = (x & 31) * 4, key = t * kKeys + r;
      const bool ok = key < len;
      if (sizeof(T) == 2) {   // bf16 widened: exact in one tf32 part
        *reinterpret_cast<float4*>(K + r * kPitch + piece) = ok ? widen(kg + key * p.skt + piece) : make_float4(0.f, 0.f, 0.f, 0.f);
        *reinterpret_cast<float4*>(K + kTile + r * kPitch + piece) = ok ? widen(vg + key * p.svt + piece) : make_float4(0.f, 0.f, 0.f, 0.f);
        continue;
      }
      copy16(K + r * kPitch + piece, ok ? kg + key * p.skt + piece : kg, ok ? 16u : 0u);
      copy16(K + kTile + r * kPitch + piece, ok ? vg + key * p.svt + piece : vg, ok ? 16u : 0u);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(0);
  const T* qg = static_cast<const T*>(p.q) + static_cast<int64_t>(s0 + tok0) * p.sqt + kvh * G * p.sqh;
  for (int x = threadIdx.x; x < kRows * 32; x += kThreads) {
    const int r = x >> 5, piece = (x & 31) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < rows) v = widen(qg + r / G * p.sqt + r % G * p.sqh + piece);
    *reinterpret_cast<float4*>(Q + r * kPitch + piece) = v;
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
      alpha[h] = fast_exp2((m[h] - ref) * p.scale2);
      m[h] = mx;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < kKeys / 8; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = sc[j][h * 2 + e];
          x = fast_exp2((x - ref) * p.scale2);   // the difference first: large scores cost no accuracy
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
    bool nan = false;
    if (r < rows) {   // every row attends to itself: s >= 1, or NaN
      T* out = static_cast<T*>(p.out) + static_cast<int64_t>(s0 + tok0 + r / G) * p.sot + (kvh * G + r % G) * p.soh;
#pragma unroll
      for (int n = 0; n < kD / 8; ++n) {
        const float2 y = make_float2(o[n][h * 2] / s, o[n][h * 2 + 1] / s);
        nan |= y.x != y.x || y.y != y.y;
        if (sizeof(T) == 4) *reinterpret_cast<float2*>(out + n * 8 + c * 2) = y;
        else *reinterpret_cast<uint32_t*>(out + n * 8 + c * 2) = pack_bf16x2(y.x, y.y);
      }
    }
    unsigned again = __ballot_sync(0xffffffffu, nan);
    for (int x = 0; again; ++x, again >>= 4)
      if (again & 0xFu) {   // the four lanes of row x
        const int rr = warp * 16 + h * 8 + x;
        redo_row<T>(p, s0, tok0 + rr / G, kvh * G + rr % G);
      }
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
        a->out, a->sot, a->soh, a->sm_scale * 1.4426950408889634f, a->zero_rest};
  const int TP = f32::kRows / (a->H / a->HK);
  const int64_t grid = (static_cast<int64_t>(a->T) / TP + a->B + 1) * a->HK;   // tiles at most
  if (grid > INT32_MAX) return RB_ERR_CAPACITY;
  const auto kern = a->dtype == RB_F32 ? prompt_mma<float> : prompt_mma<uint16_t>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, f32::kSmem) != cudaSuccess)
    return RB_ERR_CUDA;
  return launch_k(kern, dim3(static_cast<unsigned>(grid)), dim3(f32::kThreads), f32::kSmem, st, true, p);
}

}  // namespace rb
