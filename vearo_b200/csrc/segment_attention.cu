// Causal attention with grouped heads over packed segments, forward and backward, on tcgen05 with half-precision pairs (split16.cuh).
//
//   row t of segment [b, e):  s_tj = scale q_t . k_j for b <= j <= t,  p = softmax(s),  o = sum p v,  lse = log sum exp s
//   backward: delta = do . o,  ds = p (do . v - delta),  dq = scale sum ds k,  dk = scale sum over the group ds q,  dv = sum p do
//
// The pack is one stream of tokens cut into tiles of 128 rows, whatever the segments: a tile's rows look back to the begin of
// the first row's segment (ahead to the end of the last row's), and only tiles that a segment border or the diagonal crosses are
// masked.  Many short segments thus share tiles, and a long one pays one partly used tile at each end.
//
// k_prepare writes every 128-row tile of a head as half-precision planes with one exponent a tile; the kernels fold the
// exponents into factors they apply anyway.  Components that are not finite are written as 0, because a product over keys
// would carry them into rows that do not see them; a row that does see one gets a NaN sum of exponentials (forward), and
// through its lse NaN gradients.
//
// The matrices of scores never leave the SM.  In every kernel eight warps hold one row each thread x half the tile's columns; the
// second product takes its left operand (P, dS; hi and lo) from tensor memory, where these warps write it, and its right
// operand from the same shared-memory tile that the first product read (MN-major instead of K-major).  The second product of each tile goes to a
// fresh accumulator that the warps add to their registers with the running rescale, so the accumulator's truncation (split16.cuh) never
// runs longer than a tile.
//   k_forward   S = Q K^T, softmax with a running maximum, O += P V
//   k_grad_v    S^T = K Q^T, P^T from the saved lse, dV += P^T dO         (all query heads of the group: no atomics)
//   k_grad_qk   dQ: S = Q K^T, dP = dO V^T, dQ += dS K;  dK: the same with the roles of rows and columns exchanged
// Every wait is bounded; when one runs out the CTA raises the device error word, frees its tensor memory and returns.
#include "segment_attention.h"
#include "split16.cuh"

namespace vb {
namespace {
using namespace tc;

constexpr int kThreads = 320;             // warp 0: TMA, warp 1: MMA, warps 2-9: rows
constexpr float kL2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// ---- planes ------------------------------------------------------------------------------------------------------------------------
// One of q, k, v, do: planes [2][heads][T][DP], and per head and tile the inverse scale, the largest row length and a bit for every row
// with a component that is not finite.
struct PlanesDev { const float* x; i64 st, sh; __half* planes; float* inv; float* len; uint32_t* bad; int heads; bool vec; };
struct PrepareDev {
  PlanesDev in[4];
  int n, T, tiles, dk, hq;
  const float* starts; int n_seg; int* begin; int* end; int* err;      // where the segment of each row begins and ends (begin null: not wanted)
  const float* o; i64 o_st, o_sh; const float* lse;                     // for do: delta and the lse in base 2, padded to whole tiles
  float* delta; float* lse2;
};

// Where the segment of row t begins and ends (rows of no segment: an empty range).  Offsets that decrease or leave [0, T] are
// reported; whatever they are, every range stays inside [0, T].
__device__ __forceinline__ void find_segment(const PrepareDev& p, int t) {
  for (int i = t; i <= p.n_seg; i += p.tiles * 128) {
    const float s = p.starts[i];
    if (!(s > -0.5f)) atomicOr(p.err, ERRBIT_NEG_ID);
    else if (!(s < (float)p.T + 0.5f) || (i > 0 && !(p.starts[i - 1] <= s))) atomicOr(p.err, ERRBIT_OOB_ID);
  }
  if (t >= p.T) return;
  int lo = 0, hi = p.n_seg + 1;          // offsets [0, lo) are <= t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (roundf(p.starts[mid]) <= (float)t) lo = mid + 1; else hi = mid;
  }
  int b = p.T, e = 0;
  if (lo > 0 && lo <= p.n_seg) {
    const float fb = roundf(p.starts[lo - 1]), fe = roundf(p.starts[lo]);
    b = fb > 0.0f ? (int)fb : 0;
    e = fe < (float)p.T ? (int)fe : p.T;
    if (!(b <= t && t < e)) { b = p.T; e = 0; }
  }
  p.begin[t] = b; p.end[t] = e;
}

template <int DP>
__global__ void __launch_bounds__(256) k_prepare(PrepareDev p) {
  constexpr int kLanes = DP / 4, kRows = 256 / kLanes, kPasses = 128 / kRows;      // lanes of a row, rows of a pass
  __shared__ float red[8];
  __shared__ uint32_t bad[4];
  const int tile = blockIdx.x;
  int h = blockIdx.y, which = 0;
  while (h >= p.in[which].heads) h -= p.in[which++].heads;
  const PlanesDev& x = p.in[which];
  if (p.begin && blockIdx.y == 0 && threadIdx.x < 128) find_segment(p, tile * 128 + threadIdx.x);
  if (threadIdx.x < 4) bad[threadIdx.x] = 0;
  __syncthreads();
  const int c = (threadIdx.x % kLanes) * 4, r0 = threadIdx.x / kLanes;
  float4 v[kPasses];
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = i * kRows + r0;
    const i64 t = (i64)tile * 128 + r;
    v[i] = make_float4(0, 0, 0, 0);
    if (t < p.T && c < p.dk) {
      const float* s = x.x + t * x.st + h * x.sh + c;
      if (x.vec) v[i] = *reinterpret_cast<const float4*>(s);
      else { v[i].x = s[0]; if (c + 1 < p.dk) v[i].y = s[1]; if (c + 2 < p.dk) v[i].z = s[2]; if (c + 3 < p.dk) v[i].w = s[3]; }
    }
    if (p.delta && which == 3) {      // delta of the row, and its lse in base 2 (a row of no segment: +infinity, so that every p is 0)
      float d = 0.0f;
      if (t < p.T && c < p.dk) {
        const float* o = p.o + t * p.o_st + h * p.o_sh + c;
        d = v[i].x * o[0];
        if (c + 1 < p.dk) d = fmaf(v[i].y, o[1], d);
        if (c + 2 < p.dk) d = fmaf(v[i].z, o[2], d);
        if (c + 3 < p.dk) d = fmaf(v[i].w, o[3], d);
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
      if (c == 0) {
        float l = t < p.T ? p.lse[(i64)h * p.T + t] : -INFINITY;
        const bool dead = l == -INFINITY;
        if (d != d) l = d;             // (a gradient that is not finite: dv sees it through p)
        p.lse2[((i64)h * p.tiles + tile) * 128 + r] = dead ? INFINITY : l * kL2e;
        p.delta[((i64)h * p.tiles + tile) * 128 + r] = dead ? 0.0f : d;
      }
    }
    const float a = finite_abs(v[i].x), b = finite_abs(v[i].y), cc = finite_abs(v[i].z), d = finite_abs(v[i].w);
    const bool fine = a == fabsf(v[i].x) && b == fabsf(v[i].y) && cc == fabsf(v[i].z) && d == fabsf(v[i].w);
    if (!fine) {
      if (a != fabsf(v[i].x)) v[i].x = 0.0f;
      if (b != fabsf(v[i].y)) v[i].y = 0.0f;
      if (cc != fabsf(v[i].z)) v[i].z = 0.0f;
      if (d != fabsf(v[i].w)) v[i].w = 0.0f;
      atomicOr(&bad[r >> 5], 1u << (r & 31));
    }
    m = fmaxf(m, fmaxf(fmaxf(a, b), fmaxf(cc, d)));
  }
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[wid] = m;
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, red[i]);
  float inv;
  const float s = block_scale(m, &inv);
  float top = 0.0f;
  const i64 plane = (i64)x.heads * p.T * DP;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const i64 t = (i64)tile * 128 + i * kRows + r0;
    const float4 y = make_float4(v[i].x * s, v[i].y * s, v[i].z * s, v[i].w * s);
    float ss = y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    top = fmaxf(top, ss);
    if (t < p.T) {
      uint2 hi, lo;
      split2_finite(y.x, y.y, &hi.x, &lo.x);
      split2_finite(y.z, y.w, &hi.y, &lo.y);
      __half* to = x.planes + ((i64)h * p.T + t) * DP + c;
      *reinterpret_cast<uint2*>(to) = hi;
      *reinterpret_cast<uint2*>(to + plane) = lo;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  __syncthreads();
  if (lane == 0) red[wid] = top;
  __syncthreads();
  const i64 at = (i64)h * p.tiles + tile;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, red[i]);
    x.inv[at] = inv;
    x.len[at] = sqrtf(top) * inv;
  }
  if (threadIdx.x < 4) x.bad[at * 4 + threadIdx.x] = bad[threadIdx.x];
}

// ---- what the three kernels share -------------------------------------------------------------------------------------------------
// A tile of ROWS rows in shared memory: hi plane, lo plane, each of DP / 64 chunks of ROWS x 128 bytes.
template <int ROWS, int DP> __device__ constexpr int plane_bytes() { return ROWS * DP * 2; }
template <int ROWS, int DP>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int row, int head) {
  mbar_arrive_expect_tx(bar, 2 * plane_bytes<ROWS, DP>());
#pragma unroll
  for (int pl = 0; pl < 2; ++pl)
#pragma unroll
    for (int c = 0; c < DP / 64; ++c) tma_load_4d(dst + pl * plane_bytes<ROWS, DP>() + c * ROWS * 128, map, bar, c * 64, row, head, pl);
}
// D[128, N] = A[128, DP] B[N, DP]^T, both K-major tiles; the cross products first
template <int N, int DP>
__device__ __forceinline__ void product_rows(uint32_t d, uint32_t a, uint32_t b) {
  const uint32_t idesc = idesc16(128, N, 0, 0);
  const uint64_t ah = desc16(a, 0), al = desc16(a + plane_bytes<128, DP>(), 0), bh = desc16(b, 0), bl = desc16(b + plane_bytes<N, DP>(), 0);
  uint32_t on = 0;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    const uint64_t oa = ((k >> 2) * 128 * 128 + (k & 3) * 32) >> 4, ob = ((k >> 2) * N * 128 + (k & 3) * 32) >> 4;
    mma_f16(d, al + oa, bh + ob, idesc, on);
    on = 1;
    mma_f16(d, ah + oa, bl + ob, idesc, 1);
  }
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    const uint64_t oa = ((k >> 2) * 128 * 128 + (k & 3) * 32) >> 4, ob = ((k >> 2) * N * 128 + (k & 3) * 32) >> 4;
    mma_f16(d, ah + oa, bh + ob, idesc, 1);
  }
}
// D[128, DP] = A[128, K] B[K, DP], A in tensor memory (per half of the columns: K / 4 columns of hi, then of lo), B a tile of K rows
template <int K, int DP>
__device__ __forceinline__ void product_cols(uint32_t d, uint32_t a, uint32_t b) {
  const uint32_t idesc = idesc16(128, DP, 0, 1);
  const uint64_t bh = desc16(b, K * 128), bl = desc16(b + plane_bytes<K, DP>(), K * 128);
  uint32_t on = 0;
#pragma unroll
  for (int k = 0; k < K / 16; ++k) {
    const uint32_t hi = a + (k / (K / 32)) * (K / 2) + (k % (K / 32)) * 8, lo = hi + K / 4;
    mma_f16_ta(d, lo, bh + k * 128, idesc, on);
    on = 1;
    mma_f16_ta(d, hi, bl + k * 128, idesc, 1);
  }
#pragma unroll
  for (int k = 0; k < K / 16; ++k) {
    const uint32_t hi = a + (k / (K / 32)) * (K / 2) + (k % (K / 32)) * 8;
    mma_f16_ta(d, hi, bh + k * 128, idesc, 1);
  }
}
// 16 columns of this thread's lane, from registers
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
// the half W of a row's columns as the left operand of product_cols: W / 2 columns of hi, W / 2 of lo
template <int W>
__device__ __forceinline__ void store_operand(uint32_t taddr, const float (&v)[W]) {
#pragma unroll
  for (int i = 0; i < W; i += 32) {
    uint32_t hi[16], lo[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) split2_finite(v[i + 2 * j], v[i + 2 * j + 1], &hi[j], &lo[j]);
    tmem_st16(taddr + i / 2, hi);
    tmem_st16(taddr + W / 2 + i / 2, lo);
  }
}
template <int W>
__device__ __forceinline__ void load_row(uint32_t taddr, float (&v)[W]) {
#pragma unroll
  for (int i = 0; i < W; i += 32) tmem_ld32(taddr + i, reinterpret_cast<uint32_t*>(v) + i);
  tmem_wait_ld();
}
// acc = acc * keep + part * f over this thread's half of an accumulator
template <int W>
__device__ __forceinline__ void add_part(uint32_t taddr, float (&acc)[W], float keep, float f) {
#pragma unroll
  for (int i = 0; i < W; i += 32) {
    uint32_t v[32];
    tmem_ld32(taddr + i, v);
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 32; ++j) acc[i + j] = fmaf(__uint_as_float(v[j]), f, acc[i + j] * keep);
  }
}
// this thread's half of a row of the result, components [c0, c0 + W) of dk
template <int W>
__device__ __forceinline__ void store_row(float* row, const float (&acc)[W], int c0, int dk, float f) {
  if ((dk & 3) == 0) {
#pragma unroll
    for (int i = 0; i < W; i += 4)
      if (c0 + i < dk) *reinterpret_cast<float4*>(row + c0 + i) = make_float4(acc[i] * f, acc[i + 1] * f, acc[i + 2] * f, acc[i + 3] * f);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) if (c0 + i < dk) row[c0 + i] = acc[i] * f;
  }
}
__device__ __forceinline__ void tmem_alloc(uint32_t* slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(512u) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}
// copies already issued get a bounded time to land before a CTA that gave up exits
__device__ __forceinline__ void let_land(uint64_t* bars, int n) {
  for (int i = 0; i < n; ++i) {
    uint32_t addr = smem_u32(&bars[i]), done = 0;
    for (uint32_t k = 0; k < (1u << 14) && !done; ++k)
      asm volatile("{\n\t.reg .pred q;\n\tmbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(done) : "r"(addr), "r"(0u) : "memory");
  }
}
// smallest and largest of an int over the first 128 threads, for all of the CTA
__device__ __forceinline__ void range_of(int v, int* lo, int* hi, int* sm) {
  if (threadIdx.x == 0) { sm[0] = 0x7fffffff; sm[1] = -1; }
  __syncthreads();
  if (threadIdx.x < 128) {
    const int a = __reduce_min_sync(0xffffffffu, v), b = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) { atomicMin(&sm[0], a); atomicMax(&sm[1], b); }
  }
  __syncthreads();
  *lo = sm[0]; *hi = sm[1];
}

struct Side { const float* inv; const float* len; const uint32_t* bad; };
struct AttnParams {
  int T, tiles, hq, hk, dk;
  float scale;
  const int* begin; const int* end;
  Side q, k, v, g;
  const float* lse2; const float* delta;      // [hq][tiles * 128]
  float* out; float* lse;                     // forward: o, lse; backward: the gradient
  int* err;
};

// ---- forward ----------------------------------------------------------------------------------------------------------------------
template <int DP> struct FwdSmem {
  static constexpr int kTile = 2 * plane_bytes<128, DP>(), kStages = DP == 64 ? 2 : 1;
  static constexpr int kBars = 1 + 4 * kStages + 2 + 1 + 1;
  static constexpr int kTotal = 1024 + kTile * (1 + 2 * kStages) + 512 * 4 + kBars * 8 + 64;
};
template <int DP>
__global__ void __launch_bounds__(kThreads, 1)
k_forward(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnParams p) {
  using L = FwdSmem<DP>;
  constexpr int NS = L::kStages, W = DP / 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *sq = smem, *sk = smem + L::kTile, *sv = sk + NS * L::kTile;
  float* xchg = (float*)(sv + NS * L::kTile);                 // [2 tiles][2 halves][128]
  uint64_t* bars = (uint64_t*)(xchg + 512);
  uint64_t *b_q = bars, *b_kfull = bars + 1, *b_vfull = b_kfull + NS, *b_kfree = b_vfull + NS, *b_vfree = b_kfree + NS, *b_s = b_vfree + NS, *b_p = b_s + 2, *b_o = b_p + 1;
  int* ints = (int*)(b_o + 1);
  uint32_t* tmem_slot = (uint32_t*)ints + 2;
  volatile int* abort_flag = ints + 3;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.x % p.hq, hk = h / (p.hq / p.hk), qt = p.tiles - 1 - (int)(blockIdx.x / p.hq);      // long tiles first
  if (threadIdx.x == 0) {
    mbar_init(b_q, 1);
    for (int i = 0; i < NS; ++i) { mbar_init(&b_kfull[i], 1); mbar_init(&b_vfull[i], 1); mbar_init(&b_kfree[i], 1); mbar_init(&b_vfree[i], 1); }
    mbar_init(&b_s[0], 1); mbar_init(&b_s[1], 1); mbar_init(b_p, 8); mbar_init(b_o, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(tmem_slot);
  const int first = threadIdx.x < 128 && qt * 128 + (int)threadIdx.x < p.T ? p.begin[qt * 128 + threadIdx.x] : p.T;
  int b_min, b_max;
  range_of(first, &b_min, &b_max, ints);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_s = tmem, t_p = tmem + 256, t_o = tmem + 384;
  const int kb0 = b_min < p.T ? b_min / 128 : qt + 1, n = qt + 1 - kb0;      // key tiles (none: no row of the tile has a segment)

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      bool ok = true;
      load_tile<128, DP>(sq, &map_q, b_q, qt * 128, h);
      for (int j = 0; j < n && ok; ++j) {
        const int st = j % NS, ph = ((j / NS) - 1) & 1;
        if (j >= NS) ok = mbar_wait(&b_kfree[st], ph, abort_flag);
        if (!ok) break;
        load_tile<128, DP>(sk + st * L::kTile, &map_k, &b_kfull[st], (kb0 + j) * 128, hk);
        if (j >= NS) ok = mbar_wait(&b_vfree[st], ph, abort_flag);
        if (!ok) break;
        load_tile<128, DP>(sv + st * L::kTile, &map_v, &b_vfull[st], (kb0 + j) * 128, hk);
      }
      if (*abort_flag) let_land(bars, 1 + 2 * NS);
    }
  } else if (warp == 1) {
    if (lane == 0 && n > 0) {
      bool ok = mbar_wait(b_q, 0, abort_flag);
      auto scores = [&](int j) -> bool {
        const int st = j % NS;
        if (!mbar_wait(&b_kfull[st], (j / NS) & 1, abort_flag)) return false;
        tc_fence_after();
        product_rows<128, DP>(t_s + (j & 1) * 128, smem_u32(sq), smem_u32(sk + st * L::kTile));
        mma_commit(&b_kfree[st]);
        mma_commit(&b_s[j & 1]);
        return true;
      };
      if (ok) ok = scores(0);
      if (ok && n > 1) ok = scores(1);
      for (int j = 0; j < n && ok; ++j) {
        const int st = j % NS;
        ok = mbar_wait(b_p, j & 1, abort_flag) && mbar_wait(&b_vfull[st], (j / NS) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        product_cols<128, DP>(t_o, t_p, smem_u32(sv + st * L::kTile));
        mma_commit(&b_vfree[st]);
        mma_commit(b_o);
        if (j + 2 < n) ok = scores(j + 2);      // (this tile's scores have been read: P says so)
      }
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2, row = quarter * 32 + lane, t = qt * 128 + row;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const int begin = t < p.T ? p.begin[t] : p.T;
    const i64 kvt = (i64)hk * p.tiles;
    const float sc0 = p.scale * kL2e * p.q.inv[(i64)h * p.tiles + qt];
    float acc[W], m = -INFINITY, l = 0.0f, keep = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] = 0.0f;
    bool ok = true;                             // (a wait that ran out does not end the loop: the other half of the rows meets this one in it)
    for (int j = 0; j < n; ++j) {
      const int kb = kb0 + j, c0 = kb * 128 + half * 64;
      const float sc = fmaxf(sc0 * p.k.inv[kvt + kb], 1e-37f);      // (masked scores are -infinity times this)
      ok = mbar_wait(&b_s[j & 1], (j >> 1) & 1, abort_flag) && ok;
      tc_fence_after();
      float v[64];
      load_row<64>(t_s + (j & 1) * 128 + half * 64 + lane_off, v);
      if (kb == qt || kb * 128 < b_max) {       // the diagonal or the begin of a segment crosses the tile
        const int a = begin - c0, z = t - c0;
#pragma unroll
        for (int i = 0; i < 64; ++i) if (i < a || i > z) v[i] = -INFINITY;
      }
      const uint32_t* kb_bad = p.k.bad + (kvt + kb) * 4 + half * 2;
      const uint32_t* vb_bad = p.v.bad + (kvt + kb) * 4 + half * 2;
      const uint32_t bad0 = kb_bad[0] | vb_bad[0], bad1 = kb_bad[1] | vb_bad[1];
      if (bad0 | bad1) {                        // a visible key or value that is not finite
        for (int i = 0; i < 64; ++i)
          if (((i < 32 ? bad0 >> i : bad1 >> (i - 32)) & 1) && c0 + i >= begin && c0 + i <= t) l = __int_as_float(0x7fffffff);
      }
      float bm = v[0];
#pragma unroll
      for (int i = 1; i < 64; ++i) bm = fmaxf(bm, v[i]);
      float* x = xchg + (j & 1) * 256;
      x[half * 128 + row] = bm;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");      // the two halves of these rows
      bm = fmaxf(bm, x[(1 - half) * 128 + row]) * sc;
      const float mn = fmaxf(m, bm), ref = mn > -INFINITY ? mn : 0.0f;
      const float shrink = m > -INFINITY ? exp2_fast(m - ref) : 0.0f;
      const float off = 14.0f - ref;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 64; ++i) { v[i] = exp2_fast(fmaf(v[i], sc, off)); sum += v[i]; }
      l = l * shrink + sum;
      m = mn;
      if (j > 0) {                              // the last tile's product has read P and is in its accumulator
        ok = mbar_wait(b_o, (j - 1) & 1, abort_flag) && ok;
        tc_fence_after();
        add_part<W>(t_o + half * W + lane_off, acc, keep, p.v.inv[kvt + kb - 1]);
      }
      store_operand<64>(t_p + half * 64 + lane_off, v);
      keep = shrink;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(b_p);
    }
    if (n > 0) {
      ok = mbar_wait(b_o, (n - 1) & 1, abort_flag) && ok;
      tc_fence_after();
      add_part<W>(t_o + half * W + lane_off, acc, keep, p.v.inv[kvt + qt]);
    }
    {
      float* x = xchg + (n & 1) * 256;
      x[half * 128 + row] = l;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
      l += x[(1 - half) * 128 + row];
      if (ok && t < p.T) {
        const uint32_t qbad = p.q.bad[((i64)h * p.tiles + qt) * 4 + quarter];
        if (begin <= t && ((qbad >> lane) & 1)) l = __int_as_float(0x7fffffff);
        const bool dead = l == 0.0f;
        store_row<W>(p.out + ((i64)t * p.hq + h) * p.dk, acc, half * W, p.dk, dead ? 0.0f : 1.0f / l);
        if (half == 0 && p.lse) p.lse[(i64)h * p.T + t] = dead ? -INFINITY : (m - 14.0f) * kLn2 + logf(l);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_free(tmem); }
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.err, ERRBIT_WAIT_TIMEOUT);
}

// ---- dV ---------------------------------------------------------------------------------------------------------------------------
// One CTA per 128 keys of a key head.  Steps: every query head of the group x every tile of 128 queries from the keys' own to the last
// one that sees them.
template <int DP> struct GradVSmem {
  static constexpr int kTile = 2 * plane_bytes<128, DP>(), kStages = DP == 64 ? 2 : 1;
  static constexpr int kBars = 1 + 4 * kStages + 2 + 1 + 1;
  static constexpr int kTotal = 1024 + kTile * (1 + 2 * kStages) + kBars * 8 + 64;
};
template <int DP>
__global__ void __launch_bounds__(kThreads, 1)
k_grad_v(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_g, const __grid_constant__ AttnParams p) {
  using L = GradVSmem<DP>;
  constexpr int NS = L::kStages, W = DP / 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *sk = smem, *sq = smem + L::kTile, *sg = sq + NS * L::kTile;
  uint64_t* bars = (uint64_t*)(sg + NS * L::kTile);
  uint64_t *b_k = bars, *b_qfull = bars + 1, *b_gfull = b_qfull + NS, *b_qfree = b_gfull + NS, *b_gfree = b_qfree + NS, *b_s = b_gfree + NS, *b_p = b_s + 2, *b_o = b_p + 1;
  int* ints = (int*)(b_o + 1);
  uint32_t* tmem_slot = (uint32_t*)ints + 2;
  volatile int* abort_flag = ints + 3;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = blockIdx.x % p.hk, kt = blockIdx.x / p.hk, group = p.hq / p.hk;
  if (threadIdx.x == 0) {
    mbar_init(b_k, 1);
    for (int i = 0; i < NS; ++i) { mbar_init(&b_qfull[i], 1); mbar_init(&b_gfull[i], 1); mbar_init(&b_qfree[i], 1); mbar_init(&b_gfree[i], 1); }
    mbar_init(&b_s[0], 1); mbar_init(&b_s[1], 1); mbar_init(b_p, 8); mbar_init(b_o, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(tmem_slot);
  const int last = threadIdx.x < 128 && kt * 128 + (int)threadIdx.x < p.T ? p.end[kt * 128 + threadIdx.x] : 0;
  int e_min, e_max;
  range_of(last, &e_min, &e_max, ints);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_s = tmem, t_p = tmem + 256, t_o = tmem + 384;
  const int per = e_max > 0 ? (e_max - 1) / 128 - kt + 1 : 0, n = per * group;

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      bool ok = true;
      load_tile<128, DP>(sk, &map_k, b_k, kt * 128, hk);
      for (int j = 0; j < n && ok; ++j) {
        const int st = j % NS, ph = ((j / NS) - 1) & 1, h = hk * group + j / per, i = kt + j % per;
        if (j >= NS) ok = mbar_wait(&b_qfree[st], ph, abort_flag);
        if (!ok) break;
        load_tile<128, DP>(sq + st * L::kTile, &map_q, &b_qfull[st], i * 128, h);
        if (j >= NS) ok = mbar_wait(&b_gfree[st], ph, abort_flag);
        if (!ok) break;
        load_tile<128, DP>(sg + st * L::kTile, &map_g, &b_gfull[st], i * 128, h);
      }
      if (*abort_flag) let_land(bars, 1 + 2 * NS);
    }
  } else if (warp == 1) {
    if (lane == 0 && n > 0) {
      bool ok = mbar_wait(b_k, 0, abort_flag);
      auto scores = [&](int j) -> bool {
        const int st = j % NS;
        if (!mbar_wait(&b_qfull[st], (j / NS) & 1, abort_flag)) return false;
        tc_fence_after();
        product_rows<128, DP>(t_s + (j & 1) * 128, smem_u32(sk), smem_u32(sq + st * L::kTile));
        mma_commit(&b_qfree[st]);
        mma_commit(&b_s[j & 1]);
        return true;
      };
      if (ok) ok = scores(0);
      if (ok && n > 1) ok = scores(1);
      for (int j = 0; j < n && ok; ++j) {
        const int st = j % NS;
        ok = mbar_wait(b_p, j & 1, abort_flag) && mbar_wait(&b_gfull[st], (j / NS) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        product_cols<128, DP>(t_o, t_p, smem_u32(sg + st * L::kTile));
        mma_commit(&b_gfree[st]);
        mma_commit(b_o);
        if (j + 2 < n) ok = scores(j + 2);
      }
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2, row = quarter * 32 + lane, t = kt * 128 + row;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const int end = t < p.T ? p.end[t] : 0;
    const float sc0 = p.scale * kL2e * p.k.inv[(i64)hk * p.tiles + kt];
    float acc[W], f_last = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] = 0.0f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const i64 at = (i64)(hk * group + j / per) * p.tiles + kt + j % per;
      const int i0 = (kt + j % per) * 128, c0 = i0 + half * 64;
      const float sc = sc0 * p.q.inv[at];
      const float4* lse = reinterpret_cast<const float4*>(p.lse2 + at * 128 + half * 64);
      if (!mbar_wait(&b_s[j & 1], (j >> 1) & 1, abort_flag)) { ok = false; break; }
      tc_fence_after();
      float v[64];
      load_row<64>(t_s + (j & 1) * 128 + half * 64 + lane_off, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float4 x = lse[i];
        v[4 * i] = exp2_fast(fmaf(v[4 * i], sc, 14.0f - x.x)); v[4 * i + 1] = exp2_fast(fmaf(v[4 * i + 1], sc, 14.0f - x.y));
        v[4 * i + 2] = exp2_fast(fmaf(v[4 * i + 2], sc, 14.0f - x.z)); v[4 * i + 3] = exp2_fast(fmaf(v[4 * i + 3], sc, 14.0f - x.w));
      }
      if (i0 == kt * 128 || i0 + 128 > e_min) {
        const int a = t - c0, z = end - c0;
#pragma unroll
        for (int i = 0; i < 64; ++i) if (i < a || i >= z) v[i] = 0.0f;
      }
      if (j > 0) {
        if (!mbar_wait(b_o, (j - 1) & 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        add_part<W>(t_o + half * W + lane_off, acc, 1.0f, f_last);
      }
      store_operand<64>(t_p + half * 64 + lane_off, v);
      f_last = p.g.inv[at];
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(b_p);
    }
    if (ok && n > 0) {
      ok = mbar_wait(b_o, (n - 1) & 1, abort_flag);
      if (ok) {
        tc_fence_after();
        add_part<W>(t_o + half * W + lane_off, acc, 1.0f, f_last);
      }
    }
    if (ok && t < p.T) store_row<W>(p.out + ((i64)t * p.hk + hk) * p.dk, acc, half * W, p.dk, 1.0f / 16384.0f);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_free(tmem); }
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.err, ERRBIT_WAIT_TIMEOUT);
}

// ---- dQ and dK --------------------------------------------------------------------------------------------------------------------
// X (128 rows, resident: q and do, or k and v), Y streamed in tiles of N rows (k and v, or q and do):
//   S = X1 Y1^T, dP = X2 Y2^T, dS = p (dP - delta), result += dS Y1.
// dS goes where S was; S has two buffers, so the next tile's S and dP are formed while dS Y1 runs.
template <int DP> struct GradSmem {
  static constexpr int N = DP == 64 ? 128 : 64;                       // 128-wide heads: 64 rows of Y at a time fit beside X
  static constexpr int kTileX = 2 * plane_bytes<128, DP>(), kTileY = 2 * plane_bytes<N, DP>();
  static constexpr int kStages2 = DP == 64 ? 2 : 1;                   // Y1 is held through the last product (two tiles), Y2 is not
  static constexpr int kBars = 2 + 4 + 2 * kStages2 + 2 + 1 + 1 + 1;
  static constexpr int kTotal = 1024 + 2 * kTileX + (2 + kStages2) * kTileY + kBars * 8 + 64;
};
template <int DP, bool DK>
__global__ void __launch_bounds__(kThreads, 1)
k_grad_qk(const __grid_constant__ CUtensorMap map_x1, const __grid_constant__ CUtensorMap map_x2, const __grid_constant__ CUtensorMap map_y1,
          const __grid_constant__ CUtensorMap map_y2, const __grid_constant__ AttnParams p) {
  using L = GradSmem<DP>;
  constexpr int N = L::N, H = N / 2, W = DP / 2, NS2 = L::kStages2, R = 128 / N;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *x1 = smem, *x2 = x1 + L::kTileX, *y1 = x2 + L::kTileX, *y2 = y1 + 2 * L::kTileY;
  uint64_t* bars = (uint64_t*)(y2 + NS2 * L::kTileY);
  uint64_t *b_x = bars, *b_y1full = bars + 2, *b_y2full = b_y1full + 2, *b_y1free = b_y2full + NS2, *b_y2free = b_y1free + 2, *b_s = b_y2free + NS2, *b_dp = b_s + 2,
           *b_ds = b_dp + 1, *b_o = b_ds + 1;
  int* ints = (int*)(b_o + 1);
  uint32_t* tmem_slot = (uint32_t*)ints + 2;
  volatile int* abort_flag = ints + 3;
  float* vmax_slot = (float*)ints + 4;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.hq / p.hk, heads = DK ? p.hk : p.hq, hx = blockIdx.x % heads, hk = DK ? hx : hx / group;
  const int xt = DK ? blockIdx.x / heads : p.tiles - 1 - (int)(blockIdx.x / heads);
  if (threadIdx.x == 0) {
    mbar_init(&b_x[0], 1); mbar_init(&b_x[1], 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&b_y1full[i], 1); mbar_init(&b_y1free[i], 1); mbar_init(&b_s[i], 1); }
    for (int i = 0; i < NS2; ++i) { mbar_init(&b_y2full[i], 1); mbar_init(&b_y2free[i], 1); }
    mbar_init(b_dp, 1); mbar_init(b_ds, 8); mbar_init(b_o, 1);
    *abort_flag = 0;
    *vmax_slot = 0.0f;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(tmem_slot);
  const int tx = xt * 128 + (int)threadIdx.x;
  const int edge = DK ? (threadIdx.x < 128 && tx < p.T ? p.end[tx] : 0) : (threadIdx.x < 128 && tx < p.T ? p.begin[tx] : p.T);
  int e_min, e_max;
  range_of(edge, &e_min, &e_max, ints);
  {   // longest value row of the head: the scale of dS has to hold |do| |v| twice
    float m = 0.0f;
    for (int i = threadIdx.x; i < p.tiles; i += kThreads) m = fmaxf(m, p.v.len[(i64)hk * p.tiles + i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) atomicMax((int*)vmax_slot, __float_as_int(m));      // (not negative: ordered like its bits)
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_s = tmem, t_dp = tmem + 256, t_o = tmem + 384;
  const float vmax = *vmax_slot;
  // tiles of Y, in steps of N rows
  int y0, per;
  if (DK) { y0 = xt * R; per = e_max > 0 ? (e_max - 1) / N - y0 + 1 : 0; }
  else { const int last = xt * 128 + 127 < p.T ? xt * 128 + 127 : p.T - 1; y0 = e_min / N; per = e_min < p.T ? last / N - y0 + 1 : 0; }
  const int n = DK ? per * group : per;

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      bool ok = true;
      load_tile<128, DP>(x1, &map_x1, &b_x[0], xt * 128, hx);
      for (int j = 0; j < n && ok; ++j) {
        const int hy = DK ? hk * group + j / per : hk, y = (y0 + (DK ? j % per : j)) * N;
        if (j >= 2) ok = mbar_wait(&b_y1free[j & 1], ((j >> 1) - 1) & 1, abort_flag);
        if (!ok) break;
        load_tile<N, DP>(y1 + (j & 1) * L::kTileY, &map_y1, &b_y1full[j & 1], y, hy);
        if (j == 0) load_tile<128, DP>(x2, &map_x2, &b_x[1], xt * 128, hx);
        const int st = j % NS2;
        if (j >= NS2) ok = mbar_wait(&b_y2free[st], ((j / NS2) - 1) & 1, abort_flag);
        if (!ok) break;
        load_tile<N, DP>(y2 + st * L::kTileY, &map_y2, &b_y2full[st], y, hy);
      }
      if (*abort_flag) let_land(bars, 4 + NS2);
    }
  } else if (warp == 1) {
    if (lane == 0 && n > 0) {
      bool ok = mbar_wait(&b_x[0], 0, abort_flag);
      auto scores = [&](int j) -> bool {      // (buffer j & 1 held dS of tile j - 2, which its product has read)
        if (!mbar_wait(&b_y1full[j & 1], (j >> 1) & 1, abort_flag)) return false;
        if (j >= 2 && !mbar_wait(b_o, j & 1, abort_flag)) return false;
        tc_fence_after();
        product_rows<N, DP>(t_s + (j & 1) * 128, smem_u32(x1), smem_u32(y1 + (j & 1) * L::kTileY));
        mma_commit(&b_s[j & 1]);
        return true;
      };
      auto other = [&](int j) -> bool {
        const int st = j % NS2;
        if (!mbar_wait(&b_y2full[st], (j / NS2) & 1, abort_flag)) return false;
        tc_fence_after();
        product_rows<N, DP>(t_dp, smem_u32(x2), smem_u32(y2 + st * L::kTileY));
        mma_commit(&b_y2free[st]);
        mma_commit(b_dp);
        return true;
      };
      if (ok) ok = scores(0) && mbar_wait(&b_x[1], 0, abort_flag) && other(0);
      if (ok && n > 1) ok = scores(1);
      for (int j = 0; j < n && ok; ++j) {
        ok = mbar_wait(b_ds, j & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (j + 1 < n) ok = other(j + 1);
        if (!ok) break;
        product_cols<N, DP>(t_o, t_s + (j & 1) * 128, smem_u32(y1 + (j & 1) * L::kTileY));
        mma_commit(&b_y1free[j & 1]);
        mma_commit(b_o);
        if (j + 2 < n) ok = scores(j + 2);
      }
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2, row = quarter * 32 + lane, t = xt * 128 + row;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const int mine = DK ? (t < p.T ? p.end[t] : 0) : (t < p.T ? p.begin[t] : p.T);
    const i64 x_at = (i64)hx * p.tiles + xt, v_row = (i64)hk * p.tiles;
    const float s_x = p.scale * kL2e * (DK ? p.k.inv[x_at] : p.q.inv[x_at]);
    // 2^e with 2 |do| |v| 2^e below 2^14, and its inverse
    auto ds_scale = [&](float len, float* inverse) -> float {
      const float b = 2.0f * len * vmax;
      int e = b > 0.0f ? 13 - ((int)(__float_as_uint(b) >> 23) - 127) : 0;
      e = e > 100 ? 100 : (e < -100 ? -100 : e);
      *inverse = __uint_as_float((uint32_t)(127 - e) << 23);
      return __uint_as_float((uint32_t)(127 + e) << 23);
    };
    float back, f_last = 0.0f, lse_row = 0.0f, delta_row = 0.0f, f2 = 0.0f, fx = 0.0f;
    if (!DK) {
      f2 = ds_scale(p.g.len[x_at], &back) * (1.0f / 16384.0f);      // (p carries 2^14)
      fx = p.g.inv[x_at] * f2;
      lse_row = 14.0f - p.lse2[x_at * 128 + row];
      delta_row = p.delta[x_at * 128 + row] * f2;
    }
    float acc[W];
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] = 0.0f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int hy = DK ? hk * group + j / per : hk, y = (y0 + (DK ? j % per : j)) * N, c0 = y + half * H;
      const i64 y_at = (i64)hy * p.tiles + y / 128;
      const float sc = s_x * (DK ? p.q.inv[y_at] : p.k.inv[y_at]);
      float f1, f_this;
      const float4 *lse4 = nullptr, *delta4 = nullptr;
      if (DK) {
        f2 = ds_scale(p.g.len[y_at], &back) * (1.0f / 16384.0f);
        f1 = p.g.inv[y_at] * f2 * p.v.inv[x_at];
        f_this = p.q.inv[y_at] * back;
        lse4 = reinterpret_cast<const float4*>(p.lse2 + (i64)hy * p.tiles * 128 + c0);
        delta4 = reinterpret_cast<const float4*>(p.delta + (i64)hy * p.tiles * 128 + c0);
      } else {
        f1 = fx * p.v.inv[y_at];
        f_this = p.k.inv[y_at] * back;
      }
      if (!mbar_wait(&b_s[j & 1], (j >> 1) & 1, abort_flag)) { ok = false; break; }
      tc_fence_after();
      float v[H];
      load_row<H>(t_s + (j & 1) * 128 + half * H + lane_off, v);
      if (DK) {
#pragma unroll
        for (int i = 0; i < H / 4; ++i) {
          const float4 x = lse4[i];
          v[4 * i] = exp2_fast(fmaf(v[4 * i], sc, 14.0f - x.x)); v[4 * i + 1] = exp2_fast(fmaf(v[4 * i + 1], sc, 14.0f - x.y));
          v[4 * i + 2] = exp2_fast(fmaf(v[4 * i + 2], sc, 14.0f - x.z)); v[4 * i + 3] = exp2_fast(fmaf(v[4 * i + 3], sc, 14.0f - x.w));
        }
      } else {
#pragma unroll
        for (int i = 0; i < H; ++i) v[i] = exp2_fast(fmaf(v[i], sc, lse_row));
      }
      const bool crossed = DK ? y < xt * 128 + 128 || y + N > e_min : y + N > xt * 128 || y < e_max;
      if (!mbar_wait(b_dp, j & 1, abort_flag)) { ok = false; break; }
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < H; c += 32) {
        uint32_t d[32];
        tmem_ld32(t_dp + half * H + c + lane_off, d);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          float4 de = make_float4(delta_row, delta_row, delta_row, delta_row);
          if (DK) { de = delta4[(c + i) / 4]; de.x *= f2; de.y *= f2; de.z *= f2; de.w *= f2; }
          v[c + i] *= fmaf(__uint_as_float(d[i]), f1, -de.x); v[c + i + 1] *= fmaf(__uint_as_float(d[i + 1]), f1, -de.y);
          v[c + i + 2] *= fmaf(__uint_as_float(d[i + 2]), f1, -de.z); v[c + i + 3] *= fmaf(__uint_as_float(d[i + 3]), f1, -de.w);
        }
      }
      if (crossed) {
        const int a = (DK ? t : mine) - c0, z = (DK ? mine - 1 : t) - c0;
#pragma unroll
        for (int i = 0; i < H; ++i) if (i < a || i > z) v[i] = 0.0f;
      }
      if (j > 0) {
        if (!mbar_wait(b_o, (j - 1) & 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        add_part<W>(t_o + half * W + lane_off, acc, 1.0f, f_last);
      }
      // (both halves of these rows have read S before either writes dS over it: dS of a half lies within its own half of S)
      store_operand<H>(t_s + (j & 1) * 128 + half * H + lane_off, v);
      f_last = f_this;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(b_ds);
    }
    if (ok && n > 0) {
      ok = mbar_wait(b_o, (n - 1) & 1, abort_flag);
      if (ok) {
        tc_fence_after();
        add_part<W>(t_o + half * W + lane_off, acc, 1.0f, f_last);
      }
    }
    if (ok && t < p.T) store_row<W>(p.out + ((i64)t * (DK ? p.hk : p.hq) + hx) * p.dk, acc, half * W, p.dk, p.scale);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_free(tmem); }
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.err, ERRBIT_WAIT_TIMEOUT);
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) return (EncodeTiledFn)p;
    cudaGetLastError();
    return (EncodeTiledFn) nullptr;
  }();
  return fn;
}
int make_map(CUtensorMap* map, const PlanesDev& x, int T, int dp, int rows) {
  if (!encode_fn()) return set_error(VB_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t row = (cuuint64_t)dp * 2;
  cuuint64_t dims[4] = {(cuuint64_t)dp, (cuuint64_t)T, (cuuint64_t)x.heads, 2}, strides[3] = {row, row * T, row * T * x.heads};
  cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, estr[4] = {1, 1, 1, 1};
  CUresult r = encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, x.planes, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(VB_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
  return VB_OK;
}

// Workspace of a call: the planes of q, k, v (and do), their per-tile values, the rows' segments.
struct Work {
  Temp hold;
  PrepareDev prep{};
  AttnParams p{};
  int dp = 64;
};
int prepare(const SegShape& s, const SegHeads* in, const int* heads, int n, const float* starts, i64 n_seg, const SegHeads* o, const float* lse, Work& w) {
  const int tiles = (int)((s.T + 127) / 128), dp = s.dk <= 64 ? 64 : 128;
  w.dp = dp;
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t a = at; at += (bytes + 255) / 256 * 256; return a; };
  size_t planes[4], inv[4], len[4], bad[4];
  for (int i = 0; i < n; ++i) {
    planes[i] = take((size_t)2 * heads[i] * s.T * dp * 2);
    inv[i] = take((size_t)heads[i] * tiles * 4); len[i] = take((size_t)heads[i] * tiles * 4); bad[i] = take((size_t)heads[i] * tiles * 16);
  }
  const size_t begin = take((size_t)s.T * 4), end = take((size_t)s.T * 4);
  const size_t delta = o ? take((size_t)s.hq * tiles * 512) : 0, lse2 = o ? take((size_t)s.hq * tiles * 512) : 0;
  VB_TRY(scratch_alloc(at, &w.hold.p));
  uint8_t* base = (uint8_t*)w.hold.p;
  PrepareDev& d = w.prep;
  d.n = n; d.T = (int)s.T; d.tiles = tiles; d.dk = s.dk; d.hq = s.hq;
  Side* sides[4] = {&w.p.q, &w.p.k, &w.p.v, &w.p.g};
  int all = 0;
  for (int i = 0; i < n; ++i) {
    d.in[i] = PlanesDev{in[i].p, in[i].st, in[i].sh, (__half*)(base + planes[i]), (float*)(base + inv[i]), (float*)(base + len[i]), (uint32_t*)(base + bad[i]), heads[i],
                        s.dk % 4 == 0 && in[i].st % 4 == 0 && in[i].sh % 4 == 0 && (reinterpret_cast<uintptr_t>(in[i].p) & 15) == 0};
    *sides[i] = Side{d.in[i].inv, d.in[i].len, d.in[i].bad};
    all += heads[i];
  }
  d.starts = starts; d.n_seg = (int)n_seg; d.begin = (int*)(base + begin); d.end = (int*)(base + end); d.err = ctx().d_err;
  if (o) { d.o = o->p; d.o_st = o->st; d.o_sh = o->sh; d.lse = lse; d.delta = (float*)(base + delta); d.lse2 = (float*)(base + lse2); }
  AttnParams& p = w.p;
  p.T = (int)s.T; p.tiles = tiles; p.hq = s.hq; p.hk = s.hk; p.dk = s.dk; p.scale = s.scale;
  p.begin = d.begin; p.end = d.end; p.lse2 = d.lse2; p.delta = d.delta; p.err = ctx().d_err;
  ProfScope prof("segment_attn_prepare", 8.0 * (double)s.T * all * s.dk);
  if (dp == 64) k_prepare<64><<<dim3(tiles, all), 256, 0, ctx().stream>>>(d);
  else k_prepare<128><<<dim3(tiles, all), 256, 0, ctx().stream>>>(d);
  VB_LAUNCH_CHECK();
  return VB_OK;
}
template <class K>
int allow_smem(K kernel, int bytes) {
  VB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return VB_OK;
}

template <int DP>
int forward(Work& w) {
  static const int ready = allow_smem(k_forward<DP>, FwdSmem<DP>::kTotal);
  VB_TRY(ready);
  CUtensorMap mq, mk, mv;
  VB_TRY(make_map(&mq, w.prep.in[0], w.p.T, DP, 128)); VB_TRY(make_map(&mk, w.prep.in[1], w.p.T, DP, 128)); VB_TRY(make_map(&mv, w.prep.in[2], w.p.T, DP, 128));
  k_forward<DP><<<(unsigned)w.p.hq * w.p.tiles, kThreads, FwdSmem<DP>::kTotal, ctx().stream>>>(mq, mk, mv, w.p);
  VB_LAUNCH_CHECK();
  return VB_OK;
}
template <int DP>
int backward(Work& w, float* dq, float* dk, float* dv) {
  static const int ready_v = allow_smem(k_grad_v<DP>, GradVSmem<DP>::kTotal), ready_q = allow_smem(k_grad_qk<DP, false>, GradSmem<DP>::kTotal),
                   ready_k = allow_smem(k_grad_qk<DP, true>, GradSmem<DP>::kTotal);
  VB_TRY(ready_v); VB_TRY(ready_q); VB_TRY(ready_k);
  constexpr int N = GradSmem<DP>::N;
  CUtensorMap q, k, v, g, qn, kn, vn, gn;
  const PlanesDev* in = w.prep.in;
  VB_TRY(make_map(&q, in[0], w.p.T, DP, 128)); VB_TRY(make_map(&k, in[1], w.p.T, DP, 128)); VB_TRY(make_map(&v, in[2], w.p.T, DP, 128)); VB_TRY(make_map(&g, in[3], w.p.T, DP, 128));
  VB_TRY(make_map(&qn, in[0], w.p.T, DP, N)); VB_TRY(make_map(&kn, in[1], w.p.T, DP, N)); VB_TRY(make_map(&vn, in[2], w.p.T, DP, N)); VB_TRY(make_map(&gn, in[3], w.p.T, DP, N));
  w.p.out = dv;
  k_grad_v<DP><<<(unsigned)w.p.hk * w.p.tiles, kThreads, GradVSmem<DP>::kTotal, ctx().stream>>>(k, q, g, w.p);
  VB_LAUNCH_CHECK();
  w.p.out = dk;
  k_grad_qk<DP, true><<<(unsigned)w.p.hk * w.p.tiles, kThreads, GradSmem<DP>::kTotal, ctx().stream>>>(k, v, qn, gn, w.p);
  VB_LAUNCH_CHECK();
  w.p.out = dq;
  k_grad_qk<DP, false><<<(unsigned)w.p.hq * w.p.tiles, kThreads, GradSmem<DP>::kTotal, ctx().stream>>>(q, g, kn, vn, w.p);
  VB_LAUNCH_CHECK();
  return VB_OK;
}

}  // namespace

int launch_segment_attention(const SegShape& s, const SegHeads& q, const SegHeads& k, const SegHeads& v, const float* starts, i64 n, float* out, float* lse) {
  Work w;
  const SegHeads in[3] = {q, k, v};
  const int heads[3] = {s.hq, s.hk, s.hk};
  VB_TRY(prepare(s, in, heads, 3, starts, n, nullptr, nullptr, w));
  w.p.out = out; w.p.lse = lse;
  ProfScope prof("segment_attn", 2.0 * (double)s.T * (double)s.T * s.hq * s.dk);
  return w.dp == 64 ? forward<64>(w) : forward<128>(w);
}
int launch_segment_attention_backward(const SegShape& s, const SegHeads& q, const SegHeads& k, const SegHeads& v, const float* starts, i64 n,
                                      const SegHeads& out, const float* lse, const SegHeads& g, float* dq, float* dk, float* dv) {
  Work w;
  const SegHeads in[4] = {q, k, v, g};
  const int heads[4] = {s.hq, s.hk, s.hk, s.hq};
  VB_TRY(prepare(s, in, heads, 4, starts, n, &out, lse, w));
  ProfScope prof("segment_attn_bwd", 5.0 * (double)s.T * (double)s.T * s.hq * s.dk);
  return w.dp == 64 ? backward<64>(w, dq, dk, dv) : backward<128>(w, dq, dk, dv);
}

}  // namespace vb
