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
// The matrices of scores never leave the SM.  In every kernel a thread of the sixteen row warps holds a quarter of a row of the tile; the
// second product takes its left operand (P, dS; hi and lo) from tensor memory, where these warps write it, and its right
// operand from the same shared-memory tile that the first product read (MN-major instead of K-major).  The second product of each tile goes to a
// fresh accumulator that the warps add to their registers with the running rescale, so the accumulator's truncation (split16.cuh) never
// runs longer than a tile.
//   k_forward   S = Q K^T, softmax with a running maximum, O += P V
//   k_backward  dV: S^T = K Q^T, P^T from the saved lse, dV += P^T dO, over the query heads of the group (no atomics)
//               dQ: S = Q K^T, dP = dO V^T, dQ += dS K;  dK: the same with the roles of rows and columns exchanged
// Every wait is bounded; when one runs out the CTA raises the device error word, frees its tensor memory and returns.
//
// Bound by the tensor cores where texts are long (16384 tokens, 8 + 2 heads of 128: k_forward 1067 us, 517 TFLOP/s useful, 1550 issued, at the
// 1.53 GHz that the power limit leaves), by what a CTA does before its first tile and after its last where they are short: about 10 of 23
// thousand cycles for four tiles (4096 tokens in 9 texts, 16 + 4 heads of 64: k_forward 53 us, k_backward 130 to 146; 8 texts of 1024, 12 heads: 71), and by
// the chain of tiles of the longest text where there are fewer CTAs than SMs (1357 of 1531 tokens, 6 + 2 heads of 80: 35 and 66 us).
// 128 x 128 tiles and one CTA an SM: two streamed operands, four planes each, fill shared memory, and scores in two buffers with what
// follows from them tensor memory; two smaller CTAs an SM, and one that takes tiles from a counter, measured no better.
#include "segment_attention.h"
#include "split16.cuh"

namespace vb {
namespace {
using namespace tc;

constexpr int kGroups = 4, kRowWarps = 4 * kGroups, kThreads = 32 * (2 + kRowWarps);      // warp 0: TMA, warp 1: MMA, the others: rows
constexpr float kL2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float2 lo2(const float4& v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ float2 hi2(const float4& v) { return make_float2(v.z, v.w); }

// ---- planes ------------------------------------------------------------------------------------------------------------------------
// One of q, k, v, do: planes [2][heads][T][DP], and per head and tile the inverse scale (negative where a component is not finite), the
// largest row length and a bit for every row with a component that is not finite.
struct PlanesDev { const float* x; i64 st, sh; __half* planes; float* inv; float* len; uint32_t* bad; int heads; bool vec; };
struct PrepareDev {
  PlanesDev in[4];
  int n, T, tiles, dk, hq;
  const float* starts; int n_seg; int* begin; int* end; int4* plan; int* err;      // where the segment of each row begins and ends, and the tiles' order with their rows' ranges
  const float* o; i64 o_st, o_sh; bool o_vec; const float* lse;                     // for do: delta and 14 - lse in base 2, padded to whole tiles
  float* delta; float* lift;
  float* text_len;                                                                  // [key heads][T], for v: longest of the rows of t's text in t's tile
};

// The offset of the segment that row t is in (-1: none), as an index into the offsets.
__device__ __forceinline__ int segment_of(const PrepareDev& p, const float* starts, int t) {
  int lo = 0, hi = p.n_seg + 1;          // offsets [0, lo) are <= t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (roundf(starts[mid]) <= (float)t) lo = mid + 1; else hi = mid;
  }
  return lo > 0 && lo <= p.n_seg ? lo - 1 : -1;
}
// Where the segment of row t begins and ends (rows of no segment: (T, 0)); whatever the offsets are, inside [0, T].
__device__ __forceinline__ int2 segment_at(const PrepareDev& p, const float* starts, int t) {
  const int s = segment_of(p, starts, t);
  if (s < 0) return make_int2(p.T, 0);
  const float fb = roundf(starts[s]), fe = roundf(starts[s + 1]);
  const int b = fb > 0.0f ? (int)fb : 0, e = fe < (float)p.T ? (int)fe : p.T;
  return b <= t && t < e ? make_int2(b, e) : make_int2(p.T, 0);
}
// Offsets that decrease or leave [0, T] are reported.
__device__ __forceinline__ void check_offset(const float* starts, int i, int T, int* err) {
  const float s = starts[i];
  if (!(s > -0.5f)) atomicOr(err, ERRBIT_NEG_ID);
  else if (!(roundf(s) <= (float)T) || (i > 0 && !(starts[i - 1] <= s))) atomicOr(err, ERRBIT_OOB_ID);
}
// of a pack without rows, which has no other work
__global__ void __launch_bounds__(256) k_check_offsets(const float* __restrict__ starts, int n, int* err) {
  for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) check_offset(starts, i, 0, err);
}
// A row's segment.
__device__ __forceinline__ void find_segment(const PrepareDev& p, const float* starts, int t) {
  for (int i = t; i <= p.n_seg; i += p.tiles * 128) check_offset(starts, i, p.T, p.err);
  if (t >= p.T) return;
  const int2 r = segment_at(p, starts, t);
  p.begin[t] = r.x; p.end[t] = r.y;
}
// rows [x, y) are those with a segment
__device__ __forceinline__ int2 live_rows(const PrepareDev& p, const float* starts) {
  const float first = roundf(starts[0]), behind = roundf(starts[p.n_seg]);
  return make_int2(first > 0.0f ? (int)fminf(first, (float)p.T) : 0, behind < (float)p.T ? (int)fmaxf(behind, 0.0f) : p.T);
}

// What the other kernels want to know of a tile, in the order in which they take the tiles: (tile, smallest and largest begin of its rows' segments) for
// tiles of queries (which = 0), (tile, smallest and largest end) for tiles of keys (1); a row of no segment counts as (T, 0).  The order is by the
// work that the rows have ahead of them, the most first: a sort by count into 1024 classes, four a thread.  (Tiles of a class come in any
// order: it decides when a tile is worked on, not how.)
constexpr int kClasses = 1024;
__device__ void plan_tiles(const PrepareDev& p, const float* starts, int which, int* classes, int* warp_sums) {
  int4* plan = p.plan + which * p.tiles;
  *reinterpret_cast<int4*>(classes + threadIdx.x * 4) = make_int4(0, 0, 0, 0);
  const int2 live = live_rows(p, starts);
  auto look = [&](int tile) -> int4 {      // and its class
    const int first = max(tile * 128, live.x), last = min(tile * 128 + 127, live.y - 1);
    int2 a = make_int2(p.T, 0), b = a;
    if (first <= last) { a = segment_at(p, starts, first); b = segment_at(p, starts, last); }
    const bool dead = first > tile * 128 || last < tile * 128 + 127;
    int4 r;
    int n;
    if (which == 0) { r = make_int4(tile, min(a.x, b.x), dead ? p.T : max(a.x, b.x), 0); n = r.y < p.T ? tile - r.y / 128 : 0; }
    else { r = make_int4(tile, dead ? 0 : min(a.y, b.y), max(a.y, b.y), 0); n = r.z > 0 ? (r.z - 1) / 128 - tile : 0; }
    r.w = kClasses - 1 - max(0, min(n, kClasses - 1));
    return r;
  };
  __syncthreads();
  int4 mine = make_int4(0, 0, 0, 0);       // (a thread's first tile is looked at once)
  for (int i = threadIdx.x; i < p.tiles; i += 256) {
    const int4 r = look(i);
    if (i == (int)threadIdx.x) mine = r;
    atomicAdd(&classes[r.w], 1);
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;      // counts into places
  const int4 n = *reinterpret_cast<int4*>(classes + threadIdx.x * 4);
  int before = n.x + n.y + n.z + n.w;
  const int all = before;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += x; }
  if (lane == 31) warp_sums[wid] = before;
  __syncthreads();
  before -= all;
  for (int i = 0; i < wid; ++i) before += warp_sums[i];
  *reinterpret_cast<int4*>(classes + threadIdx.x * 4) = make_int4(before, before + n.x, before + n.x + n.y, before + n.x + n.y + n.z);
  __syncthreads();
  for (int i = threadIdx.x; i < p.tiles; i += 256) {
    const int4 r = i == (int)threadIdx.x ? mine : look(i);
    plan[atomicAdd(&classes[r.w], 1)] = r;
  }
}

// A CTA turns 128 rows of a head into planes.  The first head's CTAs find their rows' segments as well, and one or two CTAs more plan the
// order of the tiles.  All that a CTA wants of global memory, but the two ends of the offsets, is asked for before the first of it is used, and the offsets are searched
// in shared memory where they fit: with few tiles the kernel is as long as its longest chain of waits (1531 tokens, 6 + 2 heads of 80, for the
// gradient: 23.6 us with the offsets searched and delta formed a load at a time, 12.6 so).  HBM-bound with many: 8192 rows of 36 heads of 64 in
// 25 us, 6 TB/s read and written.
template <int DP, bool GRAD>
__global__ void __launch_bounds__(256, DP == 64 ? 4 : 2) k_prepare(PrepareDev p) {
  constexpr int kLanes = DP / 4, kRows = 256 / kLanes, kPasses = 128 / kRows;      // lanes of a row, rows of a pass
  __shared__ float red[8], of_row[128], offsets[1024];      // of_row: delta (do), lengths (v)
  __shared__ int text_top[128], first_row[128];             // (v) first_row: of the tile's rows, the first of the row's text; -1: no text
  __shared__ uint32_t bad[4];
  __shared__ __align__(16) int classes[kClasses];
  const int tile = blockIdx.x;
  const bool plans = tile == p.tiles;
  if (plans && blockIdx.y > (GRAD ? 1 : 0)) return;
  int h = blockIdx.y, which = 0;
  while (h >= p.in[which].heads) h -= p.in[which++].heads;
  const PlanesDev& x = p.in[which];
  const int c = (threadIdx.x % kLanes) * 4, r0 = threadIdx.x / kLanes;
  float4 v[kPasses];
  const bool mine = c < p.dk;
  const i64 t0 = (i64)tile * 128 + r0;
  // Rows before the first segment and behind the last may hold anything: they are not read, and as zeros do not reach the tile's exponent.
  const int2 live = live_rows(p, p.starts);
  const float* src = x.x + t0 * x.st + h * x.sh + c;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    v[i] = make_float4(0, 0, 0, 0);
    if (mine && t0 + i * kRows >= live.x && t0 + i * kRows < live.y) {
      const float* s = src + i * kRows * x.st;
      if (x.vec) v[i] = __ldcs(reinterpret_cast<const float4*>(s));
      else { v[i].x = s[0]; if (c + 1 < p.dk) v[i].y = s[1]; if (c + 2 < p.dk) v[i].z = s[2]; if (c + 3 < p.dk) v[i].w = s[3]; }
    }
  }
  const bool with_delta = GRAD && which == 3;
  float lse = -INFINITY;
  if (with_delta && threadIdx.x < 128 && tile * 128 + (int)threadIdx.x < p.T) lse = p.lse[(i64)h * p.T + tile * 128 + threadIdx.x];
  if (threadIdx.x < 4) bad[threadIdx.x] = 0;
  const bool with_lengths = GRAD && which == 2;
  if (plans || blockIdx.y == 0 || with_lengths) {
    const float* starts = p.starts;
    if (p.n_seg < 1024) {
      for (int i = threadIdx.x; i <= p.n_seg; i += 256) offsets[i] = p.starts[i];
      starts = offsets;
    }
    __syncthreads();
    if (plans) { plan_tiles(p, starts, blockIdx.y, classes, (int*)red); return; }
    if (threadIdx.x < 128 && blockIdx.y == 0) find_segment(p, starts, tile * 128 + threadIdx.x);
    if (threadIdx.x < 128 && with_lengths) {
      const int t = tile * 128 + threadIdx.x, begin = t < p.T ? segment_at(p, starts, t).x : p.T;
      first_row[threadIdx.x] = begin <= t ? max(begin - tile * 128, 0) : -1;
      text_top[threadIdx.x] = 0;
    }
  } else __syncthreads();
  if (with_delta) {      // delta of the rows
    const float* o = p.o + t0 * p.o_st + h * p.o_sh + c;
    constexpr int kBatch = DP == 64 ? 4 : 8;
#pragma unroll
    for (int i0 = 0; i0 < kPasses; i0 += kBatch) {
      float4 y[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        y[i] = make_float4(0, 0, 0, 0);
        if (mine && t0 + (i0 + i) * kRows < p.T) {
          const float* s = o + (i0 + i) * kRows * p.o_st;
          if (p.o_vec) y[i] = *reinterpret_cast<const float4*>(s);
          else { y[i].x = s[0]; if (c + 1 < p.dk) y[i].y = s[1]; if (c + 2 < p.dk) y[i].z = s[2]; if (c + 3 < p.dk) y[i].w = s[3]; }
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float4 g = v[i0 + i];
        float d = g.x * y[i].x;
        d = fmaf(g.y, y[i].y, d); d = fmaf(g.z, y[i].z, d); d = fmaf(g.w, y[i].w, d);
#pragma unroll
        for (int k = kLanes / 2; k > 0; k >>= 1) d += __shfl_xor_sync(0xffffffffu, d, k);
        if (c == 0) of_row[(i0 + i) * kRows + r0] = d;
      }
    }
  }
  float m = 0.0f;
  bool fine = true;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const float a = fmaxf(fabsf(v[i].x), fabsf(v[i].y)), b = fmaxf(fabsf(v[i].z), fabsf(v[i].w));
    const float sum = (v[i].x + v[i].y) * 0.0f + (v[i].z + v[i].w) * 0.0f;      // 0, or NaN where a component is not finite (or a sum overflows: looked at below)
    fine = fine && sum == 0.0f;
    m = fmaxf(m, fmaxf(a, b));
  }
  if (!fine) {
    m = 0.0f;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const float4 y = v[i];
      v[i] = make_float4(is_finite(y.x) ? y.x : 0.0f, is_finite(y.y) ? y.y : 0.0f, is_finite(y.z) ? y.z : 0.0f, is_finite(y.w) ? y.w : 0.0f);
      if (!(is_finite(y.x) && is_finite(y.y) && is_finite(y.z) && is_finite(y.w))) { const int r = i * kRows + r0; atomicOr(&bad[r >> 5], 1u << (r & 31)); }
      m = fmaxf(m, fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w))));
    }
  }
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[wid] = m;
  __syncthreads();
  if (with_delta && threadIdx.x < 128) {      // and 14 minus their lse in base 2 (a row of no segment: -infinity, so that every p is 0)
    const float d = of_row[threadIdx.x];
    const bool dead = lse == -INFINITY;
    // A row of do with a component that is not finite, which the planes hold as 0: every gradient that the row enters sees it through p.  (One
    // infinity leaves delta infinite and not NaN.)
    if (!is_finite(d) || ((bad[threadIdx.x >> 5] >> (threadIdx.x & 31)) & 1)) lse = __int_as_float(0x7fffffff);
    const i64 at = ((i64)h * p.tiles + tile) * 128 + threadIdx.x;
    p.lift[at] = dead ? -INFINITY : 14.0f - lse * kL2e;
    p.delta[at] = dead ? 0.0f : d;
  }
  m = red[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, red[i]);
  float inv;
  const float s = block_scale(m, &inv);
  float top = 0.0f;
  const i64 plane = (i64)x.heads * p.T * DP;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const i64 t = t0 + i * kRows;
    const float4 y = make_float4(v[i].x * s, v[i].y * s, v[i].z * s, v[i].w * s);
    float ss = y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    top = fmaxf(top, ss);
    if (with_lengths && c == 0) of_row[i * kRows + r0] = sqrtf(ss) * inv;
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
  const int first = with_lengths && threadIdx.x < 128 ? first_row[threadIdx.x] : -1;
  if (first >= 0) atomicMax(&text_top[first], __float_as_int(of_row[threadIdx.x]));      // (lengths are not negative: ordered as integers)
  __syncthreads();
  if (with_lengths && threadIdx.x < 128 && tile * 128 + (int)threadIdx.x < p.T)
    p.text_len[(i64)h * p.T + tile * 128 + threadIdx.x] = first >= 0 ? __int_as_float(text_top[first]) : 0.0f;
  const i64 at = (i64)h * p.tiles + tile;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, red[i]);
    x.inv[at] = bad[0] | bad[1] | bad[2] | bad[3] ? -inv : inv;      // (the sign: look at the tile's row bits)
    x.len[at] = sqrtf(top) * inv;
  }
  if (threadIdx.x < 4) x.bad[at * 4 + threadIdx.x] = bad[threadIdx.x];
}

// ---- what the kernels share ---------------------------------------------------------------------------------------------------------
// A tile of ROWS rows in shared memory: hi plane, lo plane, each of DP / 64 chunks of ROWS x 128 bytes.
template <int ROWS, int DP> __host__ __device__ constexpr int plane_bytes() { return ROWS * DP * 2; }
template <int ROWS, int DP>
__device__ __forceinline__ void load_plane(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int row, int head, int pl) {
  mbar_arrive_expect_tx(bar, plane_bytes<ROWS, DP>());
#pragma unroll
  for (int c = 0; c < DP / 64; ++c) tma_load_4d(dst + c * ROWS * 128, map, bar, c * 64, row, head, pl);
}
template <int ROWS, int DP>
__device__ __forceinline__ void copy_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int row, int head) {
#pragma unroll
  for (int pl = 0; pl < 2; ++pl)
#pragma unroll
    for (int c = 0; c < DP / 64; ++c) tma_load_4d(dst + pl * plane_bytes<ROWS, DP>() + c * ROWS * 128, map, bar, c * 64, row, head, pl);
}
template <int ROWS, int DP>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int row, int head) {
  mbar_arrive_expect_tx(bar, 2 * plane_bytes<ROWS, DP>());
  copy_tile<ROWS, DP>(dst, map, bar, row, head);
}
// D[128, N] (+)= A[128, DP] B[N, DP]^T for one plane of each, K-major tiles in shared memory; or A in tensor memory (DP / 2 columns).
// The first 16 `steps` components alone: beyond the head size the planes are 0.
template <int N, int DP>
__device__ __forceinline__ void rows_by_rows(uint32_t leader, int steps, uint32_t d, uint32_t a, uint32_t b, uint32_t on) {
  const uint64_t da = desc16(a, 0), db = desc16(b, 0);
#pragma unroll
  for (int k = 0; k < DP / 16; ++k, on = 1)
    if (k < steps) mma_f16(leader, d, da + (((k >> 2) * 128 * 128 + (k & 3) * 32) >> 4), db + (((k >> 2) * N * 128 + (k & 3) * 32) >> 4), idesc16(128, N, 0, 0), on);
}
template <int N, int DP>
__device__ __forceinline__ void kept_by_rows(uint32_t leader, int steps, uint32_t d, uint32_t a, uint32_t b, uint32_t on) {
  const uint64_t db = desc16(b, 0);
#pragma unroll
  for (int k = 0; k < DP / 16; ++k, on = 1)
    if (k < steps) mma_f16_ta(leader, d, a + k * 8, db + (((k >> 2) * N * 128 + (k & 3) * 32) >> 4), idesc16(128, N, 0, 0), on);
}
// D[128, DP] (+)= A[128, K] B[K, DP], A in tensor memory (per quarter of the columns: K / 8 columns of hi, then of lo), B a plane of K rows
template <int K, int DP, bool LO>
__device__ __forceinline__ void kept_by_cols(uint32_t leader, uint32_t d, uint32_t a, uint32_t b, uint32_t on) {
  constexpr int kSteps = K / 16 / kGroups;       // of a quarter
  const uint64_t db = desc16(b, K * 128);
#pragma unroll
  for (int k = 0; k < K / 16; ++k, on = 1)
    mma_f16_ta(leader, d, a + (k / kSteps) * (K / kGroups) + (k % kSteps) * 8 + (LO ? kSteps * 8 : 0), db + k * 128, idesc16(128, DP, 0, 1), on);
}
// 16 columns of this thread's lane, from and to registers
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
template <int W>
__device__ __forceinline__ void load_cols(uint32_t taddr, float (&v)[W]) {
  static_assert(W == 16 || W == 32, "one load");
  if constexpr (W == 32) tmem_ld32(taddr, reinterpret_cast<uint32_t*>(v)); else tmem_ld16(taddr, reinterpret_cast<uint32_t*>(v));
  wait_for_cols<W>(reinterpret_cast<uint32_t*>(v));
}
// the quarter of a row's columns as the left operand of product_cols: W / 2 columns of hi, W / 2 of lo
template <int W>
__device__ __forceinline__ void split_operand(const float (&v)[W], uint32_t (&r)[W]) {
#pragma unroll
  for (int j = 0; j < W / 2; ++j) split2_finite(v[2 * j], v[2 * j + 1], &r[j], &r[W / 2 + j]);
}
template <int W>
__device__ __forceinline__ void store_operand(uint32_t taddr, const uint32_t (&r)[W]) {
  if constexpr (W == 32) tmem_st32(taddr, r); else tmem_st16(taddr, r);
}
// acc = acc * keep + part * f over this thread's quarter of an accumulator
template <int W>
__device__ __forceinline__ void add_part(uint32_t taddr, float (&acc)[W], float keep, float f) {
  float v[W];
  load_cols<W>(taddr, v);
  const float2 k2 = make_float2(keep, keep), f2 = make_float2(f, f);
#pragma unroll
  for (int j = 0; j < W; j += 2) {
    const float2 a = fma2(make_float2(v[j], v[j + 1]), f2, mul2(make_float2(acc[j], acc[j + 1]), k2));
    acc[j] = a.x; acc[j + 1] = a.y;
  }
}
template <int W>
__device__ __forceinline__ void add_part(uint32_t taddr, float (&acc)[W], float f) {
  float v[W];
  load_cols<W>(taddr, v);
  const float2 f2 = make_float2(f, f);
#pragma unroll
  for (int j = 0; j < W; j += 2) {
    const float2 a = fma2(make_float2(v[j], v[j + 1]), f2, make_float2(acc[j], acc[j + 1]));
    acc[j] = a.x; acc[j + 1] = a.y;
  }
}
// This warp's 32 rows x W components of the result, through its own part of a tile buffer that no product reads any more: a thread holds
// a row, but a store that takes 16 bytes of each of 32 rows costs an instruction's time for every one of them (4000 cycles a
// tile; so 600).  out: row 0 of the warp's rows, component 0 of the head; c0: the warp's first component; live: rows that exist.
template <int W>
__device__ __forceinline__ void store_rows(float4* stage, const float (&acc)[W], float f, float* out, i64 stride, int live, int c0, int dk, int lane) {
  constexpr int C = W / 4, R = 32 / C;            // 16-byte pieces of a row, rows of one store
  constexpr int kShift = W == 16 ? 1 : 0;
#pragma unroll
  for (int c = 0; c < C; ++c) stage[lane * C + (c ^ ((lane >> kShift) & (C - 1)))] = make_float4(acc[4 * c] * f, acc[4 * c + 1] * f, acc[4 * c + 2] * f, acc[4 * c + 3] * f);
  __syncwarp();
  const int c = lane % C, at = c0 + 4 * c;
#pragma unroll
  for (int i = 0; i < 32 / R; ++i) {
    const int r = i * R + lane / C;
    const float4 v = stage[r * C + (c ^ ((r >> kShift) & (C - 1)))];
    if (r >= live || at >= dk) continue;
    float* o = out + r * stride + at;
    if ((dk & 3) == 0) *reinterpret_cast<float4*>(o) = v;
    else { o[0] = v.x; if (at + 1 < dk) o[1] = v.y; if (at + 2 < dk) o[2] = v.z; if (at + 3 < dk) o[3] = v.w; }
  }
}
// p 2^14 of a quarter of a row: 2^(score - lse + 14), one lse a row or one a column
template <int W>
__device__ __forceinline__ void weights_of_row(float (&v)[W], float sc, float off) {
  const float2 s2 = make_float2(sc, sc), o2 = make_float2(off, off);
#pragma unroll
  for (int i = 0; i < W; i += 2) {
    const float2 x = fma2(make_float2(v[i], v[i + 1]), s2, o2);
    v[i] = exp2_fast(x.x); v[i + 1] = exp2_fast(x.y);
  }
}
// the same as the left operand of product_cols (W / 2 registers of hi, W / 2 of lo), and their sum
template <int W>
__device__ __forceinline__ float split_weights(const float (&v)[W], float sc, float off, uint32_t (&r)[W]) {
  const float2 s2 = make_float2(sc, sc), o2 = make_float2(off, off);
  float2 a = make_float2(0.0f, 0.0f), b = a;
#pragma unroll
  for (int i = 0; i < W; i += 4) {
    float2 x = fma2(make_float2(v[i], v[i + 1]), s2, o2), y = fma2(make_float2(v[i + 2], v[i + 3]), s2, o2);
    x.x = exp2_fast(x.x); x.y = exp2_fast(x.y); y.x = exp2_fast(y.x); y.y = exp2_fast(y.y);
    a = add2(a, x); b = add2(b, y);
    split2_finite(x.x, x.y, &r[i / 2], &r[W / 2 + i / 2]);
    split2_finite(y.x, y.y, &r[i / 2 + 1], &r[W / 2 + i / 2 + 1]);
  }
  a = add2(a, b);
  return a.x + a.y;
}
template <int W>
__device__ __forceinline__ void weights_of_cols(float (&v)[W], float sc, const float* lift) {
  const float2 s2 = make_float2(sc, sc);
#pragma unroll
  for (int i = 0; i < W; i += 4) {
    const float4 l = *reinterpret_cast<const float4*>(lift + i);
    const float2 a = fma2(make_float2(v[i], v[i + 1]), s2, lo2(l)), b = fma2(make_float2(v[i + 2], v[i + 3]), s2, hi2(l));
    v[i] = exp2_fast(a.x); v[i + 1] = exp2_fast(a.y); v[i + 2] = exp2_fast(b.x); v[i + 3] = exp2_fast(b.y);
  }
}
template <int W>
__device__ __forceinline__ void keep_columns(float (&v)[W], int first, int last, float other) {
#pragma unroll
  for (int i = 0; i < W; ++i) if (i < first || i > last) v[i] = other;
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}
// a row warp has written its operand (and read the last accumulator)
__device__ __forceinline__ void operand_written(uint64_t* bar, int lane) {
  tmem_wait_st();
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}
// where a row warp's thread stands in a tile
struct Seat {
  int lane, quarter, group, row;
  uint32_t lane_off;
  __device__ __forceinline__ Seat() {
    const int warp = threadIdx.x >> 5;
    lane = threadIdx.x & 31; quarter = warp & 3; group = (warp - 2) >> 2; row = quarter * 32 + lane; lane_off = (uint32_t)(quarter * 32) << 16;
  }
};

struct Side { const __half* planes; const float* inv; const float* len; const uint32_t* bad; };
struct AttnParams {
  int T, tiles, hq, hk, dk;
  int steps;                                  // of 16 components in a head
  float scale;
  const int* begin; const int* end;
  const int4* plan;                           // [2][tiles] (plan_tiles)
  Side q, k, v, g;
  const float* lift; const float* delta;      // [hq][tiles * 128]: 14 - lse in base 2 (a weight comes with a factor of 2^14), delta
  const float* text_len;                      // (PrepareDev)
  float* out; float* lse;                     // forward
  float *dq, *dk_, *dv;                       // backward; with parts > 1 dk_ and dv are [parts][T, hk, dk], summed afterwards
  int parts;                                  // a key head's group of query heads is dealt to this many CTAs
  int* err;
};

// ---- forward ----------------------------------------------------------------------------------------------------------------------
// What the row warps want of a tile besides its matrices, put into shared memory with it: a few of its factors, and for tiles whose columns
// are queries their lift and delta (read from global memory where they are used they cost two trips to L2 a tile, 1900 of 5700 cycles).
template <int N, int VECTORS> struct Notes { float4 f; float v[VECTORS][N]; };
__device__ __forceinline__ void copy_note(float* dst, const float* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void expect_more(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// The resident tile (Q, or K in the dV kernel) and a ring of planes, streamed in the order in which the products take them: half a tile
// at a time, so that 128-wide heads too have a product's worth of planes in flight.
template <int DP> struct StreamSmem {
  static constexpr int kPlane = plane_bytes<128, DP>(), kSlots = DP == 64 ? 10 : 5;
  // (dV) Tile j's notes lie in slot j % kNotes.  Its planes are the stream's numbers 4 j - 2 and 4 j - 1, those of do 4 j + 4 and 4 j + 5, and the
// last are released when P of tile j has been formed: the slot is filled again only after that, as the plane which comes with it has waited.
  static constexpr int kNotes = DP == 64 ? 4 : 3, kNoteBytes = kNotes * (int)sizeof(Notes<128, 1>);
  static_assert(4 * kNotes - 2 - kSlots >= 4, "a note is overwritten while it is read");
  static constexpr int kBars = 1 + 2 * kSlots + 2 + 1 + 1 + kNotes;
  static constexpr int kTotal = 1024 + kPlane * (2 + kSlots) + kNoteBytes + kBars * 8 + 64;
};
// One CTA an SM, sixteen row warps.  Scores have two buffers, so the next tile's are formed while the row warps are at this one's; a
// weight is split into its halves where its exponential comes out, so that the special-function and the arithmetic pipes work at
// the same time, and before the wait for the last product, which still reads the last P.
template <int DP> struct FwdCfg {
  static constexpr int kPlane = plane_bytes<128, DP>(), kSlots = DP == 64 ? 10 : 5, kBars = 1 + 2 * kSlots + 2 + 1 + 1;
  static constexpr int kBuffers = DP == 64 ? 2 : 1, kExchange = kBuffers * kGroups * 128 * 4;      // row maxima, and accumulators: one buffer where there is no room for two
  static constexpr int kNeed = kPlane * (2 + kSlots) + kExchange + kBars * 8 + 64;
  static constexpr int kTotal = kNeed + 1024 < 232448 ? kNeed + 1024 : 232448;               // (227 KB: with wide heads 840 of the 1024 bytes for alignment are left)
};
template <int DP>
__global__ void __launch_bounds__(kThreads, 1)
k_forward(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnParams p) {
  using L = FwdCfg<DP>;
  constexpr int NS = L::kSlots, G = kGroups, W = DP / G, H = 128 / G, NB = L::kBuffers;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t shift = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  uint8_t* smem = smem_raw + shift;
  if (shift + L::kNeed > L::kTotal) {      // (an aligned base, as every launch has had, always fits)
    if (threadIdx.x == 0) atomicOr(p.err, ERRBIT_BOUNDS);
    return;
  }
  uint8_t *sq = smem, *ring = smem + 2 * L::kPlane;
  uint64_t* bars = (uint64_t*)(ring + NS * L::kPlane);
  uint64_t *b_x = bars, *b_full = bars + 1, *b_free = b_full + NS, *b_s = b_free + NS, *b_p = b_s + 2, *b_o = b_p + 1;
  int* ints = (int*)(b_o + 1);
  uint32_t* tmem_slot = (uint32_t*)ints + 2;
  volatile int* abort_flag = ints + 3;
  float* xchg = (float*)(ints + 4);                           // [NB tiles][groups][128]

  const int warp = threadIdx.x >> 5;
  const int h = blockIdx.x % p.hq, hk = h / (p.hq / p.hk);
  if (warp == 0) { prefetch_map(&map_q); prefetch_map(&map_k); prefetch_map(&map_v); }
  if (warp == 0) {
    for (int i = threadIdx.x; i < L::kBars; i += 32) mbar_init(&bars[i], &bars[i] == b_p ? kRowWarps : 1);
    if (threadIdx.x == 0) *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();      // (the copies below come before the other warps have seen the barriers)
    __syncwarp();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  wait_for_last_kernel();
  const int4 tile = p.plan[blockIdx.x / p.hq];
  const int qt = tile.x, b_min = tile.y, b_max = tile.z;
  const int kb0 = b_min < p.T ? b_min / 128 : qt + 1, n = qt + 1 - kb0;      // key tiles (none: no row of the tile has a segment)
  // the producer's place in the ring, and its first copies, under way while the rest of the CTA sets up
  uint32_t in_slot = 0, in_phase = 1;      // (the first round waits on the phase before the first: free)
  auto fetch = [&](const CUtensorMap* map, int j) -> bool {      // lo, then hi: the order in which the products take them
    for (int pl = 1; pl >= 0; --pl) {
      if (!mbar_wait(&b_free[in_slot], in_phase, abort_flag)) return false;
      load_plane<128, DP>(ring + in_slot * L::kPlane, map, &b_full[in_slot], (kb0 + j) * 128, hk, pl);
      if (++in_slot == NS) { in_slot = 0; in_phase ^= 1; }
    }
    return true;
  };
  bool fetched = true;
  if (threadIdx.x == 0 && n > 0) {
    load_tile<128, DP>(sq, &map_q, b_x, qt * 128, h);
    fetched = fetch(&map_k, 0) && (n < 2 || fetch(&map_k, 1));
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_s = tmem, t_p = tmem + 256, t_o = tmem + 384, o_step = (NB - 1) * DP;      // (from one accumulator to the next)

  if (warp == 0) {
    if (threadIdx.x == 0 && n > 0) {
      bool ok = fetched;
      for (int j = 0; j < n && ok; ++j) ok = fetch(&map_v, j) && (j + 2 >= n || fetch(&map_k, j + 2));
      if (*abort_flag) let_land(bars, 1 + NS);
    }
  } else if (warp == 1) {
    if (n > 0) {
      const uint32_t leader = elect_leader();
      uint32_t slot = 0, phase = 0;
      bool ok = warp_wait(b_x, 0, abort_flag);
      auto next = [&]() -> bool { const bool r = warp_wait(&b_full[slot], phase, abort_flag); tc_fence_after(); return r; };
      auto release = [&]() { commit_by(leader, &b_free[slot]); if (++slot == NS) { slot = 0; phase ^= 1; } };
      const uint32_t x_hi = smem_u32(sq), x_lo = x_hi + L::kPlane, r0 = smem_u32(ring);
      auto scores = [&](int j) -> bool {
        const uint32_t d = t_s + (j & 1) * 128;
        if (!next()) return false;
        rows_by_rows<128, DP>(leader, p.steps, d, x_hi, r0 + slot * L::kPlane, 0);
        release();
        if (!next()) return false;
        rows_by_rows<128, DP>(leader, p.steps, d, x_lo, r0 + slot * L::kPlane, 1);
        rows_by_rows<128, DP>(leader, p.steps, d, x_hi, r0 + slot * L::kPlane, 1);
        release();
        commit_by(leader, &b_s[j & 1]);
        return true;
      };
      if (ok) ok = scores(0);
      if (ok && n > 1) ok = scores(1);
      for (int j = 0; j < n && ok; ++j) {
        ok = warp_wait(b_p, j & 1, abort_flag) && next();
        if (!ok) break;
        kept_by_cols<128, DP, false>(leader, t_o + (j & 1) * o_step, t_p, r0 + slot * L::kPlane, 0);
        release();
        ok = next();
        if (!ok) break;
        kept_by_cols<128, DP, true>(leader, t_o + (j & 1) * o_step, t_p, r0 + slot * L::kPlane, 1);
        kept_by_cols<128, DP, false>(leader, t_o + (j & 1) * o_step, t_p, r0 + slot * L::kPlane, 1);
        release();
        commit_by(leader, b_o);
        if (j + 2 < n) ok = scores(j + 2);      // (this tile's scores have been read: P says so)
      }
    }
  } else {
    const Seat at;
    const int t = qt * 128 + at.row;
    const int begin = t < p.T ? p.begin[t] : p.T;
    const i64 kvt = (i64)hk * p.tiles;
    const float q_inv = p.q.inv[(i64)h * p.tiles + qt], sc0 = p.scale * kL2e * fabsf(q_inv);
    float acc[W], m = -INFINITY, l = 0.0f, keep = 0.0f, v_last = 0.0f;
    float k_inv = n > 0 ? p.k.inv[kvt + kb0] : 0.0f, v_inv = n > 0 ? p.v.inv[kvt + kb0] : 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] = 0.0f;
    bool ok = true;                             // (a wait that ran out does not end the loop: the other quarters of the rows meet this one in it)
    for (int j = 0; j < n; ++j) {
      const int kb = kb0 + j, c0 = kb * 128 + at.group * H;
      const float sc = fmaxf(sc0 * fabsf(k_inv), 1e-37f);      // (masked scores are -infinity times this)
      const bool bad = k_inv < 0.0f || v_inv < 0.0f;
      const bool crossed = kb == qt || kb * 128 < b_max;       // by the diagonal or the begin of a segment
      const float v_this = fabsf(v_inv);
      if (j + 1 < n) { k_inv = p.k.inv[kvt + kb + 1]; v_inv = p.v.inv[kvt + kb + 1]; }
      ok = mbar_wait(&b_s[j & 1], (j >> 1) & 1, abort_flag) && ok;
      tc_fence_after();
      float v[H];
      load_cols<H>(t_s + (j & 1) * 128 + at.group * H + at.lane_off, v);
      if (crossed) keep_columns<H>(v, begin - c0, t - c0, -INFINITY);
      if (bad) {                                // a visible key or value that is not finite
        const uint32_t bits = p.k.bad[(kvt + kb) * 4 + at.group] | p.v.bad[(kvt + kb) * 4 + at.group];
        for (int i = 0; i < H; ++i) if (((bits >> i) & 1) && c0 + i >= begin && c0 + i <= t) l = __int_as_float(0x7fffffff);
      }
      float m0 = fmaxf(v[0], v[1]), m1 = fmaxf(v[2], v[3]);
#pragma unroll
      for (int i = 4; i < H; i += 4) { m0 = fmaxf(m0, fmaxf(v[i], v[i + 1])); m1 = fmaxf(m1, fmaxf(v[i + 2], v[i + 3])); }
      float* x = xchg + (j & (NB - 1)) * G * 128 + at.row;
      if (NB == 1) asm volatile("bar.sync %0, 128;" ::"r"(1 + at.quarter) : "memory");
      x[at.group * 128] = fmaxf(m0, m1);
      asm volatile("bar.sync %0, 128;" ::"r"(1 + at.quarter) : "memory");      // the four quarters of these rows
      const float mn = fmaxf(m, fmaxf(fmaxf(x[0], x[128]), fmaxf(x[256], x[384])) * sc), ref = mn > -INFINITY ? mn : 0.0f;
      const float shrink = m > -INFINITY ? exp2_fast(m - ref) : 0.0f;
      uint32_t r[H];
      l = l * shrink + split_weights<H>(v, sc, 14.0f - ref, r);
      m = mn;
      if (j > 0) {                              // the last tile's product has read P and is in its accumulator
        ok = mbar_wait(b_o, (j - 1) & 1, abort_flag) && ok;
        tc_fence_after();
      }
      tmem_st32(t_p + at.group * H + at.lane_off, r);
      if (j > 0 && NB == 1) add_part<W>(t_o + at.group * W + at.lane_off, acc, keep, v_last);
      operand_written(b_p, at.lane);
      if (j > 0 && NB == 2) add_part<W>(t_o + ((j - 1) & 1) * o_step + at.group * W + at.lane_off, acc, keep, v_last);
      keep = shrink; v_last = v_this;
    }
    // the row's sum, while the last product is formed
    float* x = xchg + (n & (NB - 1)) * G * 128 + at.row;
    if (NB == 1) asm volatile("bar.sync %0, 128;" ::"r"(1 + at.quarter) : "memory");
    x[at.group * 128] = l;
    asm volatile("bar.sync %0, 128;" ::"r"(1 + at.quarter) : "memory");
    l = (x[0] + x[128]) + (x[256] + x[384]);
    if (q_inv < 0.0f && begin <= t && ((p.q.bad[((i64)h * p.tiles + qt) * 4 + at.quarter] >> at.lane) & 1)) l = __int_as_float(0x7fffffff);
    const bool dead = l == 0.0f;
    if (n > 0) {
      ok = mbar_wait(b_o, (n - 1) & 1, abort_flag) && ok;
      tc_fence_after();
      add_part<W>(t_o + ((n - 1) & 1) * o_step + at.group * W + at.lane_off, acc, keep, v_last);
    }
    const int row0 = qt * 128 + at.quarter * 32;
    if (ok) {
      store_rows<W>((float4*)sq + (at.quarter * G + at.group) * 8 * W, acc, dead ? 0.0f : 1.0f / l, p.out + ((i64)row0 * p.hq + h) * p.dk, (i64)p.hq * p.dk, p.T - row0,
                    at.group * W, p.dk, at.lane);
      if (t < p.T && at.group == 0 && p.lse) p.lse[(i64)h * p.T + t] = dead ? -INFINITY : (m - 14.0f) * kLn2 + logf(l);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_free(tmem, 512); }
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.err, ERRBIT_WAIT_TIMEOUT);
}

// ---- backward ---------------------------------------------------------------------------------------------------------------------
// One launch for the three gradients: CTAs that make dK come first (three products for every query head of the group), then dV (two),
// then dQ, so that the long ones start first and the short ones fill the gaps.
struct BwdMaps { CUtensorMap q, k, g, qn, kn, vn, gn; };      // boxes of 128 rows, and of N rows (GradSmem)

// dV of 128 keys: every query head of the CTA's part of the group x every tile of 128 queries from the keys' own to the last one that
// sees them.
template <int DP>
__device__ __forceinline__ void grad_v(uint8_t* smem, const BwdMaps& maps, const AttnParams& p, int block) {
  using L = StreamSmem<DP>;
  constexpr int NS = L::kSlots, W = DP / kGroups, H = 128 / kGroups;
  uint8_t *sk = smem, *ring = smem + 2 * L::kPlane;
  Notes<128, 1>* notes = (Notes<128, 1>*)(ring + NS * L::kPlane);
  uint64_t* bars = (uint64_t*)((uint8_t*)notes + L::kNoteBytes);
  uint64_t *b_x = bars, *b_full = bars + 1, *b_note = b_full + NS, *b_free = b_note + L::kNotes, *b_s = b_free + NS, *b_p = b_s + 2, *b_o = b_p + 1;
  int* ints = (int*)(b_o + 1);
  uint32_t* tmem_slot = (uint32_t*)ints + 2;
  volatile int* abort_flag = ints + 3;

  const int warp = threadIdx.x >> 5;
  const int part = block % p.parts, hk = block / p.parts % p.hk, heads = p.hq / p.hk / p.parts, h0 = (hk * p.parts + part) * heads;
  if (warp == 0) {
    for (int i = threadIdx.x; i < L::kBars; i += 32) mbar_init(&bars[i], &bars[i] == b_p ? kRowWarps : 1);
    if (threadIdx.x == 0) *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();      // (the copies below come before the other warps have seen the barriers)
    __syncwarp();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  wait_for_last_kernel();
  const int4 planned = p.plan[p.tiles + block / p.parts / p.hk];
  const int kt = planned.x, e_min = planned.y, e_max = planned.z;
  const int per = e_max > 0 ? (e_max - 1) / 128 - kt + 1 : 0, n = per * heads;
  // the producer's place in the ring and in the stream, and its first copies, under way while the rest of the CTA sets up
  uint32_t in_slot = 0, in_phase = 1;      // (the first round waits on the phase before the first: free)
  struct Place { int i, head, note; } q_at{0, h0, 0}, g_at{0, h0, 0};
  auto fetch = [&](const CUtensorMap* map, Place& at) -> bool {      // lo, then hi: the order in which the products take them
    for (int pl = 1; pl >= 0; --pl) {
      if (!mbar_wait(&b_free[in_slot], in_phase, abort_flag)) return false;
      load_plane<128, DP>(ring + in_slot * L::kPlane, map, &b_full[in_slot], (kt + at.i) * 128, at.head, pl);
      if (++in_slot == NS) { in_slot = 0; in_phase ^= 1; }
    }
    return true;
  };
  auto on = [&](Place& at) { if (++at.i == per) { at.i = 0; ++at.head; } };
  auto note_q = [&]() {                    // (its slot is free: the planes have waited for later products than the slot's last)
    const i64 tile = (i64)q_at.head * p.tiles + kt + q_at.i;
    Notes<128, 1>& to = notes[q_at.note];
    uint64_t* bar = &b_note[q_at.note];
    expect_more(bar, 512);
    copy_note(to.v[0], p.lift + tile * 128, 512, bar);
    to.f = make_float4(p.scale * kL2e * fabsf(p.k.inv[(i64)hk * p.tiles + kt]) * fabsf(p.q.inv[tile]), fabsf(p.g.inv[tile]), 0.0f, 0.0f);
    mbar_arrive(bar);
    if (++q_at.note == L::kNotes) q_at.note = 0;
    on(q_at);
  };
  auto fetch_q = [&]() -> bool { if (!fetch(&maps.q, q_at)) return false; note_q(); return true; };
  auto fetch_g = [&]() -> bool { const bool r = fetch(&maps.g, g_at); on(g_at); return r; };
  bool fetched = true;
  if (threadIdx.x == 0 && n > 0) {
    load_tile<128, DP>(sk, &maps.k, b_x, kt * 128, hk);
    fetched = fetch(&maps.q, q_at);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_s = tmem, t_p = tmem + 256, t_o = tmem + 384;

  if (warp == 0) {
    if (threadIdx.x == 0 && n > 0) {
      note_q();
      bool ok = fetched && (n < 2 || fetch_q());
      for (int j = 0; j < n && ok; ++j) ok = fetch_g() && (j + 2 >= n || fetch_q());
      if (*abort_flag) let_land(bars, 1 + NS + L::kNotes);
    }
  } else if (warp == 1) {
    if (n > 0) {
      const uint32_t leader = elect_leader();
      uint32_t slot = 0, phase = 0;
      bool ok = warp_wait(b_x, 0, abort_flag);
      auto next = [&]() -> bool { const bool r = warp_wait(&b_full[slot], phase, abort_flag); tc_fence_after(); return r; };
      auto release = [&]() { commit_by(leader, &b_free[slot]); if (++slot == NS) { slot = 0; phase ^= 1; } };
      const uint32_t x_hi = smem_u32(sk), x_lo = x_hi + L::kPlane, r0 = smem_u32(ring);
      auto scores = [&](int j) -> bool {
        const uint32_t d = t_s + (j & 1) * 128;
        if (!next()) return false;
        rows_by_rows<128, DP>(leader, p.steps, d, x_hi, r0 + slot * L::kPlane, 0);
        release();
        if (!next()) return false;
        rows_by_rows<128, DP>(leader, p.steps, d, x_lo, r0 + slot * L::kPlane, 1);
        rows_by_rows<128, DP>(leader, p.steps, d, x_hi, r0 + slot * L::kPlane, 1);
        release();
        commit_by(leader, &b_s[j & 1]);
        return true;
      };
      if (ok) ok = scores(0);
      if (ok && n > 1) ok = scores(1);
      for (int j = 0; j < n && ok; ++j) {
        ok = warp_wait(b_p, j & 1, abort_flag) && next();
        if (!ok) break;
        kept_by_cols<128, DP, false>(leader, t_o, t_p, r0 + slot * L::kPlane, 0);
        release();
        ok = next();
        if (!ok) break;
        kept_by_cols<128, DP, true>(leader, t_o, t_p, r0 + slot * L::kPlane, 1);
        kept_by_cols<128, DP, false>(leader, t_o, t_p, r0 + slot * L::kPlane, 1);
        release();
        commit_by(leader, b_o);
        if (j + 2 < n) ok = scores(j + 2);      // (this tile's scores have been read: P says so)
      }
    }
  } else {
    const Seat at;
    const int t = kt * 128 + at.row;
    const int end = t < p.T ? p.end[t] : 0;
    float acc[W], f_last = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] = 0.0f;
    bool ok = true;
    int qt = kt, note = 0;
    uint32_t note_phase = 0;
    for (int j = 0; j < n; ++j) {
      const int c0 = qt * 128 + at.group * H;
      if (!mbar_wait(&b_note[note], note_phase, abort_flag)) { ok = false; break; }
      const float4 f = notes[note].f;
      const float f_this = f.y;
      if (!mbar_wait(&b_s[j & 1], (j >> 1) & 1, abort_flag)) { ok = false; break; }
      tc_fence_after();
      uint32_t r[H];
      {
        float v[H];
        load_cols<H>(t_s + (j & 1) * 128 + at.group * H + at.lane_off, v);
        weights_of_cols<H>(v, f.x, notes[note].v[0] + at.group * H);
        if (qt == kt || qt * 128 + 128 > e_min) keep_columns<H>(v, t - c0, end - 1 - c0, 0.0f);
        split_operand<H>(v, r);
      }
      if (++note == L::kNotes) { note = 0; note_phase ^= 1; }
      if (++qt == kt + per) qt = kt;
      if (j > 0) {
        if (!mbar_wait(b_o, (j - 1) & 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
      }
      store_operand<H>(t_p + at.group * H + at.lane_off, r);
      if (j > 0) add_part<W>(t_o + at.group * W + at.lane_off, acc, f_last);
      operand_written(b_p, at.lane);
      f_last = f_this;
    }
    if (ok && n > 0) {
      ok = mbar_wait(b_o, (n - 1) & 1, abort_flag);
      if (ok) {
        tc_fence_after();
        add_part<W>(t_o + at.group * W + at.lane_off, acc, f_last);
      }
    }
    const int row0 = kt * 128 + at.quarter * 32;
    if (ok)
      store_rows<W>((float4*)sk + (at.quarter * kGroups + at.group) * 8 * W, acc, 1.0f / 16384.0f, p.dv + (((i64)part * p.T + row0) * p.hk + hk) * p.dk,
                    (i64)p.hk * p.dk, p.T - row0, at.group * W, p.dk, at.lane);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_free(tmem, 512); }
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.err, ERRBIT_WAIT_TIMEOUT);
}

// dQ and dK.  X (128 rows, resident: q and do, or k and v), Y streamed in tiles of N rows (k and v, or q and do):
//   S = X1 Y1^T, dP = X2 Y2^T, dS = p (dP - delta), result += dS Y1.
// dS goes where S was; S has two buffers, so the next tile's S and dP are formed while dS Y1 runs.  Y1 is held from S to the last
// product, so it has three buffers; X2 is kept in tensor memory, as the left operand of dP, to leave room for them.
// 2^e with 2 |do| |v| 2^e below 2^14, over the weights' 2^14, and 2^-e
struct DsScale { float to, back; };
__device__ __forceinline__ DsScale ds_scale(float len, float vmax) {
  const float b = 2.0f * len * vmax;
  int e = b > 0.0f ? 13 - ((int)(__float_as_uint(b) >> 23) - 127) : 0;
  e = e > 100 ? 100 : (e < -100 ? -100 : e);
  return DsScale{__uint_as_float((uint32_t)(127 + e) << 23) * (1.0f / 16384.0f), __uint_as_float((uint32_t)(127 - e) << 23)};
}
template <int DP> struct GradSmem {
  static constexpr int N = DP == 64 ? 128 : 64;                       // 128-wide heads: 64 rows of Y at a time
  static constexpr int kTileX = 2 * plane_bytes<128, DP>(), kTileY = 2 * plane_bytes<N, DP>();
  static constexpr int kY1 = 3, kY2 = 2;
  static constexpr int kBars = 2 + 2 * kY1 + 2 * kY2 + 2 + 1 + 1 + 1;
  static constexpr int kNoteBytes = kY1 * (int)sizeof(Notes<N, 2>);     // (with the tile of Y1)
  static constexpr int kTotal = 1024 + kTileX + (kY1 + kY2) * kTileY + kNoteBytes + kBars * 8 + 64;
  static_assert(kTotal <= 227 * 1024, "shared memory");
};
template <int DP, bool DK>
__device__ __forceinline__ void grad_qk(uint8_t* smem, const BwdMaps& maps, const AttnParams& p, int block) {
  using L = GradSmem<DP>;
  constexpr int N = L::N, H = N / kGroups, W = DP / kGroups, N1 = L::kY1, N2 = L::kY2, R = 128 / N;
  uint8_t *x1 = smem, *y1 = x1 + L::kTileX, *y2 = y1 + N1 * L::kTileY;
  Notes<N, 2>* notes = (Notes<N, 2>*)(y2 + N2 * L::kTileY);
  uint64_t* bars = (uint64_t*)((uint8_t*)notes + L::kNoteBytes);
  uint64_t *b_x = bars, *b_y1full = bars + 1, *b_y2full = b_y1full + N1, *b_y1free = b_y2full + N2, *b_y2free = b_y1free + N1, *b_s = b_y2free + N2, *b_dp = b_s + 2,
           *b_ds = b_dp + 1, *b_o = b_ds + 1, *b_x2 = b_o + 1;
  int* ints = (int*)(b_x2 + 1);
  uint32_t* tmem_slot = (uint32_t*)ints + 2;
  volatile int* abort_flag = ints + 3;

  const int warp = threadIdx.x >> 5;
  const int part = DK ? block % p.parts : 0, rest = DK ? block / p.parts : block, x_heads = DK ? p.hk : p.hq;
  const int hx = rest % x_heads, hk = DK ? hx : hx / (p.hq / p.hk), heads = DK ? p.hq / p.hk / p.parts : 1, h0 = DK ? (hk * p.parts + part) * heads : hx;
  if (warp == 0) {
    for (int i = threadIdx.x; i < L::kBars; i += 32) mbar_init(&bars[i], &bars[i] == b_x2 || &bars[i] == b_ds ? kRowWarps : 1);
    if (threadIdx.x == 0) *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();      // (the copies below come before the other warps have seen the barriers)
    __syncwarp();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  wait_for_last_kernel();
  const int4 planned = p.plan[(DK ? p.tiles : 0) + rest / x_heads];
  const int xt = planned.x, e_min = planned.y, e_max = planned.z;      // (DK: of the ends, else of the begins)
  // tiles of Y, in steps of N rows
  int y0, per;
  if (DK) { y0 = xt * R; per = e_max > 0 ? (e_max - 1) / N - y0 + 1 : 0; }
  else { const int last = xt * 128 + 127 < p.T ? xt * 128 + 127 : p.T - 1; y0 = e_min / N; per = e_min < p.T ? last / N - y0 + 1 : 0; }
  const int n = per * heads;
  const CUtensorMap *map_x1 = DK ? &maps.k : &maps.q, *map_y1 = DK ? &maps.qn : &maps.kn, *map_y2 = DK ? &maps.gn : &maps.vn;
  const i64 x_at = (i64)hx * p.tiles + xt;
  // The producer: copies of tile (hy, i) into slots s1 and s2, then what goes with it.  The first two tiles are under way while the rest of
  // the CTA sets up.
  struct Place { int hy, i; } tile_in{DK ? h0 : hk, 0}, note_in = tile_in;
  auto on = [&](Place& at) { if (++at.i == per) { at.i = 0; ++at.hy; } };
  int s1 = 0, s2 = 0, note_s1 = 0;
  auto copy_y1 = [&]() {                   // (the note's arrival completes the barrier's count)
    const int y = (y0 + tile_in.i) * N;
    expect_more(&b_y1full[s1], L::kTileY + (DK ? 2 * N * 4 : 0));
    copy_tile<N, DP>(y1 + s1 * L::kTileY, map_y1, &b_y1full[s1], y, tile_in.hy);
    if (DK) {
      const i64 r = (i64)tile_in.hy * p.tiles * 128 + y;
      copy_note(notes[s1].v[0], p.lift + r, N * 4, &b_y1full[s1]);
      copy_note(notes[s1].v[1], p.delta + r, N * 4, &b_y1full[s1]);
    }
    if (++s1 == N1) s1 = 0;
  };
  auto copy_y2 = [&]() {
    load_tile<N, DP>(y2 + s2 * L::kTileY, map_y2, &b_y2full[s2], (y0 + tile_in.i) * N, tile_in.hy);
    if (++s2 == N2) s2 = 0;
    on(tile_in);
  };
  auto write_note = [&]() {                // factors of S, of dP; of what dS is scaled by; of the product
    const i64 y_at = (i64)note_in.hy * p.tiles + (y0 + note_in.i) * N / 128;
    const float s_x = p.scale * kL2e * fabsf(DK ? p.k.inv[x_at] : p.q.inv[x_at]), fx2 = fabsf(DK ? p.v.inv[x_at] : p.g.inv[x_at]);
    const float a = fabsf(DK ? p.q.inv[y_at] : p.k.inv[y_at]), b = fabsf(DK ? p.g.inv[y_at] : p.v.inv[y_at]);
    notes[note_s1].f = make_float4(s_x * a, b * fx2, DK ? p.g.len[y_at] : 0.0f, a);
    mbar_arrive(&b_y1full[note_s1]);
    if (++note_s1 == N1) note_s1 = 0;
    on(note_in);
  };
  const Seat at;
  uint4 x2[DP / 16];                       // row warps: half a row of X2, hi from groups 0 and 1, lo from 2 and 3
  // The scale of a row of dS has to hold |do| |v| twice, delta being an average of do . v: the longest value row that the row's text has (DK), or has
  // up to the row's tile (dQ).  Texts differ in size, so no other's values count: its own rows of the tiles where it begins and ends, and the
  // whole tiles between them.
  float vmax = 0.0f;
  int begin = p.T, end = 0;                // of the row's text
  if (threadIdx.x == 0 && n > 0) {
    load_tile<128, DP>(x1, map_x1, b_x, xt * 128, hx);
    copy_y1(); copy_y2();
    if (n > 1) { copy_y1(); copy_y2(); }
  } else if (warp >= 2) {
    const Side& side = DK ? p.v : p.g;
    const int t = xt * 128 + at.row;
    const uint4* src = reinterpret_cast<const uint4*>(side.planes + ((i64)(at.group >> 1) * x_heads * p.T + (i64)hx * p.T + t) * DP) + (at.group & 1) * (DP / 16);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) x2[i] = t < p.T ? src[i] : make_uint4(0, 0, 0, 0);
    const float *own = p.text_len + (i64)hk * p.T, *whole = p.v.len + (i64)hk * p.tiles;
    if (t < p.T) { begin = p.begin[t]; end = p.end[t]; vmax = own[t]; }
    // the text that reaches back out of the tile, if any of the warp's rows is in it, and the one that reaches ahead
    const int b = (int)__reduce_min_sync(0xffffffffu, (unsigned)begin), e = (int)__reduce_max_sync(0xffffffffu, (unsigned)end);
    float back = 0.0f, ahead = 0.0f;
    if (b < xt * 128) {
      if (at.lane == 0) back = own[b];
      for (int i = b / 128 + 1 + at.lane; i < xt; i += 32) back = fmaxf(back, whole[i]);
    }
    if (DK && e > xt * 128 + 128) {
      if (at.lane == 0) ahead = own[e - 1];
      for (int i = xt + 1 + at.lane; i < (e - 1) / 128; i += 32) ahead = fmaxf(ahead, whole[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { back = fmaxf(back, __shfl_xor_sync(0xffffffffu, back, o)); ahead = fmaxf(ahead, __shfl_xor_sync(0xffffffffu, ahead, o)); }
    if (begin < xt * 128) vmax = fmaxf(vmax, back);
    if (end > xt * 128 + 128) vmax = fmaxf(vmax, ahead);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_s = tmem, t_dp = tmem + 2 * N, t_x2 = tmem + 3 * N, t_o = t_x2 + DP;      // (DP columns of X2: hi, lo)

  if (warp == 0) {
    if (threadIdx.x == 0 && n > 0) {
      write_note();
      if (n > 1) write_note();
      uint32_t phase1 = 1, phase2 = 0;     // (the third slot of Y1 is free, the first of Y2 when its product has been formed)
      for (int j = 2; j < n; ++j) {
        if (!mbar_wait(&b_y1free[s1], phase1, abort_flag)) break;
        copy_y1();
        if (s1 == 0) phase1 ^= 1;
        write_note();
        if (!mbar_wait(&b_y2free[s2], phase2, abort_flag)) break;
        copy_y2();
        if (s2 == 0) phase2 ^= 1;
      }
      if (*abort_flag) let_land(bars, 1 + N1 + N2);
    }
  } else if (warp == 1) {
    if (n > 0) {
      const uint32_t leader = elect_leader();
      constexpr int kPX = plane_bytes<128, DP>(), kPY = plane_bytes<N, DP>();
      bool ok = warp_wait(b_x, 0, abort_flag);
      uint32_t y1_in = 0, y1_phase = 0, y1_out = 0;
      auto scores = [&](int j) -> bool {      // (buffer j & 1 held dS of tile j - 2, which its product has read)
        if (!warp_wait(&b_y1full[y1_in], y1_phase, abort_flag)) return false;
        if (j >= 2 && !warp_wait(b_o, j & 1, abort_flag)) return false;
        tc_fence_after();
        const uint32_t d = t_s + (j & 1) * N, x = smem_u32(x1), y = smem_u32(y1 + y1_in * L::kTileY);
        if (++y1_in == N1) { y1_in = 0; y1_phase ^= 1; }
        rows_by_rows<N, DP>(leader, p.steps, d, x + kPX, y, 0);
        rows_by_rows<N, DP>(leader, p.steps, d, x, y + kPY, 1);
        rows_by_rows<N, DP>(leader, p.steps, d, x, y, 1);
        commit_by(leader, &b_s[j & 1]);
        return true;
      };
      auto other = [&](int j) -> bool {
        if (!warp_wait(&b_y2full[j % N2], (j / N2) & 1, abort_flag)) return false;
        tc_fence_after();
        const uint32_t y = smem_u32(y2 + (j % N2) * L::kTileY);
        kept_by_rows<N, DP>(leader, p.steps, t_dp, t_x2 + DP / 2, y, 0);
        kept_by_rows<N, DP>(leader, p.steps, t_dp, t_x2, y + kPY, 1);
        kept_by_rows<N, DP>(leader, p.steps, t_dp, t_x2, y, 1);
        commit_by(leader, &b_y2free[j % N2]);
        commit_by(leader, b_dp);
        return true;
      };
      if (ok) ok = scores(0) && warp_wait(b_x2, 0, abort_flag) && other(0);
      if (ok && n > 1) ok = scores(1);
      for (int j = 0; j < n && ok; ++j) {
        ok = warp_wait(b_ds, j & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (j + 1 < n) ok = other(j + 1);
        if (!ok) break;
        const uint32_t ds = t_s + (j & 1) * N, y = smem_u32(y1 + y1_out * L::kTileY);
        kept_by_cols<N, DP, true>(leader, t_o, ds, y, 0);
        kept_by_cols<N, DP, false>(leader, t_o, ds, y + kPY, 1);
        kept_by_cols<N, DP, false>(leader, t_o, ds, y, 1);
        commit_by(leader, &b_y1free[y1_out]);
        if (++y1_out == N1) y1_out = 0;
        commit_by(leader, b_o);
        if (j + 2 < n) ok = scores(j + 2);
      }
    }
  } else {
    const int t = xt * 128 + at.row;
    // The columns that the row sees, without itself where it is the first of its segment: such a query sees one key, whose weight is 1 whatever the
    // score, so its dS is 0, where do . v - delta would be the difference of two roundings of one sum.  (NaN stays NaN.)
    int from = p.T, to = 0;
    bool lone = false;
    if (t < p.T) {
      lone = begin == t;
      if (DK) { from = lone ? t + 1 : t; to = end - 1; }
      else { from = begin; to = t; }
    }
    if constexpr (DP == 64) tmem_st16(t_x2 + at.group * 16 + at.lane_off, reinterpret_cast<const uint32_t*>(x2));
    else tmem_st32(t_x2 + at.group * 32 + at.lane_off, reinterpret_cast<const uint32_t*>(x2));
    operand_written(b_x2, at.lane);
    // (addresses of this thread's quarters as sums of their own: taken apart at every use, one build read S of groups 1 to 3 fifteen columns off)
    const uint32_t my_s = t_s + at.group * H + at.lane_off, my_dp = my_s + 2 * N, my_o = t_o + at.group * W + at.lane_off;
    DsScale ds{};
    if (!DK) ds = ds_scale(p.g.len[x_at], vmax);
    float lift_row = 0.0f, delta_row = 0.0f;
    if (!DK) { const i64 r = ((i64)hx * p.tiles + xt) * 128 + at.row; lift_row = p.lift[r]; delta_row = p.delta[r]; if (lone && lift_row == lift_row) to = t - 1; }
    float acc[W], f_last = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] = 0.0f;
    bool ok = true;
    int y = y0 * N, slot = 0;
    uint32_t phase = 0;
    for (int j = 0; j < n; ++j) {
      const int c0 = y + at.group * H;
      const bool crossed = DK ? y < xt * 128 + 128 || y + N > e_min : y + N > xt * 128 || y < e_max;
      // (the slot is filled again only after the product of this tile, which waits for this tile's dS)
      if (!mbar_wait(&b_y1full[slot], phase, abort_flag)) { ok = false; break; }
      const Notes<N, 2>& note = notes[slot];
      const float4 f = note.f;
      if (DK) ds = ds_scale(f.z, vmax);
      if (!mbar_wait(&b_s[j & 1], (j >> 1) & 1, abort_flag)) { ok = false; break; }
      tc_fence_after();
      float v[H];
      load_cols<H>(my_s + (j & 1) * N, v);
      if (DK) weights_of_cols<H>(v, f.x, note.v[0] + at.group * H);
      else weights_of_row<H>(v, f.x, lift_row);
      if (!mbar_wait(b_dp, j & 1, abort_flag)) { ok = false; break; }
      tc_fence_after();
      {
        float d[H];
        load_cols<H>(my_dp, d);
        const float f_dp = f.y * ds.to;
        const float2 f1 = make_float2(f_dp, f_dp), f2 = make_float2(-ds.to, -ds.to);
        float2 da = mul2(make_float2(delta_row, delta_row), f2), db = da;
#pragma unroll
        for (int i = 0; i < H; i += 4) {
          if (DK) { const float4 e = *reinterpret_cast<const float4*>(note.v[1] + at.group * H + i); da = mul2(lo2(e), f2); db = mul2(hi2(e), f2); }
          const float2 a = mul2(make_float2(v[i], v[i + 1]), fma2(make_float2(d[i], d[i + 1]), f1, da));
          const float2 b = mul2(make_float2(v[i + 2], v[i + 3]), fma2(make_float2(d[i + 2], d[i + 3]), f1, db));
          v[i] = a.x; v[i + 1] = a.y; v[i + 2] = b.x; v[i + 3] = b.y;
        }
      }
      if (crossed) {
        int lo = from - c0;
        if (DK && lone && t >= c0 && t < c0 + H && note.v[0][at.group * H + t - c0] != note.v[0][at.group * H + t - c0]) --lo;
        keep_columns<H>(v, lo, to - c0, 0.0f);
      }
      uint32_t r[H];
      split_operand<H>(v, r);
      // (a quarter's dS lies within its own quarter of S)
      store_operand<H>(my_s + (j & 1) * N, r);
      if (j > 0) {
        if (!mbar_wait(b_o, (j - 1) & 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        add_part<W>(my_o, acc, f_last);
      }
      operand_written(b_ds, at.lane);
      f_last = f.w * ds.back;
      if (++slot == N1) { slot = 0; phase ^= 1; }
      y += N;
      if (DK && y == (y0 + per) * N) y = y0 * N;
    }
    if (ok && n > 0) {
      ok = mbar_wait(b_o, (n - 1) & 1, abort_flag);
      if (ok) {
        tc_fence_after();
        add_part<W>(my_o, acc, f_last);
      }
    }
    const int row0 = xt * 128 + at.quarter * 32;
    if (ok)
      store_rows<W>((float4*)x1 + (at.quarter * kGroups + at.group) * 8 * W, acc, p.scale,
                    DK ? p.dk_ + (((i64)part * p.T + row0) * p.hk + hk) * p.dk : p.dq + ((i64)row0 * p.hq + hx) * p.dk, (i64)x_heads * p.dk, p.T - row0, at.group * W,
                    p.dk, at.lane);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_free(tmem, 512); }
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.err, ERRBIT_WAIT_TIMEOUT);
}
template <int DP>
__global__ void __launch_bounds__(kThreads, 1) k_backward(const __grid_constant__ BwdMaps maps, const __grid_constant__ AttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int keys = p.tiles * p.hk * p.parts, b = blockIdx.x;
  if (b < keys) grad_qk<DP, true>(smem, maps, p, b);
  else if (b < 2 * keys) grad_v<DP>(smem, maps, p, b - keys);
  else grad_qk<DP, false>(smem, maps, p, b - 2 * keys);
}
__device__ __forceinline__ float plus(float a, float b) { return a + b; }
__device__ __forceinline__ float4 plus(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
// the parts of dK and dV added in order
template <class V>
__global__ void __launch_bounds__(256) k_add_parts(const V* __restrict__ a, const V* __restrict__ b, V* __restrict__ oa, V* __restrict__ ob, i64 n, int parts) {
  wait_for_last_kernel();
  for (i64 i = (i64)blockIdx.x * 256 + threadIdx.x; i < 2 * n; i += (i64)gridDim.x * 256) {
    const V* src = i < n ? a + i : b + (i - n);
    V s = src[0];
    for (int k = 1; k < parts; ++k) s = plus(s, src[(i64)k * n]);
    if (i < n) oa[i] = s; else ob[i - n] = s;
  }
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
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
  const size_t begin = take((size_t)s.T * 4), end = take((size_t)s.T * 4), plan = take((size_t)tiles * 2 * sizeof(int4));
  const size_t delta = o ? take((size_t)s.hq * tiles * 512) : 0, lift = o ? take((size_t)s.hq * tiles * 512) : 0, text_len = o ? take((size_t)s.hk * s.T * 4) : 0;
  VB_TRY(scratch_alloc(at, &w.hold.p));
  uint8_t* base = (uint8_t*)w.hold.p;
  PrepareDev& d = w.prep;
  d.n = n; d.T = (int)s.T; d.tiles = tiles; d.dk = s.dk; d.hq = s.hq;
  Side* sides[4] = {&w.p.q, &w.p.k, &w.p.v, &w.p.g};
  int all = 0;
  for (int i = 0; i < n; ++i) {
    d.in[i] = PlanesDev{in[i].p, in[i].st, in[i].sh, (__half*)(base + planes[i]), (float*)(base + inv[i]), (float*)(base + len[i]), (uint32_t*)(base + bad[i]), heads[i],
                        s.dk % 4 == 0 && in[i].st % 4 == 0 && in[i].sh % 4 == 0 && (reinterpret_cast<uintptr_t>(in[i].p) & 15) == 0};
    *sides[i] = Side{d.in[i].planes, d.in[i].inv, d.in[i].len, d.in[i].bad};
    all += heads[i];
  }
  d.starts = starts; d.n_seg = (int)n_seg; d.begin = (int*)(base + begin); d.end = (int*)(base + end); d.plan = (int4*)(base + plan); d.err = ctx().d_err;
  if (o) { d.o = o->p; d.o_st = o->st; d.o_sh = o->sh; d.lse = lse;
           d.o_vec = s.dk % 4 == 0 && o->st % 4 == 0 && o->sh % 4 == 0 && (reinterpret_cast<uintptr_t>(o->p) & 15) == 0; d.delta = (float*)(base + delta); d.lift = (float*)(base + lift);
           d.text_len = (float*)(base + text_len); }
  AttnParams& p = w.p;
  p.T = (int)s.T; p.tiles = tiles; p.hq = s.hq; p.hk = s.hk; p.dk = s.dk; p.steps = (s.dk + 15) / 16; p.scale = s.scale;
  p.begin = d.begin; p.end = d.end; p.plan = d.plan; p.lift = d.lift; p.delta = d.delta; p.text_len = d.text_len; p.err = ctx().d_err;
  ProfScope prof("segment_attn_prepare", 8.0 * (double)s.T * all * s.dk);
  const dim3 grid(tiles + 1, all);
  if (dp == 64) { if (o) k_prepare<64, true><<<grid, 256, 0, ctx().stream>>>(d); else k_prepare<64, false><<<grid, 256, 0, ctx().stream>>>(d); }
  else if (o) k_prepare<128, true><<<grid, 256, 0, ctx().stream>>>(d);
  else k_prepare<128, false><<<grid, 256, 0, ctx().stream>>>(d);
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
  static const int ready = allow_smem(k_forward<DP>, FwdCfg<DP>::kTotal);
  VB_TRY(ready);
  CUtensorMap mq, mk, mv;
  VB_TRY(make_map(&mq, w.prep.in[0], w.p.T, DP, 128)); VB_TRY(make_map(&mk, w.prep.in[1], w.p.T, DP, 128)); VB_TRY(make_map(&mv, w.prep.in[2], w.p.T, DP, 128));
  return launch_early(k_forward<DP>, dim3((unsigned)w.p.hq * w.p.tiles), dim3(kThreads), FwdCfg<DP>::kTotal, mq, mk, mv, w.p);
}
template <int DP>
int backward(Work& w, float* dq, float* dk, float* dv) {
  constexpr int N = GradSmem<DP>::N, kSmem = GradSmem<DP>::kTotal > StreamSmem<DP>::kTotal ? GradSmem<DP>::kTotal : StreamSmem<DP>::kTotal;
  static const int ready = allow_smem(k_backward<DP>, kSmem);
  VB_TRY(ready);
  BwdMaps m;
  const PlanesDev* in = w.prep.in;
  AttnParams& p = w.p;
  VB_TRY(make_map(&m.q, in[0], p.T, DP, 128)); VB_TRY(make_map(&m.k, in[1], p.T, DP, 128)); VB_TRY(make_map(&m.g, in[3], p.T, DP, 128));
  VB_TRY(make_map(&m.qn, in[0], p.T, DP, N)); VB_TRY(make_map(&m.kn, in[1], p.T, DP, N)); VB_TRY(make_map(&m.vn, in[2], p.T, DP, N)); VB_TRY(make_map(&m.gn, in[3], p.T, DP, N));
  // A CTA that walks the query heads of a whole group is the longest of the launch, and dealing the group to several costs their parts' sums and
  // more CTAs.  So it is dealt out until a CTA's heads are no more than an SM's share of the launch: 3 tiles' worth for every query head.
  // Gradient, group in one CTA / dealt to as many as make four for every SM / by this rule: 4096 tokens in 9 texts, 16 + 4 heads of 64 131 / 176 / 131 us;
  // 1531 in 3, 6 + 2 of 80 113 / 63 / 63; 1024 in one, 16 + 2 of 64 122 / 53 / 45; 8192 in 4, 16 + 4 of 128 884 / 1000 / 889.  It counts tiles and not the
  // lengths of texts, which the host does not know; by the rule / in two parts: 4096 in one text, 8 + 2 of 64 234 / 186; 600 in two, 4 + 1 of 96 37 / 33.
  const int group = p.hq / p.hk;
  p.parts = 1;
  for (int d = 2; d <= group && (i64)group * ctx().sm_count > 3 * (i64)p.tiles * p.hq * p.parts; ++d) if (group % d == 0) p.parts = d;
  const i64 n = (i64)p.T * p.hk * p.dk;
  Temp hold;
  p.dq = dq; p.dk_ = dk; p.dv = dv;
  if (p.parts > 1) {
    VB_TRY(scratch_alloc((size_t)(2 * p.parts * n) * sizeof(float), &hold.p));
    p.dk_ = (float*)hold.p; p.dv = p.dk_ + p.parts * n;
  }
  VB_TRY(launch_early(k_backward<DP>, dim3((unsigned)(p.tiles * (2 * p.hk * p.parts + p.hq))), dim3(kThreads), kSmem, m, p));
  if (p.parts > 1) {
    const i64 cap = (i64)ctx().sm_count * 8;
    const bool vec = n % 4 == 0 && ((reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv)) & 15) == 0;
    const i64 m = vec ? n / 4 : n, ctas = (2 * m + 255) / 256;
    const dim3 grid((unsigned)(ctas < cap ? ctas : cap));
    if (vec) return launch_early(k_add_parts<float4>, grid, dim3(256), 0, (const float4*)p.dk_, (const float4*)p.dv, (float4*)dk, (float4*)dv, m, p.parts);
    return launch_early(k_add_parts<float>, grid, dim3(256), 0, (const float*)p.dk_, (const float*)p.dv, dk, dv, m, p.parts);
  }
  return VB_OK;
}

}  // namespace

int launch_check_offsets(const float* starts, i64 n) {
  const i64 ctas = (n + 256) / 256, cap = ctx().sm_count;
  k_check_offsets<<<(unsigned)(ctas < cap ? ctas : cap), 256, 0, ctx().stream>>>(starts, (int)n + 1, ctx().d_err);
  VB_LAUNCH_CHECK();
  return VB_OK;
}
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
