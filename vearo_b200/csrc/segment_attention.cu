// Causal attention with grouped heads over packed segments, forward and backward.
//
//   row t of segment [b, e):  s_tj = scale q_t . k_j for b <= j <= t,  p = softmax(s),  o = sum p v,  lse = log sum exp s
//   backward: delta = do . o,  ds = p (do . v - delta),  dq = scale sum ds k,  dk = scale sum over the group ds q,  dv = sum p do
//
// One warp per row and head; a lane holds every 32nd component.
#include "segment_attention.h"

namespace vb {
namespace {

// Where the segment of each row begins and ends (rows of no segment: an empty range).  Offsets that decrease or leave [0, T] are
// reported; whatever they are, every range stays inside [0, T].
__global__ void __launch_bounds__(256) k_segments(const float* __restrict__ starts, int n, int T, int* __restrict__ begin, int* __restrict__ end, int* err) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  for (int i = t; i <= n; i += gridDim.x * 256) {
    const float s = starts[i];
    if (!(s > -0.5f)) atomicOr(err, ERRBIT_NEG_ID);
    else if (!(s < (float)T + 0.5f) || (i > 0 && !(starts[i - 1] <= s))) atomicOr(err, ERRBIT_OOB_ID);
  }
  if (t >= T) return;
  int lo = 0, hi = n + 1;          // offsets [0, lo) are <= t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (roundf(starts[mid]) <= (float)t) lo = mid + 1; else hi = mid;
  }
  int b = T, e = 0;
  if (lo > 0 && lo <= n) {
    const float fb = roundf(starts[lo - 1]), fe = roundf(starts[lo]);
    b = fb > 0.0f ? (int)fb : 0;
    e = fe < (float)T ? (int)fe : T;
    if (!(b <= t && t < e)) { b = T; e = 0; }
  }
  begin[t] = b; end[t] = e;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ void load_head(const SegHeads& x, i64 t, int h, int dk, int lane, float (&r)[4]) {
  const float* p = x.p + t * x.st + h * x.sh;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = lane + 32 * i < dk ? p[lane + 32 * i] : 0.0f;
}
__device__ __forceinline__ float dot(const float (&a)[4], const float (&b)[4]) { return warp_sum(a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3]); }
__device__ __forceinline__ void store_head(float* p, int dk, int lane, const float (&r)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) if (lane + 32 * i < dk) p[lane + 32 * i] = r[i];
}

__global__ void __launch_bounds__(128) k_attn_rows(SegShape s, SegHeads q, SegHeads k, SegHeads v, const int* __restrict__ begin, float* __restrict__ out, float* __restrict__ lse) {
  const int lane = threadIdx.x & 31, h = blockIdx.y, hk = h / (s.hq / s.hk);
  const i64 t = (i64)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (t >= s.T) return;
  float a[4], b[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.0f;
  load_head(q, t, h, s.dk, lane, a);
  for (i64 j = begin[t]; j <= t; ++j) {
    load_head(k, j, hk, s.dk, lane, b);
    const float x = dot(a, b) * s.scale, top = fmaxf(m, x);
    const float keep = expf(m - top), p = expf(x - top);
    load_head(v, j, hk, s.dk, lane, b);
    l = l * keep + p; m = top;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * keep + p * b[i];
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = begin[t] <= t ? o[i] * inv : 0.0f;
  store_head(out + (t * s.hq + h) * s.dk, s.dk, lane, o);
  if (lane == 0 && lse) lse[h * s.T + t] = begin[t] <= t ? m + logf(l) : -INFINITY;
}
__global__ void __launch_bounds__(128) k_attn_dq(SegShape s, SegHeads q, SegHeads k, SegHeads v, SegHeads o, SegHeads g, const int* __restrict__ begin,
                                                 const float* __restrict__ lse, float* __restrict__ delta, float* __restrict__ dq) {
  const int lane = threadIdx.x & 31, h = blockIdx.y, hk = h / (s.hq / s.hk);
  const i64 t = (i64)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (t >= s.T) return;
  float a[4], b[4], gg[4], oo[4], acc[4] = {0, 0, 0, 0};
  load_head(q, t, h, s.dk, lane, a); load_head(g, t, h, s.dk, lane, gg); load_head(o, t, h, s.dk, lane, oo);
  const float d = dot(gg, oo), L = lse[h * s.T + t];
  if (lane == 0) delta[h * s.T + t] = d;
  for (i64 j = begin[t]; j <= t; ++j) {
    load_head(k, j, hk, s.dk, lane, b);
    const float p = expf(dot(a, b) * s.scale - L);
    float vv[4];
    load_head(v, j, hk, s.dk, lane, vv);
    const float ds = p * (dot(gg, vv) - d) * s.scale;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += ds * b[i];
  }
  store_head(dq + (t * s.hq + h) * s.dk, s.dk, lane, acc);
}
__global__ void __launch_bounds__(128) k_attn_dkv(SegShape s, SegHeads q, SegHeads k, SegHeads v, SegHeads g, const int* __restrict__ end, const float* __restrict__ lse,
                                                  const float* __restrict__ delta, float* __restrict__ dk, float* __restrict__ dv) {
  const int lane = threadIdx.x & 31, hk = blockIdx.y, group = s.hq / s.hk;
  const i64 j = (i64)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (j >= s.T) return;
  float kk[4], vv[4], ak[4] = {0, 0, 0, 0}, av[4] = {0, 0, 0, 0};
  load_head(k, j, hk, s.dk, lane, kk); load_head(v, j, hk, s.dk, lane, vv);
  for (int h = hk * group; h < (hk + 1) * group; ++h)
    for (i64 t = j; t < end[j]; ++t) {
      float a[4], gg[4];
      load_head(q, t, h, s.dk, lane, a); load_head(g, t, h, s.dk, lane, gg);
      const float p = expf(dot(a, kk) * s.scale - lse[h * s.T + t]);
      const float ds = p * (dot(gg, vv) - delta[h * s.T + t]) * s.scale;
#pragma unroll
      for (int i = 0; i < 4; ++i) { ak[i] += ds * a[i]; av[i] += p * gg[i]; }
    }
  store_head(dk + (j * s.hk + hk) * s.dk, s.dk, lane, ak);
  store_head(dv + (j * s.hk + hk) * s.dk, s.dk, lane, av);
}

int segments(const SegShape& s, const float* starts, i64 n, Temp& hold, int** begin, int** end) {
  VB_TRY(scratch_alloc((size_t)s.T * 8, &hold.p));
  *begin = (int*)hold.p; *end = *begin + s.T;
  k_segments<<<(unsigned)((s.T + 255) / 256), 256, 0, ctx().stream>>>(starts, (int)n, (int)s.T, *begin, *end, ctx().d_err);
  VB_LAUNCH_CHECK();
  return VB_OK;
}

}  // namespace

int launch_segment_attention(const SegShape& s, const SegHeads& q, const SegHeads& k, const SegHeads& v, const float* starts, i64 n, float* out, float* lse) {
  Temp hs;
  int *begin, *end;
  VB_TRY(segments(s, starts, n, hs, &begin, &end));
  k_attn_rows<<<dim3((unsigned)((s.T + 3) / 4), s.hq), 128, 0, ctx().stream>>>(s, q, k, v, begin, out, lse);
  VB_LAUNCH_CHECK();
  return VB_OK;
}
int launch_segment_attention_backward(const SegShape& s, const SegHeads& q, const SegHeads& k, const SegHeads& v, const float* starts, i64 n,
                                      const SegHeads& out, const float* lse, const SegHeads& g, float* dq, float* dk, float* dv) {
  Temp hs, hd;
  int *begin, *end;
  VB_TRY(segments(s, starts, n, hs, &begin, &end));
  VB_TRY(scratch_alloc((size_t)s.T * s.hq * sizeof(float), &hd.p));
  k_attn_dq<<<dim3((unsigned)((s.T + 3) / 4), s.hq), 128, 0, ctx().stream>>>(s, q, k, v, out, g, begin, lse, (float*)hd.p, dq);
  VB_LAUNCH_CHECK();
  k_attn_dkv<<<dim3((unsigned)((s.T + 3) / 4), s.hk), 128, 0, ctx().stream>>>(s, q, k, v, g, end, lse, (const float*)hd.p, dk, dv);
  VB_LAUNCH_CHECK();
  return VB_OK;
}

}  // namespace vb
