// RMS norm of every query and key head with the rotary position turn in the same pass, forward and backward.
//
//   x-hat = x / sqrt(mean(x^2) + eps),  y = w * x-hat,  (y_a, y_b) -> (y_a c - y_b s, y_a s + y_b c)   for the pair j of a head,
//   c, s = cos, sin of position * theta^(-2j / rot): pairs are (j, j + rot/2), or (2j, 2j + 1) when interleaved; components from
//   rot on are not turned.
//   backward: g' = the turn undone on g;  dx = (w g' - x-hat mean(w g' x-hat)) / sqrt(mean(x^2) + eps);  dw = sum g' x-hat.
//
// HBM-bound: reads each head once and writes it once (backward: reads x and g, writes dx).  Eight lanes own a head, each lane
// "units" of eight components that hold both members of its pairs (two runs of four, rot/2 apart, or eight neighbours), so the
// turn needs no exchange and the norm three shuffles; loads and stores are 16 bytes.  A warp takes a token, or 4 HEADS heads of one,
// queries and keys in one row: it asks for all of them, forms the token's cosines and sines in shared memory while they are on their way,
// and meets no other warp (CTAs that shared the cosines of a few tokens stood at their barriers).  8192 tokens x 16 heads of 64: forward 14.1 us,
// 4.8 TB/s, with the barriers 16.5; backward 21.3 us, 4.7 TB/s, with the barriers 26, and 4.9 us for the sums of the weights' gradients.
// The angle is formed in turns: position times frequency / 2 pi in 64 bits (the
// frequencies are 64-bit host values in the kernel's parameters), the fraction of a quarter turn in 32, so far positions lose
// nothing.  Head sizes, rotated widths or addresses that do not fit the 16-byte units take a scalar kernel, one warp per head.
#include "common.h"
#include "qk_norm_rope.h"
#include "split16.cuh"

namespace vb {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kLanes = 8, kGroups = kThreads / kLanes;

// cosine and sine of `pos` turns-per-position `rev`, argument reduced to an eighth of a turn before it is rounded to 32 bits
__device__ __forceinline__ float2 turn_of(double pos, double rev) {
  const double q = pos * rev * 4.0;               // quarter turns
  const double n = rint(q);
  float s, c;
  sincospif(0.5f * (float)(q - n), &s, &c);
  const int k = (int)(n - 4.0 * floor(n * 0.25));  // (a position that is not finite leaves c and s NaN whatever k is)
  if (k & 1) { const float t = c; c = -s; s = t; }
  if (k & 2) { c = -c; s = -s; }
  return make_float2(c, s);
}

__device__ __forceinline__ float group_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  v += __shfl_xor_sync(0xffffffffu, v, 2);
  return v + __shfl_xor_sync(0xffffffffu, v, 4);
}

// offsets inside a head of the two runs of four components that make unit u; u counts the rotated units first
template <bool INTER>
__device__ __forceinline__ void unit_at(int u, int rot, int& a, int& b) {
  if (!INTER && 8 * u < rot) { a = 4 * u; b = rot / 2 + 4 * u; }
  else { a = 8 * u; b = 8 * u + 4; }
}
// the eight components of a unit turned (or turned back, sign = -1); cs: this token's cosines and sines
template <bool INTER>
__device__ __forceinline__ void turn_unit(float4& x, float4& y, const float2* cs, int u, float sign) {
  if (INTER) {        // pairs 4u .. 4u + 3: (x.x, x.y), (x.z, x.w), (y.x, y.y), (y.z, y.w)
    const float2 t0 = cs[4 * u], t1 = cs[4 * u + 1], t2 = cs[4 * u + 2], t3 = cs[4 * u + 3];
    const float4 p = x, q = y;
    x.x = p.x * t0.x - sign * p.y * t0.y; x.y = sign * p.x * t0.y + p.y * t0.x;
    x.z = p.z * t1.x - sign * p.w * t1.y; x.w = sign * p.z * t1.y + p.w * t1.x;
    y.x = q.x * t2.x - sign * q.y * t2.y; y.y = sign * q.x * t2.y + q.y * t2.x;
    y.z = q.z * t3.x - sign * q.w * t3.y; y.w = sign * q.z * t3.y + q.w * t3.x;
  } else {
    const float4 p = x, q = y;
    const float2 t0 = cs[4 * u], t1 = cs[4 * u + 1], t2 = cs[4 * u + 2], t3 = cs[4 * u + 3];
    x.x = p.x * t0.x - sign * q.x * t0.y; y.x = sign * p.x * t0.y + q.x * t0.x;
    x.y = p.y * t1.x - sign * q.y * t1.y; y.y = sign * p.y * t1.y + q.y * t1.x;
    x.z = p.z * t2.x - sign * q.z * t2.y; y.z = sign * p.z * t2.y + q.z * t2.x;
    x.w = p.w * t3.x - sign * q.w * t3.y; y.w = sign * p.w * t3.y + q.w * t3.x;
  }
}
__device__ __forceinline__ float dot4(float4 a, float4 b) { return a.x * b.x + a.y * b.y + a.z * b.z + a.w * b.w; }
__device__ __forceinline__ float4 mul4(float4 a, float4 b) { return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w); }
__device__ __forceinline__ float4 add4(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
__device__ __forceinline__ float4 scale4(float4 a, float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); }

// cosines and sines of a token, by one warp into its own strip
__device__ __forceinline__ void fill_turns(float2* cs, const RopeTable& tab, float pos, int half) {
  for (int j = threadIdx.x & 31; j < half; j += 32) cs[j] = turn_of((double)pos, tab.rev[j]);
}
// Head hh of token t where the queries' heads are counted first.
struct HeadAt { const float* x; int h; bool is_q; };
__device__ __forceinline__ HeadAt head_at(const HeadView& q, const HeadView& k, i64 t, int hh) {
  HeadAt a;
  a.is_q = hh < q.heads;
  a.h = a.is_q ? hh : hh - q.heads;
  a.x = a.is_q ? q.p + t * q.st + a.h * q.sh : k.p + t * k.st + a.h * k.sh;
  return a;
}

template <int UPL, bool INTER, int HEADS>
__global__ void __launch_bounds__(kThreads, 4) k_norm_rope(const __grid_constant__ RopeTable tab, HeadView q, HeadView k, const float* __restrict__ wq,
                                                        const float* __restrict__ wk, const float* __restrict__ pos, float* __restrict__ oq,
                                                        float* __restrict__ ok, i64 tokens, int dk, int rot, float eps) {
  extern __shared__ float2 turns[];
  const int lane = threadIdx.x & (kLanes - 1), wid = threadIdx.x >> 5, h0 = blockIdx.y * 4 * HEADS + ((threadIdx.x & 31) >> 3);
  const i64 t = (i64)blockIdx.x * kWarps + wid;
  if (t >= tokens) return;
  const int heads = q.heads + (k.p ? k.heads : 0), half = rot / 2;
  float4 a[HEADS][UPL], b[HEADS][UPL];
#pragma unroll
  for (int n = 0; n < HEADS; ++n) {
    const HeadAt at = head_at(q, k, t, h0 + 4 * n);
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      const int u = lane + i * kLanes;
      int oa, ob;
      unit_at<INTER>(u, rot, oa, ob);
      a[n][i] = b[n][i] = make_float4(0, 0, 0, 0);
      if (h0 + 4 * n < heads && 8 * u < dk) { a[n][i] = *reinterpret_cast<const float4*>(at.x + oa); b[n][i] = *reinterpret_cast<const float4*>(at.x + ob); }
    }
  }
  float2* cs = turns + wid * half;
  fill_turns(cs, tab, pos[t], half);
  __syncwarp();
  const float rdk = 1.0f / (float)dk;
#pragma unroll
  for (int n = 0; n < HEADS; ++n) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < UPL; ++i) ss += dot4(a[n][i], a[n][i]) + dot4(b[n][i], b[n][i]);
    const float inv = 1.0f / sqrtf(group_sum(ss) * rdk + eps);
    if (h0 + 4 * n >= heads) continue;
    const HeadAt at = head_at(q, k, t, h0 + 4 * n);
    const float* w = at.is_q ? wq : wk;
    float* o = (at.is_q ? oq + (t * q.heads + at.h) * (i64)dk : ok + (t * k.heads + at.h) * (i64)dk);
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      const int u = lane + i * kLanes;
      if (8 * u >= dk) continue;
      int oa, ob;
      unit_at<INTER>(u, rot, oa, ob);
      float4 ya = mul4(scale4(a[n][i], inv), *reinterpret_cast<const float4*>(w + oa)), yb = mul4(scale4(b[n][i], inv), *reinterpret_cast<const float4*>(w + ob));
      if (8 * u < rot) turn_unit<INTER>(ya, yb, cs, u, 1.0f);
      *reinterpret_cast<float4*>(o + oa) = ya;
      *reinterpret_cast<float4*>(o + ob) = yb;
    }
    __syncwarp(0xffu << (threadIdx.x & 24));
  }
}

// the CTA's sums for one weight: lanes of equal position in all groups, added in group order
template <int UPL, bool INTER>
__device__ __forceinline__ void store_weight_sums(const float4 (&acc)[2 * UPL], float* part, float* sm, int dk, int rot) {
  const int lane = threadIdx.x & (kLanes - 1), group = threadIdx.x / kLanes;
  for (int i = 0; i < UPL; ++i) {       // one unit per lane at a time: [group][8 lanes][8]
    __syncthreads();
    float4* s4 = reinterpret_cast<float4*>(sm) + (group * kLanes + lane) * 2;
#pragma unroll
    for (int j = 0; j < UPL; ++j) if (j == i) { s4[0] = acc[2 * j]; s4[1] = acc[2 * j + 1]; }
    __syncthreads();
    if (threadIdx.x < 64) {
      const int u = (int)threadIdx.x / 8 + i * kLanes, e = threadIdx.x & 7;
      if (8 * u < dk) {
        float s = 0.0f;
        for (int gr = 0; gr < kGroups; ++gr) s += sm[gr * 64 + threadIdx.x];
        int oa, ob;
        unit_at<INTER>(u, rot, oa, ob);
        part[e < 4 ? oa + e : ob + e - 4] = s;
      }
    }
  }
}
template <int UPL, bool INTER, int HEADS>
__global__ void __launch_bounds__(kThreads, UPL == 1 ? 3 : UPL == 2 ? 2 : 1) k_norm_rope_bwd(const __grid_constant__ RopeTable tab, HeadView q, HeadView k, HeadView gq, HeadView gk,
                                                            const float* __restrict__ wq, const float* __restrict__ wk, const float* __restrict__ pos,
                                                            float* __restrict__ dq, float* __restrict__ dkeys, float* __restrict__ part,
                                                            i64 tokens, int dk, int rot, float eps) {
  extern __shared__ float2 turns[];
  __shared__ __align__(16) float sums[kGroups * 64];
  const int lane = threadIdx.x & (kLanes - 1), wid = threadIdx.x >> 5, h0 = blockIdx.y * 4 * HEADS + ((threadIdx.x & 31) >> 3);
  const int heads = q.heads + (k.p ? k.heads : 0), half = rot / 2;
  float2* cs = turns + wid * half;
  const float rdk = 1.0f / (float)dk;
  float4 accq[2 * UPL], acck[2 * UPL];      // this lane's sums of g' x-hat over the heads it has seen
#pragma unroll
  for (int i = 0; i < 2 * UPL; ++i) accq[i] = acck[i] = make_float4(0, 0, 0, 0);
  for (i64 t = (i64)blockIdx.x * kWarps + wid; t < tokens; t += (i64)gridDim.x * kWarps) {
    float4 a[HEADS][UPL], b[HEADS][UPL], ga[HEADS][UPL], gb[HEADS][UPL];
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
      const float *px = head_at(q, k, t, h0 + 4 * n).x, *pg = head_at(gq, gk, t, h0 + 4 * n).x;
#pragma unroll
      for (int i = 0; i < UPL; ++i) {
        const int u = lane + i * kLanes;
        int oa, ob;
        unit_at<INTER>(u, rot, oa, ob);
        a[n][i] = b[n][i] = ga[n][i] = gb[n][i] = make_float4(0, 0, 0, 0);
        if (h0 + 4 * n < heads && 8 * u < dk) {
          a[n][i] = *reinterpret_cast<const float4*>(px + oa); b[n][i] = *reinterpret_cast<const float4*>(px + ob);
          ga[n][i] = *reinterpret_cast<const float4*>(pg + oa); gb[n][i] = *reinterpret_cast<const float4*>(pg + ob);
        }
      }
    }
    __syncwarp();      // (the last token's cosines have been read)
    fill_turns(cs, tab, pos[t], half);
    __syncwarp();
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
      const bool live = h0 + 4 * n < heads;      // (a head that is not there is all zeros: it adds nothing)
      const HeadAt at = head_at(q, k, t, live ? h0 + 4 * n : 0);
      const float* w = at.is_q ? wq : wk;
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < UPL; ++i) ss += dot4(a[n][i], a[n][i]) + dot4(b[n][i], b[n][i]);
      const float inv = 1.0f / sqrtf(group_sum(ss) * rdk + eps);
      float c = 0.0f;
#pragma unroll
      for (int i = 0; i < UPL; ++i) {
        const int u = lane + i * kLanes;
        if (8 * u >= dk) continue;
        float4 &xa = a[n][i], &xb = b[n][i], &ya = ga[n][i], &yb = gb[n][i];
        if (8 * u < rot) turn_unit<INTER>(ya, yb, cs, u, -1.0f);
        xa = scale4(xa, inv); xb = scale4(xb, inv);      // x-hat
        const float4 pa = mul4(ya, xa), pb = mul4(yb, xb);
        if (live) {
          if (at.is_q) { accq[2 * i] = add4(accq[2 * i], pa); accq[2 * i + 1] = add4(accq[2 * i + 1], pb); }
          else { acck[2 * i] = add4(acck[2 * i], pa); acck[2 * i + 1] = add4(acck[2 * i + 1], pb); }
        }
        int oa, ob;
        unit_at<INTER>(u, rot, oa, ob);
        ya = mul4(ya, *reinterpret_cast<const float4*>(w + oa)); yb = mul4(yb, *reinterpret_cast<const float4*>(w + ob));
        c += dot4(ya, xa) + dot4(yb, xb);
      }
      c = group_sum(c) * rdk;
      if (live) {
        float* o = at.is_q ? dq + (t * q.heads + at.h) * (i64)dk : dkeys + (t * k.heads + at.h) * (i64)dk;
#pragma unroll
        for (int i = 0; i < UPL; ++i) {
          const int u = lane + i * kLanes;
          if (8 * u >= dk) continue;
          int oa, ob;
          unit_at<INTER>(u, rot, oa, ob);
          *reinterpret_cast<float4*>(o + oa) = scale4(add4(ga[n][i], scale4(a[n][i], -c)), inv);
          *reinterpret_cast<float4*>(o + ob) = scale4(add4(gb[n][i], scale4(b[n][i], -c)), inv);
        }
      }
      __syncwarp();
    }
  }
  // partial sums: one row of [dk] (queries) and, where there are keys, one more behind it per CTA
  const int width = k.p ? 2 * dk : dk;
  part += ((i64)blockIdx.y * gridDim.x + blockIdx.x) * width;
  store_weight_sums<UPL, INTER>(accq, part, sums, dk, rot);
  if (k.p) store_weight_sums<UPL, INTER>(acck, part + dk, sums, dk, rot);
}

// ---- any head size, rotated width and alignment: one warp per head, components in 32-bit accesses -----------------------------
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ void pair_at(int j, int rot, bool inter, int& a, int& b) {
  a = inter ? 2 * j : j; b = inter ? 2 * j + 1 : j + rot / 2;
}
__global__ void __launch_bounds__(kThreads) k_norm_rope_any(const __grid_constant__ RopeTable tab, HeadView q, HeadView k, const float* __restrict__ wq,
                                                            const float* __restrict__ wk, const float* __restrict__ pos, float* __restrict__ oq,
                                                            float* __restrict__ ok, i64 tokens, int dk, int rot, bool inter, float eps) {
  const int lane = threadIdx.x & 31, per = q.heads + (k.p ? k.heads : 0);
  const i64 rows = tokens * per, step = (i64)gridDim.x * (kThreads / 32);
  for (i64 r = (i64)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); r < rows; r += step) {
    const i64 t = r / per;
    const int hh = (int)(r - t * per);
    const bool is_q = hh < q.heads;
    const HeadView& v = is_q ? q : k;
    const int h = is_q ? hh : hh - q.heads;
    const float* x = v.p + t * v.st + h * v.sh;
    const float* w = is_q ? wq : wk;
    float* o = (is_q ? oq : ok) + (t * v.heads + h) * (i64)dk;
    float ss = 0.0f;
    for (int i = lane; i < dk; i += 32) ss += x[i] * x[i];
    const float inv = 1.0f / sqrtf(warp_sum(ss) / (float)dk + eps);
    for (int j = lane; j < rot / 2; j += 32) {
      int a, b;
      pair_at(j, rot, inter, a, b);
      const float2 cs = turn_of((double)pos[t], tab.rev[j]);
      const float ya = x[a] * inv * w[a], yb = x[b] * inv * w[b];
      o[a] = ya * cs.x - yb * cs.y; o[b] = ya * cs.y + yb * cs.x;
    }
    for (int i = rot + lane; i < dk; i += 32) o[i] = x[i] * inv * w[i];
  }
}
// Backward: a CTA's warps take heads in turn; the products g' x-hat of a warp go to its own strip of shared memory.
__global__ void __launch_bounds__(kThreads) k_norm_rope_bwd_any(const __grid_constant__ RopeTable tab, HeadView q, HeadView k, HeadView gq, HeadView gk,
                                                                const float* __restrict__ wq, const float* __restrict__ wk,
                                                                const float* __restrict__ pos, float* __restrict__ dq, float* __restrict__ dkeys,
                                                                float* __restrict__ part, i64 tokens, int dk, int rot, bool inter, float eps) {
  extern __shared__ float strips[];      // [warps][width]
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = kThreads / 32;
  const int per = q.heads + (k.p ? k.heads : 0), width = k.p ? 2 * dk : dk;
  float* mine = strips + wid * width;
  for (int i = lane; i < width; i += 32) mine[i] = 0.0f;
  __syncwarp();
  const i64 rows = tokens * per, step = (i64)gridDim.x * nw;
  for (i64 r = (i64)blockIdx.x * nw + wid; r < rows; r += step) {
    const i64 t = r / per;
    const int hh = (int)(r - t * per);
    const bool is_q = hh < q.heads;
    const HeadView& v = is_q ? q : k;
    const HeadView& gv = is_q ? gq : gk;
    const int h = is_q ? hh : hh - q.heads;
    const float* x = v.p + t * v.st + h * v.sh;
    const float* g = gv.p + t * gv.st + h * gv.sh;
    const float* w = is_q ? wq : wk;
    float* o = (is_q ? dq : dkeys) + (t * v.heads + h) * (i64)dk;
    float* acc = mine + (is_q ? 0 : dk);
    float ss = 0.0f;
    for (int i = lane; i < dk; i += 32) ss += x[i] * x[i];
    const float inv = 1.0f / sqrtf(warp_sum(ss) / (float)dk + eps);
    float c = 0.0f;
    for (int j = lane; j < rot / 2; j += 32) {
      int a, b;
      pair_at(j, rot, inter, a, b);
      const float2 cs = turn_of((double)pos[t], tab.rev[j]);
      const float ga = g[a] * cs.x + g[b] * cs.y, gb = g[b] * cs.x - g[a] * cs.y;
      const float xa = x[a] * inv, xb = x[b] * inv;
      acc[a] += ga * xa; acc[b] += gb * xb;
      c += ga * w[a] * xa + gb * w[b] * xb;
      o[a] = ga * w[a]; o[b] = gb * w[b];          // (finished below by the same lane)
    }
    for (int i = rot + lane; i < dk; i += 32) {
      const float xi = x[i] * inv;
      acc[i] += g[i] * xi;
      c += g[i] * w[i] * xi;
      o[i] = g[i] * w[i];
    }
    c = warp_sum(c) / (float)dk;
    for (int j = lane; j < rot / 2; j += 32) {
      int a, b;
      pair_at(j, rot, inter, a, b);
      o[a] = (o[a] - x[a] * inv * c) * inv; o[b] = (o[b] - x[b] * inv * c) * inv;
    }
    for (int i = rot + lane; i < dk; i += 32) o[i] = (o[i] - x[i] * inv * c) * inv;
    __syncwarp();
  }
  __syncthreads();
  for (int i = threadIdx.x; i < width; i += blockDim.x) {
    float s = 0.0f;
    for (int j = 0; j < nw; ++j) s += strips[j * width + i];
    part[(i64)blockIdx.x * width + i] = s;
  }
}

// the CTAs' partial rows [ctas, width] added in a fixed order: the queries' weight gradient, then the keys'
__global__ void __launch_bounds__(1024) k_weight_sums(const float* __restrict__ part, float* __restrict__ gwq, float* __restrict__ gwk, int dk,
                                                      int width, int ctas) {
  __shared__ float sm[32][33];
  wait_for_last_kernel();
  const int c = (int)blockIdx.x * 32 + threadIdx.x;
  float s = 0.0f;
  if (c < width) for (int i = threadIdx.y; i < ctas; i += 32) s += part[(i64)i * width + c];
  sm[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < width) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += sm[i][threadIdx.x];
    (c < dk ? gwq : gwk)[c < dk ? c : c - dk] = t;
  }
}

bool aligned16(const HeadView& v) { return !v.p || ((reinterpret_cast<uintptr_t>(v.p) & 15) == 0 && v.st % 4 == 0 && v.sh % 4 == 0); }
bool aligned16(const float* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int launch_norm_rope(const RopeTable& tab, const HeadView& q, const HeadView& k, const float* wq, const float* wk, const float* pos,
                     float* oq, float* ok, i64 tokens, int dk, int rot, bool inter, float eps) {
  const int heads = q.heads + (k.p ? k.heads : 0);
  ProfScope prof("norm_rope", 8.0 * (double)tokens * heads * dk);
  if (dk % 8 == 0 && dk <= 256 && rot % 8 == 0 && aligned16(q) && aligned16(k) && aligned16(wq) && (!wk || aligned16(wk))) {
    const size_t smem = (size_t)kWarps * (rot / 2) * sizeof(float2);
    // heads a group of lanes: as many as keep 128 bytes of a lane on their way, one where a warp's four groups hold all heads at once
#define GO(U, I, H) k_norm_rope<U, I, H><<<dim3((unsigned)((tokens + kWarps - 1) / kWarps), (unsigned)((heads + 4 * H - 1) / (4 * H))), kThreads, smem, ctx().stream>>>( \
    tab, q, k, wq, wk, pos, oq, ok, tokens, dk, rot, eps)
#define GO_BY(U, I, H) do { if (H > 1 && heads <= 4) GO(U, I, 1); else GO(U, I, H); } while (0)
    switch ((dk + 63) / 64) {
      case 1: if (inter) GO_BY(1, true, 4); else GO_BY(1, false, 4); break;
      case 2: if (inter) GO_BY(2, true, 2); else GO_BY(2, false, 2); break;
      case 3: if (inter) GO(3, true, 1); else GO(3, false, 1); break;
      default: if (inter) GO(4, true, 1); else GO(4, false, 1); break;
    }
#undef GO_BY
#undef GO
  } else {
    i64 ctas = (tokens * heads + kThreads / 32 - 1) / (kThreads / 32), cap = (i64)ctx().sm_count * 8;
    k_norm_rope_any<<<(unsigned)(ctas < cap ? ctas : cap), kThreads, 0, ctx().stream>>>(tab, q, k, wq, wk, pos, oq, ok, tokens, dk, rot, inter, eps);
  }
  VB_LAUNCH_CHECK();
  return VB_OK;
}

int launch_norm_rope_backward(const RopeTable& tab, const HeadView& q, const HeadView& k, const HeadView& gq, const HeadView& gk, const float* wq,
                              const float* wk, const float* pos, float* dq, float* dkeys, float* gwq, float* gwk, i64 tokens, int dk, int rot, bool inter,
                              float eps) {
  const int heads = q.heads + (k.p ? k.heads : 0), width = k.p ? 2 * dk : dk;
  Temp hold;
  int ctas;
  {
    ProfScope prof("norm_rope_bwd", 12.0 * (double)tokens * heads * dk);
    if (dk % 8 == 0 && dk <= 256 && rot % 8 == 0 && aligned16(q) && aligned16(k) && aligned16(gq) && aligned16(gk) && aligned16(wq) && (!wk || aligned16(wk))) {
      const size_t smem = (size_t)kWarps * (rot / 2) * sizeof(float2);
      const i64 want = (tokens + kWarps - 1) / kWarps;
#define GO(U, I, H) do { \
    const unsigned rows = (unsigned)((heads + 4 * H - 1) / (4 * H)); \
    const i64 cap = (i64)ctx().sm_count * (U == 1 ? 3 : U == 2 ? 2 : 1) / rows > 0 ? (i64)ctx().sm_count * (U == 1 ? 3 : U == 2 ? 2 : 1) / rows : 1; \
    const unsigned cols = (unsigned)(want < cap ? want : cap); \
    ctas = (int)(rows * cols); \
    VB_TRY(scratch_alloc((size_t)ctas * width * sizeof(float), &hold.p)); \
    k_norm_rope_bwd<U, I, H><<<dim3(cols, rows), kThreads, smem, ctx().stream>>>(tab, q, k, gq, gk, wq, wk, pos, dq, dkeys, (float*)hold.p, tokens, dk, rot, eps); \
  } while (0)
#define GO_BY(U, I, H) do { if (H > 1 && heads <= 4) GO(U, I, 1); else GO(U, I, H); } while (0)
      switch ((dk + 63) / 64) {
        case 1: if (inter) GO_BY(1, true, 2); else GO_BY(1, false, 2); break;
        case 2: if (inter) GO(2, true, 1); else GO(2, false, 1); break;
        case 3: if (inter) GO(3, true, 1); else GO(3, false, 1); break;
        default: if (inter) GO(4, true, 1); else GO(4, false, 1); break;
      }
#undef GO_BY
#undef GO
    } else {
      const i64 want = (tokens * heads + kThreads / 32 - 1) / (kThreads / 32), cap = (i64)ctx().sm_count * 4;
      ctas = (int)(want < cap ? want : cap);
      VB_TRY(scratch_alloc((size_t)ctas * width * sizeof(float), &hold.p));
      k_norm_rope_bwd_any<<<(unsigned)ctas, kThreads, (size_t)(kThreads / 32) * width * sizeof(float), ctx().stream>>>(
          tab, q, k, gq, gk, wq, wk, pos, dq, dkeys, (float*)hold.p, tokens, dk, rot, inter, eps);
    }
    VB_LAUNCH_CHECK();
  }
  return launch_early(k_weight_sums, dim3((unsigned)((width + 31) / 32)), dim3(32, 32), 0, (const float*)hold.p, gwq, gwk, dk, width, ctas);
}

}  // namespace vb
