// RMS norm of every query and key head with the rotary position turn in the same pass, forward and backward.
//
//   x-hat = x / sqrt(mean(x^2) + eps),  y = w * x-hat,  (y_a, y_b) -> (y_a c - y_b s, y_a s + y_b c)   for the pair j of a head,
//   c, s = cos, sin of position * theta^(-2j / rot): pairs are (j, j + rot/2), or (2j, 2j + 1) when interleaved; components from
//   rot on are not turned.
//   backward: g' = the turn undone on g;  dx = (w g' - x-hat mean(w g' x-hat)) / sqrt(mean(x^2) + eps);  dw = sum g' x-hat.
//
// HBM-bound: reads each head once and writes it once (backward: reads x and g, writes dx).  Eight lanes own a head, each lane
// "units" of eight components that hold both members of its pairs (two runs of four, rot/2 apart, or eight neighbours), so the
// turn needs no exchange and the norm three shuffles; loads and stores are 16 bytes.  A CTA takes a few tokens and computes
// their cosines and sines once, for all heads.  The angle is formed in turns: position times frequency / 2 pi in 64 bits (the
// frequencies are 64-bit host values in the kernel's parameters), the fraction of a quarter turn in 32, so far positions lose
// nothing.  Head sizes, rotated widths or addresses that do not fit the 16-byte units take a scalar kernel, one warp per head.
#include "common.h"
#include "qk_norm_rope.h"

namespace vb {
namespace {

constexpr int kThreads = 256, kLanes = 8, kGroups = kThreads / kLanes;

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
__device__ __forceinline__ float4 scale4(float4 a, float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); }

__device__ __forceinline__ void fill_turns(float2* cs, const RopeTable& tab, const float* pos, i64 t0, int nt, int half) {
  for (int i = threadIdx.x; i < nt * half; i += blockDim.x) {
    const int t = i / half;
    cs[i] = turn_of((double)pos[t0 + t], tab.rev[i - t * half]);
  }
}

// the heads of one of the two tensors for the CTA's tokens, forward
template <int UPL, bool INTER>
__device__ __forceinline__ void forward_heads(const HeadView& x, const float* __restrict__ w, float* __restrict__ out, const float2* cs,
                                              i64 t0, int nt, int dk, int rot, float eps) {
  const int lane = threadIdx.x & (kLanes - 1), group = threadIdx.x / kLanes;
  const int half = rot / 2;
  float4 wa[UPL], wb[UPL];
  int oa[UPL], ob[UPL];
#pragma unroll
  for (int i = 0; i < UPL; ++i) {
    const int u = lane + i * kLanes;
    unit_at<INTER>(u, rot, oa[i], ob[i]);
    wa[i] = wb[i] = make_float4(0, 0, 0, 0);
    if (8 * u < dk) { wa[i] = *reinterpret_cast<const float4*>(w + oa[i]); wb[i] = *reinterpret_cast<const float4*>(w + ob[i]); }
  }
  const float rdk = 1.0f / (float)dk;
  const int rows = nt * x.heads;
  for (int r0 = 0; r0 < rows; r0 += kGroups) {      // (whole groups stay together: the shuffles below name every lane)
    const int r = r0 + group;
    const bool live = r < rows;
    const int t = live ? r / x.heads : 0, h = live ? r - t * x.heads : 0;
    const float* p = x.p + (t0 + t) * x.st + h * x.sh;
    float4 a[UPL], b[UPL];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      a[i] = b[i] = make_float4(0, 0, 0, 0);
      if (live && 8 * (lane + i * kLanes) < dk) { a[i] = *reinterpret_cast<const float4*>(p + oa[i]); b[i] = *reinterpret_cast<const float4*>(p + ob[i]); }
      ss += dot4(a[i], a[i]) + dot4(b[i], b[i]);
    }
    const float inv = 1.0f / sqrtf(group_sum(ss) * rdk + eps);
    float* o = out + ((t0 + t) * x.heads + h) * (i64)dk;
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      const int u = lane + i * kLanes;
      if (!live || 8 * u >= dk) continue;
      float4 ya = mul4(scale4(a[i], inv), wa[i]), yb = mul4(scale4(b[i], inv), wb[i]);
      if (8 * u < rot) turn_unit<INTER>(ya, yb, cs + t * half, u, 1.0f);
      *reinterpret_cast<float4*>(o + oa[i]) = ya;
      *reinterpret_cast<float4*>(o + ob[i]) = yb;
    }
  }
}
template <int UPL, bool INTER>
__global__ void __launch_bounds__(kThreads) k_norm_rope(const __grid_constant__ RopeTable tab, HeadView q, HeadView k, const float* __restrict__ wq,
                                                        const float* __restrict__ wk, const float* __restrict__ pos, float* __restrict__ oq,
                                                        float* __restrict__ ok, i64 tokens, int per_cta, int dk, int rot, float eps) {
  extern __shared__ float2 cs[];
  const i64 t0 = (i64)blockIdx.x * per_cta;
  const int nt = (int)(tokens - t0 < per_cta ? tokens - t0 : per_cta);
  fill_turns(cs, tab, pos, t0, nt, rot / 2);
  __syncthreads();
  forward_heads<UPL, INTER>(q, wq, oq, cs, t0, nt, dk, rot, eps);
  if (k.p) forward_heads<UPL, INTER>(k, wk, ok, cs, t0, nt, dk, rot, eps);
}

// ... backward; acc: this lane's sums of g' x-hat over the heads it has seen
template <int UPL, bool INTER>
__device__ __forceinline__ void backward_heads(const HeadView& x, const HeadView& g, const float* __restrict__ w, float* __restrict__ gx,
                                               const float2* cs, i64 t0, int nt, int dk, int rot, float eps, float4 (&acc)[2 * UPL]) {
  const int lane = threadIdx.x & (kLanes - 1), group = threadIdx.x / kLanes;
  const int half = rot / 2;
  const float rdk = 1.0f / (float)dk;
  const int rows = nt * x.heads;
  for (int r0 = 0; r0 < rows; r0 += kGroups) {
    const int r = r0 + group;
    const bool live = r < rows;
    const int t = live ? r / x.heads : 0, h = live ? r - t * x.heads : 0;
    const float* px = x.p + (t0 + t) * x.st + h * x.sh;
    const float* pg = g.p + (t0 + t) * g.st + h * g.sh;
    float4 a[UPL], b[UPL], ga[UPL], gb[UPL];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      const int u = lane + i * kLanes;
      int oa, ob;
      unit_at<INTER>(u, rot, oa, ob);
      a[i] = b[i] = ga[i] = gb[i] = make_float4(0, 0, 0, 0);
      if (live && 8 * u < dk) {
        a[i] = *reinterpret_cast<const float4*>(px + oa); b[i] = *reinterpret_cast<const float4*>(px + ob);
        ga[i] = *reinterpret_cast<const float4*>(pg + oa); gb[i] = *reinterpret_cast<const float4*>(pg + ob);
      }
      ss += dot4(a[i], a[i]) + dot4(b[i], b[i]);
    }
    const float inv = 1.0f / sqrtf(group_sum(ss) * rdk + eps);
    float c = 0.0f;
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      const int u = lane + i * kLanes;
      if (8 * u >= dk) continue;
      if (8 * u < rot) turn_unit<INTER>(ga[i], gb[i], cs + t * half, u, -1.0f);
      a[i] = scale4(a[i], inv); b[i] = scale4(b[i], inv);      // x-hat
      const float4 pa = mul4(ga[i], a[i]), pb = mul4(gb[i], b[i]);
      if (live) {
        acc[2 * i].x += pa.x; acc[2 * i].y += pa.y; acc[2 * i].z += pa.z; acc[2 * i].w += pa.w;
        acc[2 * i + 1].x += pb.x; acc[2 * i + 1].y += pb.y; acc[2 * i + 1].z += pb.z; acc[2 * i + 1].w += pb.w;
      }
      int oa, ob;
      unit_at<INTER>(u, rot, oa, ob);
      ga[i] = mul4(ga[i], *reinterpret_cast<const float4*>(w + oa)); gb[i] = mul4(gb[i], *reinterpret_cast<const float4*>(w + ob));
      c += dot4(ga[i], a[i]) + dot4(gb[i], b[i]);
    }
    c = group_sum(c) * rdk;
    float* o = gx + ((t0 + t) * x.heads + h) * (i64)dk;
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      const int u = lane + i * kLanes;
      if (!live || 8 * u >= dk) continue;
      int oa, ob;
      unit_at<INTER>(u, rot, oa, ob);
      float4 ra, rb;
      ra.x = (ga[i].x - a[i].x * c) * inv; ra.y = (ga[i].y - a[i].y * c) * inv; ra.z = (ga[i].z - a[i].z * c) * inv; ra.w = (ga[i].w - a[i].w * c) * inv;
      rb.x = (gb[i].x - b[i].x * c) * inv; rb.y = (gb[i].y - b[i].y * c) * inv; rb.z = (gb[i].z - b[i].z * c) * inv; rb.w = (gb[i].w - b[i].w * c) * inv;
      *reinterpret_cast<float4*>(o + oa) = ra;
      *reinterpret_cast<float4*>(o + ob) = rb;
    }
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
template <int UPL, bool INTER>
__global__ void __launch_bounds__(kThreads) k_norm_rope_bwd(const __grid_constant__ RopeTable tab, HeadView q, HeadView k, HeadView gq, HeadView gk,
                                                            const float* __restrict__ wq, const float* __restrict__ wk, const float* __restrict__ pos,
                                                            float* __restrict__ dq, float* __restrict__ dkeys, float* __restrict__ part,
                                                            i64 tokens, int per_cta, int dk, int rot, float eps) {
  extern __shared__ float2 cs[];
  __shared__ __align__(16) float sums[kGroups * 64];
  float4 accq[2 * UPL], acck[2 * UPL];
#pragma unroll
  for (int i = 0; i < 2 * UPL; ++i) accq[i] = acck[i] = make_float4(0, 0, 0, 0);
  for (i64 t0 = (i64)blockIdx.x * per_cta; t0 < tokens; t0 += (i64)gridDim.x * per_cta) {
    const int nt = (int)(tokens - t0 < per_cta ? tokens - t0 : per_cta);
    __syncthreads();
    fill_turns(cs, tab, pos, t0, nt, rot / 2);
    __syncthreads();
    backward_heads<UPL, INTER>(q, gq, wq, dq, cs, t0, nt, dk, rot, eps, accq);
    if (k.p) backward_heads<UPL, INTER>(k, gk, wk, dkeys, cs, t0, nt, dk, rot, eps, acck);
  }
  // partial sums: one row of [dk] (queries) and, where there are keys, one more behind it per CTA
  const int width = k.p ? 2 * dk : dk;
  store_weight_sums<UPL, INTER>(accq, part + (i64)blockIdx.x * width, sums, dk, rot);
  if (k.p) store_weight_sums<UPL, INTER>(acck, part + (i64)blockIdx.x * width + dk, sums, dk, rot);
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

// tokens a CTA takes: enough heads for every group of lanes, at most 8 KB of cosines and sines
int tokens_per_cta(int heads, int rot) {
  int n = (2 * kGroups + heads - 1) / heads;
  const int cap = rot > 0 ? 2048 / rot : 64;
  if (n > cap) n = cap;
  return n < 1 ? 1 : n;
}

}  // namespace

int launch_norm_rope(const RopeTable& tab, const HeadView& q, const HeadView& k, const float* wq, const float* wk, const float* pos,
                     float* oq, float* ok, i64 tokens, int dk, int rot, bool inter, float eps) {
  const int heads = q.heads + (k.p ? k.heads : 0);
  ProfScope prof("norm_rope", 8.0 * (double)tokens * heads * dk);
  if (dk % 8 == 0 && dk <= 256 && rot % 8 == 0 && aligned16(q) && aligned16(k) && aligned16(wq) && (!wk || aligned16(wk))) {
    const int per = tokens_per_cta(heads, rot);
    const i64 ctas = (tokens + per - 1) / per;
    const size_t smem = (size_t)per * (rot / 2) * sizeof(float2);
#define GO(U, I) k_norm_rope<U, I><<<(unsigned)ctas, kThreads, smem, ctx().stream>>>(tab, q, k, wq, wk, pos, oq, ok, tokens, per, dk, rot, eps)
    switch ((dk + 63) / 64) {
      case 1: if (inter) GO(1, true); else GO(1, false); break;
      case 2: if (inter) GO(2, true); else GO(2, false); break;
      case 3: if (inter) GO(3, true); else GO(3, false); break;
      default: if (inter) GO(4, true); else GO(4, false); break;
    }
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
      const int per = tokens_per_cta(heads, rot);
      const i64 want = (tokens + per - 1) / per, cap = (i64)ctx().sm_count * 4;
      ctas = (int)(want < cap ? want : cap);
      const size_t smem = (size_t)per * (rot / 2) * sizeof(float2);
      VB_TRY(scratch_alloc((size_t)ctas * width * sizeof(float), &hold.p));
#define GO(U, I) k_norm_rope_bwd<U, I><<<(unsigned)ctas, kThreads, smem, ctx().stream>>>(tab, q, k, gq, gk, wq, wk, pos, dq, dkeys, (float*)hold.p, tokens, per, dk, rot, eps)
      switch ((dk + 63) / 64) {
        case 1: if (inter) GO(1, true); else GO(1, false); break;
        case 2: if (inter) GO(2, true); else GO(2, false); break;
        case 3: if (inter) GO(3, true); else GO(3, false); break;
        default: if (inter) GO(4, true); else GO(4, false); break;
      }
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
  k_weight_sums<<<(unsigned)((width + 31) / 32), dim3(32, 32), 0, ctx().stream>>>((const float*)hold.p, gwq, gwk, dk, width, ctas);
  VB_LAUNCH_CHECK();
  return VB_OK;
}

}  // namespace vb
