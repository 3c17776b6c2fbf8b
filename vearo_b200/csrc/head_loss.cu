// The vocabulary projection with its softmax cross entropy, forward and backward, without the logits in memory.
//
//   z = x W^T,  lse_n = log sum_v exp z_nv,  loss = mean over rows with a target of (lse_n - z_n,target)
//   dz = (exp(z - lse) - onehot) g / count,   dx = dz W,   dW = dz^T x
//
// Forward: one product whose tiles leave (max, sum of exp) for each row and 128 columns, 8 bytes where the logits would be 512, and
// the target's logit; a second kernel joins the pairs of a row.  Backward: pieces of the vocabulary; a piece's logits are formed
// again and leave the tensor core as dz in half-precision planes, on one scale for dx and with a scale for 128 rows of a class for dW, and one launch
// adds the piece to dx and writes its rows of dW.  Tensor-bound: 2 N V D and 6 N V D operations, three instructions each (gemm16.cu):
// 8192 rows, 768 x 50304: 1.39 to 1.56 ms forward, as the power limit has it; 4097 rows, 1024 x 50304, with the gradients 4.9 to 5.0 ms (4.7 with the one
// scale for both).
// Up to 16 rows it is bound by the bytes of W and takes them in 32 bits, and so do small products of more rows (below).
#include "gemm16.h"
#include "head_loss.h"
#include "split16.cuh"

namespace vb {
namespace {

// Backward, one CTA: every row's target, the products' tile counters and coef = g / (rows with a target).
__global__ void __launch_bounds__(1024) k_targets(const float* __restrict__ targets, i64 n, i64 ignore, i64 vocab, int* __restrict__ out,
                                                  const float* __restrict__ g, float* __restrict__ coef, int* counters, int n_counters, int* err) {
  __shared__ int red[32];
  for (int i = threadIdx.x; i < n_counters; i += 1024) counters[i] = 0;      // of the products that follow
  int live = 0;
  for (i64 i = threadIdx.x; i < n; i += 1024) {
    const int t = read_target(targets[i], ignore, vocab, err);
    out[i] = t;
    live += t != kNoTarget;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) live += __shfl_xor_sync(0xffffffffu, live, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = live;
  __syncthreads();
  if (threadIdx.x == 0) {
    int c = 0;
    for (int i = 0; i < 32; ++i) c += red[i];
    *coef = *g / (float)(c > 0 ? c : 1);
  }
}
// lse and the row's loss from its pairs, joined in a fixed order: R rows x 1024 / R lanes a CTA; the CTA that ends last takes the mean over the
// rows, in a fixed order too.  (As a kernel of its own the mean cost 3 us of 28 at 33 x 128 x 512.)
__device__ __forceinline__ void join_pair(float& m, float& s, float2 a) {
  if (a.x > m) { s = s * expf(m - a.x) + a.y; m = a.x; }
  else if (a.y != 0.0f) s += a.y * expf(a.x - m);          // (a pair of NaN sum keeps it)
}
template <int R>
__global__ void __launch_bounds__(1024) k_join_stats(const float2* __restrict__ stats, const float* __restrict__ target_value, const int* __restrict__ target,
                                                     float* __restrict__ lse, float* nll, float* __restrict__ loss, int* ticket, int n, int pairs) {
  __shared__ float2 part[32][R];
  __shared__ float sums[32];
  __shared__ int counts[32];
  __shared__ bool last;
  wait_for_last_kernel();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x * R + tid % R;
  float m = -INFINITY, s = 0.0f;
  if (row < n) {
    int i = tid / R;
    for (; i + 3 * (1024 / R) < pairs; i += 4 * (1024 / R)) {
      float2 a[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = stats[(i64)(i + j * (1024 / R)) * n + row];
#pragma unroll
      for (int j = 0; j < 4; ++j) join_pair(m, s, a[j]);
    }
    for (; i < pairs; i += (1024 / R)) join_pair(m, s, stats[(i64)i * n + row]);
  }
  // the lanes of a row within a warp, then the warps
#pragma unroll
  for (int o = 16; o >= R; o >>= 1) {
    const float2 a = make_float2(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
    const float top = fmaxf(m, a.x);
    s = top > -INFINITY ? (m > -INFINITY ? s * expf(m - top) : s) + (a.x > -INFINITY ? a.y * expf(a.x - top) : a.y) : s + a.y;
    m = top;
  }
  if (lane < R) part[warp][lane] = make_float2(m, s);
  __syncthreads();
  if (warp < R) {
    const float2 a = part[lane][warp];
    m = a.x; s = a.y;
    float top = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    s = top > -INFINITY && m > -INFINITY ? s * expf(m - top) : s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const int r = blockIdx.x * R + warp;
    if (lane == 0 && r < n) {
      const float l = top + logf(s);
      lse[r] = l;
      nll[r] = target[r] == kNoTarget ? 0.0f : l - target_value[r];
      __threadfence();
    }
  }
  __syncthreads();
  if (tid == 0) { last = atomicAdd(ticket, 1) == (int)gridDim.x - 1; __threadfence(); }
  __syncthreads();
  if (!last) return;
  float t = 0.0f;
  int live = 0;
  for (int i = tid; i < n; i += 1024) { t += __ldcg(nll + i); live += target[i] != kNoTarget; }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { t += __shfl_xor_sync(0xffffffffu, t, o); live += __shfl_xor_sync(0xffffffffu, live, o); }
  if (lane == 0) { sums[warp] = t; counts[warp] = live; }
  __syncthreads();
  if (tid == 0) {
    float all = 0.0f;
    int c = 0;
    for (int i = 0; i < 32; ++i) { all += sums[i]; c += counts[i]; }
    *loss = c > 0 ? all / (float)c : 0.0f;
  }
}

// Eight rows a CTA where that fills more of the SMs and a row has pairs for its lanes (64 rows of 393 pairs: 15 us with 32), else 32 (4000 rows of 3
// pairs: 3 us more with eight).
int launch_join_stats(const float2* stats, const float* target_value, const int* target, float* lse, float* nll, float* loss, int* ticket, i64 n, i64 pairs) {
  if (n <= 1024 && pairs > 32)
    return launch_early(k_join_stats<8>, dim3((unsigned)((n + 7) / 8)), dim3(1024), 0, stats, target_value, target, lse, nll, loss, ticket, (int)n, (int)pairs);
  return launch_early(k_join_stats<32>, dim3((unsigned)((n + 31) / 32)), dim3(1024), 0, stats, target_value, target, lse, nll, loss, ticket, (int)n, (int)pairs);
}

// ---- few rows -------------------------------------------------------------------------------------------------------------------
// With up to 16 rows W is read for little arithmetic: splitting it into planes (read, written, read again) would cost three times its
// bytes.  Here W is read once, in 32 bits, and multiplied on the ordinary cores; backward, one pass forms a block's logits again, writes its rows of
// dW and adds its part of dx.  With W of 1024 x 50304, forward: 54 us at 1 row, 58 at 8, 70 at 16, against 140 by way of planes; with the gradients 181, 201 and 303 against 441 to 450.
// A CTA goes over blocks of 64 columns: a warp's four rows of W against the rows of x in shared memory, sums joined by a
// transposing butterfly; then (forward) a warp a row of x for the block's (max, sum), or (backward) a warp 128 of the width for dW and dx.
constexpr int kFewThreads = 512, kFewWarps = kFewThreads / 32, kFewCols = 4 * kFewWarps, kFewRows = 16, kFewWidth = 128 * kFewWarps;
struct FewParams {
  const float *x, *w, *targets;
  i64 ignore;
  int n, d, v;
  float2* stats; float* target_value; int* target; int* ticket;             // forward
  const float *lse, *g; float *gw, *gx_part;                                // backward; gw: [groups of NR rows][v][d], gx_part: [CTAs][n][d]
  int* err;
};
template <int NR, bool GRAD>
__global__ void __launch_bounds__(kFewThreads, 1) k_few_rows(FewParams p) {
  extern __shared__ float4 few_smem[];
  float* xs = reinterpret_cast<float*>(few_smem);      // [NR][d]
  float* zs = xs + NR * p.d;                           // two of [NR][kFewCols]: logits, then dz
  __shared__ int target[NR];
  __shared__ float lse[NR], coef;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row0 = blockIdx.y * NR, rows = min(NR, p.n - row0), d = p.d;
  const int blocks = (p.v + kFewCols - 1) / kFewCols;
  float4 cur[4], nxt[4];
  auto load = [&](float4 (&to)[4], int blk, int c) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int v = blk * kFewCols + warp * 4 + r;
      to[r] = v < p.v && c < d ? __ldg(reinterpret_cast<const float4*>(p.w + (i64)v * d + c)) : make_float4(0, 0, 0, 0);
    }
  };
  load(cur, blockIdx.x, lane * 4);
  if (tid < NR) {
    target[tid] = tid < rows ? read_target(p.targets[row0 + tid], p.ignore, p.v, p.err) : kNoTarget;
    if (GRAD) lse[tid] = tid < rows ? p.lse[row0 + tid] : 0.0f;
    else if (blockIdx.x == 0 && tid < rows) p.target[row0 + tid] = target[tid];
  }
  if (!GRAD && tid == 0 && blockIdx.x == 0 && blockIdx.y == 0) *p.ticket = 0;
  __syncthreads();
  if (GRAD) {
    int live = 0;
    for (int i0 = 0; i0 < p.n; i0 += kFewThreads) {
      const int i = i0 + tid;
      live += __syncthreads_count(i < p.n && read_target(p.targets[i], p.ignore, p.v, p.err) != kNoTarget);
    }
    if (tid == 0) coef = *p.g / (float)(live > 0 ? live : 1);
  }
  for (int i = tid * 4; i < NR * d; i += kFewThreads * 4) {      // (backward, a row that is left out may hold anything)
    const int n = i / d;
    *reinterpret_cast<float4*>(xs + i) = n < rows && !(GRAD && target[n] == kNoTarget) ? *reinterpret_cast<const float4*>(p.x + (i64)row0 * d + i) : make_float4(0, 0, 0, 0);
  }
  __syncthreads();
  // backward: this warp's 128 of the width, and which of the block's rows
  const int slices = (d + 127) / 128, groups = kFewWarps / slices, group = warp / slices, col = (warp % slices) * 128 + lane * 4;
  float4 dx[GRAD ? NR : 1];
#pragma unroll
  for (int n = 0; n < (GRAD ? NR : 1); ++n) dx[n] = make_float4(0, 0, 0, 0);
  for (int blk = blockIdx.x, turn = 0; blk < blocks; blk += gridDim.x, turn ^= 1) {
    float* z = zs + turn * NR * kFewCols;
    float acc[NR * 4];
#pragma unroll
    for (int i = 0; i < NR * 4; ++i) acc[i] = 0.0f;
    for (int c = lane * 4; c < (d + 127) / 128 * 128; c += 128) {
      if (c + 128 < (d + 127) / 128 * 128) load(nxt, blk, c + 128); else load(nxt, blk + gridDim.x, lane * 4);
      if (c < d) {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const float4 x = *reinterpret_cast<const float4*>(xs + n * d + c);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float a = acc[n * 4 + r];
            a = fmaf(x.x, cur[r].x, a); a = fmaf(x.y, cur[r].y, a); a = fmaf(x.z, cur[r].z, a); a = fmaf(x.w, cur[r].w, a);
            acc[n * 4 + r] = a;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) cur[r] = nxt[r];
    }
    // sums over the lanes: half of the values go to the other half of the lanes, until a lane has NR / 8 of them (or two lanes share one)
    int have = NR * 4;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (have > 1) {
        have /= 2;
#pragma unroll
        for (int i = 0; i < NR * 2; ++i) {
          if (i < have) {
            const float keep = lane & o ? acc[i + have] : acc[i], send = lane & o ? acc[i] : acc[i + have];
            acc[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
          }
        }
      } else acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], o);
    }
    if (NR >= 8 || (lane & 1) == 0) {
#pragma unroll
      for (int i = 0; i < (NR >= 8 ? NR / 8 : 1); ++i) {
        const int at = NR >= 8 ? lane * (NR / 8) + i : lane >> 1;
        z[(at >> 2) * kFewCols + warp * 4 + (at & 3)] = acc[i];
      }
    }
    __syncthreads();
    const int v0 = blk * kFewCols;
    if (!GRAD) {
      if (warp < rows) {
        const int left = p.v - v0;
        const float a = lane < left ? z[warp * kFewCols + lane] : -INFINITY, b = lane + 32 < left ? z[warp * kFewCols + lane + 32] : -INFINITY;
        float m = fmaxf(a, b);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float sum = m > -INFINITY ? expf(a - m) + expf(b - m) : (lane < left ? expf(a) : 0.0f) + (lane + 32 < left ? expf(b) : 0.0f);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) p.stats[(i64)blk * p.n + row0 + warp] = make_float2(m, sum);
        const int t = target[warp] - v0;
        if (lane == 0 && t >= 0 && t < kFewCols) p.target_value[row0 + warp] = z[warp * kFewCols + t];
      }
    } else {
      for (int i = tid; i < NR * kFewCols; i += kFewThreads) {
        const int n = i / kFewCols, v = v0 + i % kFewCols;
        z[i] = target[n] != kNoTarget && v < p.v ? coef * (expf(z[i] - lse[n]) - (target[n] == v ? 1.0f : 0.0f)) : 0.0f;
      }
      __syncthreads();
      if (group < groups && col < d) {
        for (int r0 = group * 4; r0 < kFewCols && v0 + r0 < p.v; r0 += groups * 4) {
          float4 w[4], dw[4];
          const float* src = p.w + (i64)(v0 + r0) * d + col;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            dw[r] = make_float4(0, 0, 0, 0);
            w[r] = v0 + r0 + r < p.v ? __ldg(reinterpret_cast<const float4*>(src + (i64)r * d)) : dw[r];
          }
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            const float4 x = *reinterpret_cast<const float4*>(xs + n * d + col), g4 = *reinterpret_cast<const float4*>(z + n * kFewCols + r0);
            const float g[4] = {g4.x, g4.y, g4.z, g4.w};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              dw[r].x = fmaf(g[r], x.x, dw[r].x); dw[r].y = fmaf(g[r], x.y, dw[r].y); dw[r].z = fmaf(g[r], x.z, dw[r].z); dw[r].w = fmaf(g[r], x.w, dw[r].w);
              dx[n].x = fmaf(g[r], w[r].x, dx[n].x); dx[n].y = fmaf(g[r], w[r].y, dx[n].y); dx[n].z = fmaf(g[r], w[r].z, dx[n].z); dx[n].w = fmaf(g[r], w[r].w, dx[n].w);
            }
          }
          if (p.gw) {
#pragma unroll
            for (int r = 0; r < 4; ++r) if (v0 + r0 + r < p.v) __stcs(reinterpret_cast<float4*>(p.gw + ((i64)blockIdx.y * p.v + v0 + r0 + r) * d + col), dw[r]);
          }
        }
      }
    }
  }
  if (GRAD && p.gx_part) {      // the groups' sums in order, where x was
    for (int g = 0; g < groups; ++g) {
      __syncthreads();
      if (group == g && col < d) {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          float4* to = reinterpret_cast<float4*>(xs + n * d + col);
          const float4 a = g > 0 ? *to : make_float4(0, 0, 0, 0);
          *to = make_float4(a.x + dx[n].x, a.y + dx[n].y, a.z + dx[n].z, a.w + dx[n].w);
        }
      }
    }
    __syncthreads();
    float* to = p.gx_part + ((i64)blockIdx.x * p.n + row0) * d;
    for (int i = tid * 4; i < rows * d; i += kFewThreads * 4) *reinterpret_cast<float4*>(to + i) = *reinterpret_cast<const float4*>(xs + i);
  }
}
// the CTAs' parts added in a fixed order: 32 numbers x 32 lanes of parts a CTA
__global__ void __launch_bounds__(1024) k_sum_few(const float* __restrict__ part, float* __restrict__ out, int numbers, int parts) {
  __shared__ float sm[32][33];
  const int at = blockIdx.x * 32 + threadIdx.x;
  float s = 0.0f;
  if (at < numbers) {
#pragma unroll 5
    for (int i = threadIdx.y; i < parts; i += 32) s += part[(i64)i * numbers + at];
  }
  sm[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && at < numbers) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += sm[i][threadIdx.x];
    out[at] = t;
  }
}
// the groups' parts of dW added in order
__global__ void __launch_bounds__(256) k_sum_groups(const float4* __restrict__ part, float4* __restrict__ out, int numbers, int groups) {
  wait_for_last_kernel();
  const int at = blockIdx.x * 256 + threadIdx.x;
  if (at >= numbers) return;
  float4 s = part[at];
#pragma unroll 4
  for (int i = 1; i < groups; ++i) {
    const float4 a = part[(i64)i * numbers + at];
    s = make_float4(s.x + a.x, s.y + a.y, s.z + a.z, s.w + a.w);
  }
  out[at] = s;
}
bool few_fit(i64 d) { return d % 4 == 0 && d <= kFewWidth; }
// the matrix where it is, or a copy that begins on 16 bytes (the same kernel for either: the same bits)
int on_16_bytes(const float** x, i64 numbers, Temp& hold) {
  if ((reinterpret_cast<uintptr_t>(*x) & 15) == 0) return VB_OK;
  VB_TRY(scratch_alloc((size_t)numbers * sizeof(float), &hold.p));
  VB_CUDA(cudaMemcpyAsync(hold.p, *x, (size_t)numbers * sizeof(float), cudaMemcpyDeviceToDevice, ctx().stream));
  *x = (const float*)hold.p;
  return VB_OK;
}
template <int NR, bool GRAD>
int few_rows(const FewParams& p, unsigned ctas, unsigned groups) {
  const int smem = (NR * p.d + 2 * NR * kFewCols) * 4;
  static const int ready = [] {
    VB_CUDA(cudaFuncSetAttribute(k_few_rows<NR, GRAD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (NR * kFewWidth + 2 * NR * kFewCols) * 4));
    return (int)VB_OK;
  }();
  VB_TRY(ready);
  k_few_rows<NR, GRAD><<<dim3(ctas, groups), kFewThreads, smem, ctx().stream>>>(p);
  VB_LAUNCH_CHECK();
  return VB_OK;
}
template <bool GRAD>
int few_rows(const FewParams& p, unsigned ctas, unsigned groups) {
  if (p.n <= 4) return few_rows<4, GRAD>(p, ctas, groups);
  return p.n <= 8 ? few_rows<8, GRAD>(p, ctas, groups) : few_rows<kFewRows, GRAD>(p, ctas, groups);
}

// Half-precision planes of a piece of dz: at most half a gigabyte at a time for dx, and as much for dW.
constexpr i64 kPieceBytes = (i64)512 << 20;

}  // namespace

int launch_head_loss(const float* x, const float* w, const float* targets, i64 ignore, float* loss, float* lse, i64 n, i64 d, i64 v) {
  Temp hx, hw, hs, hr;
  // Few rows, or so few blocks of logits that one wave of the ordinary cores is through before W has been split
  const i64 few_blocks = (v + kFewCols - 1) / kFewCols, few_groups = (n + kFewRows - 1) / kFewRows;
  const bool few = few_fit(d) && (n <= kFewRows || few_blocks * few_groups <= ctx().sm_count);
  const i64 pairs = few ? few_blocks : (v + 127) / 128;
  if (few) {
    VB_TRY(on_16_bytes(&x, n * d, hx)); VB_TRY(on_16_bytes(&w, v * d, hw));
    VB_TRY(scratch_alloc((size_t)(pairs * n) * sizeof(float2), &hs.p));
    VB_TRY(scratch_alloc((size_t)n * 12 + 4, &hr.p));
    float* nll = (float*)hr.p; float* tv = nll + n; int* tgt = (int*)(tv + n);
    FewParams p{};
    p.x = x; p.w = w; p.targets = targets; p.ignore = ignore; p.n = (int)n; p.d = (int)d; p.v = (int)v;
    p.stats = (float2*)hs.p; p.target_value = tv; p.target = tgt; p.ticket = tgt + n; p.err = ctx().d_err;
    VB_TRY(few_rows<false>(p, (unsigned)(few_blocks < ctx().sm_count ? few_blocks : ctx().sm_count), (unsigned)few_groups));
    return launch_join_stats((const float2*)hs.p, tv, tgt, lse, nll, loss, tgt + n, n, pairs);
  }
  VB_TRY(scratch_alloc(split16_bytes(n, d, Scale16::Row), &hx.p));
  VB_TRY(scratch_alloc(split16_bytes(v, d), &hw.p));
  VB_TRY(scratch_alloc((size_t)(pairs * n) * sizeof(float2), &hs.p));
  VB_TRY(scratch_alloc((size_t)n * 12 + 8, &hr.p));
  float* nll = (float*)hr.p; float* tv = nll + n; int* tgt = (int*)(tv + n); int* counters = tgt + n;
  const Split16 sx = split16_at(hx.p, n, d, Scale16::Row), sw = split16_at(hw.p, v, d);
  const SplitJob jobs[2] = {{x, sx}, {w, sw}};
  const TargetRows rows{targets, ignore, v, tgt, counters, 2};
  VB_TRY(launch_split16(jobs, 2, &rows));
  Product16 g{};
  g.a = Op16{sx, false}; g.b = Op16{sw, false}; g.M = n; g.N = v; g.K = d;
  g.target = tgt; g.stats = (float2*)hs.p; g.target_value = tv;
  VB_TRY(launch_gemm16(Tile16::RowStats, &g, 1, counters));
  return launch_join_stats((const float2*)hs.p, tv, tgt, lse, nll, loss, counters + 1, n, pairs);
}

int launch_head_loss_backward(const float* x, const float* w, const float* targets, i64 ignore, const float* lse, const float* g, float* gx, float* gw,
                              i64 n, i64 d, i64 v) {
  Temp hx, hk, hw, hz, hc, ht;
  const i64 few_blocks = (v + kFewCols - 1) / kFewCols, few_groups = (n + kFewRows - 1) / kFewRows;
  // Up to 16 rows, or one wave of blocks that are not wide (a block's three products take 16 x 64 x d each on the ordinary cores) and not of many groups (whose
  // parts of dW are added).  With gradients, this way / by way of planes, us: 17 rows of 64, 700 columns 38 / 52; 100 of 512, 1000: 54 / 72; 500 of 128, 256: 49 / 57;
  // and left to the planes 64 of 1024, 300: 74 / 70; 1000 of 512, 128: 96 / 78; 2000 of 256, 64: 89 / 76.
  if (few_fit(d) && (n <= kFewRows || (few_blocks * few_groups <= ctx().sm_count && d <= 512 && d * few_groups <= 8192))) {
    VB_TRY(on_16_bytes(&x, n * d, hk)); VB_TRY(on_16_bytes(&w, v * d, hw));
    const i64 ctas = few_blocks < ctx().sm_count ? few_blocks : ctx().sm_count;
    FewParams p{};
    p.x = x; p.w = w; p.targets = targets; p.ignore = ignore; p.n = (int)n; p.d = (int)d; p.v = (int)v;
    p.lse = lse; p.g = g; p.gw = gw; p.err = ctx().d_err;
    if (gx) {
      VB_TRY(scratch_alloc((size_t)(ctas * n * d) * sizeof(float), &hx.p));
      p.gx_part = (float*)hx.p;
    }
    if (gw && few_groups > 1) {
      VB_TRY(scratch_alloc((size_t)(few_groups * v * d) * sizeof(float), &hz.p));
      p.gw = (float*)hz.p;
    }
    VB_TRY(few_rows<true>(p, (unsigned)ctas, (unsigned)few_groups));
    if (gw && few_groups > 1)
      VB_TRY(launch_early(k_sum_groups, dim3((unsigned)((v * d / 4 + 255) / 256)), dim3(256), 0, (const float4*)hz.p, (float4*)gw, (int)(v * d / 4), (int)few_groups));
    if (gx) {
      const dim3 grid((unsigned)((n * d + 31) / 32));
      k_sum_few<<<grid, dim3(32, 32), 0, ctx().stream>>>((const float*)hx.p, gx, (int)(n * d), (int)ctas);
      VB_LAUNCH_CHECK();
    }
    return VB_OK;
  }
  i64 piece = kPieceBytes / (4 * n) / 256 * 256;
  if (piece < 256) piece = 256;
  const i64 pieces = (v + piece - 1) / piece;
  piece = ((v + pieces - 1) / pieces + 255) / 256 * 256;
  if (piece > v) piece = v;
  VB_TRY(scratch_alloc(split16_bytes(n, d, Scale16::Row), &hx.p));
  if (gw) VB_TRY(scratch_alloc(split16_bytes(n, d), &hk.p));
  VB_TRY(scratch_alloc(split16_bytes(v, d), &hw.p));
  if (gx) VB_TRY(scratch_alloc(split16_bytes(n, piece), &hz.p));
  if (gw) VB_TRY(scratch_alloc(split16_bytes(n, piece, Scale16::Column), &hc.p));
  VB_TRY(scratch_alloc((size_t)(n + 2 * pieces) * 4 + 16, &ht.p));
  float* coef = (float*)ht.p; int* tgt = (int*)(coef + 4); int* counters = tgt + n;
  const Split16 sx = split16_at(hx.p, n, d, Scale16::Row), sw = split16_at(hw.p, v, d);      // x for the logits, where its rows are the product's,
  const Split16 sk = gw ? split16_at(hk.p, n, d) : sx;                                  // and for dW, which sums over them
  k_targets<<<1, 1024, 0, ctx().stream>>>(targets, n, ignore, v, tgt, g, coef, counters, (int)(2 * pieces), ctx().d_err);
  VB_LAUNCH_CHECK();
  const SplitJob jobs[3] = {{w, sw}, {x, sx, tgt}, {x, sk, tgt}};        // (rows that are left out may hold anything: they must not reach dW)
  VB_TRY(launch_split16(jobs, gw ? 3 : 2));
  for (i64 v0 = 0; v0 < v; v0 += piece, counters += 2) {
    const i64 vc = v - v0 < piece ? v - v0 : piece;
    Split16 wc = sw;                                     // this piece's rows of W
    wc.planes = (uint16_t*)sw.planes + v0 * sw.ld; wc.inv = sw.inv + v0 / 128 * sw.inv_ld; wc.rows = vc;
    // A row of dx sums over classes whose probabilities add up to 1, so one scale does for all of them.  A row of dW belongs to one class, however
    // improbable: its dz are held on the scale of the largest among 128 rows (with the one scale, a class at e^-20 kept some twelve bits, one at e^-30 none).
    Split16 z{}, zc{};
    if (gx) z = split16_at(hz.p, n, vc);
    if (gw) zc = split16_at(hc.p, n, vc, Scale16::Column);
    z.inv = nullptr;
    Product16 f{};
    f.a = Op16{sx, false}; f.b = Op16{wc, false}; f.M = n; f.N = vc; f.K = d;
    f.target = tgt; f.col0 = v0; f.lse = lse; f.grad = z; f.grad_by_column = zc;
    VB_TRY(launch_gemm16(Tile16::LossGrad, &f, 1, counters));
    Product16 b[2] = {};
    int nb = 0;
    if (gx) {
      Product16& q = b[nb++];
      q.a = Op16{z, false}; q.b = Op16{wc, true}; q.M = n; q.N = d; q.K = vc;
      q.out = gx; q.ldo = d; q.add = v0 > 0; q.alpha = coef; q.alpha_host = 1.0f / 16384.0f;
    }
    if (gw) {
      Product16& q = b[nb++];
      q.a = Op16{zc, true}; q.b = Op16{sk, true}; q.M = vc; q.N = d; q.K = n;
      q.out = gw + v0 * d; q.ldo = d; q.alpha = coef; q.alpha_host = 1.0f / 16384.0f;
    }
    if (nb) VB_TRY(launch_gemm16(Tile16::Store, b, nb, counters + 1));
  }
  return VB_OK;
}

}  // namespace vb
