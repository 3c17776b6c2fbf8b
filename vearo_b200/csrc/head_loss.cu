// The vocabulary projection with its softmax cross entropy, forward and backward, without the logits in memory.
//
//   z = x W^T,  lse_n = log sum_v exp z_nv,  loss = mean over rows with a target of (lse_n - z_n,target)
//   dz = (exp(z - lse) - onehot) g / count,   dx = dz W,   dW = dz^T x
//
// Forward: one product whose tiles leave (max, sum of exp) for each row and 128 columns, 8 bytes where the logits would be 512, and
// the target's logit; a second kernel joins the pairs of a row.  Backward: pieces of the vocabulary; a piece's logits are formed
// again and leave the tensor core as dz in half-precision planes (the operand of the two products that follow), and one launch
// adds the piece to dx and writes its rows of dW.  Tensor-bound: 2 N V D and 6 N V D operations, three instructions each (gemm16.cu).
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
// lse and the row's loss from its pairs: 32 rows x 32 pair lanes a CTA, pairs joined in a fixed order; the CTA that ends last takes the
// mean over the rows, in a fixed order too.  (As a kernel of its own the mean cost 3 us of 28 at 512 x 256 x 8192.)
__global__ void __launch_bounds__(1024) k_join_stats(const float2* __restrict__ stats, const float* __restrict__ target_value, const int* __restrict__ target,
                                                     float* __restrict__ lse, float* nll, float* __restrict__ loss, int* ticket, int n, int pairs) {
  __shared__ float sm[32][33], ss[32][33];
  __shared__ bool last;
  wait_for_last_kernel();
  const int row = blockIdx.x * 32 + threadIdx.x;
  float m = -INFINITY, s = 0.0f;
  if (row < n) {
    for (int i = threadIdx.y; i < pairs; i += 32) {
      const float2 a = stats[(i64)i * n + row];
      if (a.x > m) { s = s * expf(m - a.x) + a.y; m = a.x; }
      else if (a.y != 0.0f) s += a.y * expf(a.x - m);          // (a pair of NaN sum keeps it)
    }
  }
  sm[threadIdx.y][threadIdx.x] = m; ss[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  // transposed: a warp joins the 32 partial pairs of one row
  m = sm[threadIdx.x][threadIdx.y]; s = ss[threadIdx.x][threadIdx.y];
  float top = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  s = top > -INFINITY && m > -INFINITY ? s * expf(m - top) : s;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int r = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && r < n) {
    const float l = top + logf(s);
    lse[r] = l;
    nll[r] = target[r] == kNoTarget ? 0.0f : l - target_value[r];
    __threadfence();
  }
  __syncthreads();
  const int tid = threadIdx.y * 32 + threadIdx.x;
  if (tid == 0) { last = atomicAdd(ticket, 1) == (int)gridDim.x - 1; __threadfence(); }
  __syncthreads();
  if (!last) return;
  float* sums = &sm[0][0];
  int* counts = (int*)&ss[0][0];
  float t = 0.0f;
  int live = 0;
  for (int i = tid; i < n; i += 1024) { t += __ldcg(nll + i); live += target[i] != kNoTarget; }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { t += __shfl_xor_sync(0xffffffffu, t, o); live += __shfl_xor_sync(0xffffffffu, live, o); }
  if (threadIdx.x == 0) { sums[threadIdx.y] = t; counts[threadIdx.y] = live; }
  __syncthreads();
  if (tid == 0) {
    float all = 0.0f;
    int c = 0;
    for (int i = 0; i < 32; ++i) { all += sums[i]; c += counts[i]; }
    *loss = c > 0 ? all / (float)c : 0.0f;
  }
}

// Half-precision planes of a piece of dz: at most half a gigabyte of them at a time.
constexpr i64 kPieceBytes = (i64)512 << 20;

}  // namespace

int launch_head_loss(const float* x, const float* w, const float* targets, i64 ignore, float* loss, float* lse, i64 n, i64 d, i64 v) {
  Temp hx, hw, hs, hr;
  const i64 pairs = (v + 127) / 128;
  VB_TRY(scratch_alloc(split16_bytes(n, d, true), &hx.p));
  VB_TRY(scratch_alloc(split16_bytes(v, d), &hw.p));
  VB_TRY(scratch_alloc((size_t)(pairs * n) * sizeof(float2), &hs.p));
  VB_TRY(scratch_alloc((size_t)n * 12 + 8, &hr.p));
  float* nll = (float*)hr.p; float* tv = nll + n; int* tgt = (int*)(tv + n); int* counters = tgt + n;
  const Split16 sx = split16_at(hx.p, n, d, true), sw = split16_at(hw.p, v, d);
  const SplitJob jobs[2] = {{x, sx}, {w, sw}};
  const TargetRows rows{targets, ignore, v, tgt, counters, 2};
  VB_TRY(launch_split16(jobs, 2, &rows));
  Product16 g{};
  g.a = Op16{sx, false}; g.b = Op16{sw, false}; g.M = n; g.N = v; g.K = d;
  g.target = tgt; g.stats = (float2*)hs.p; g.target_value = tv;
  VB_TRY(launch_gemm16(Tile16::RowStats, &g, 1, counters));
  return launch_early(k_join_stats, dim3((unsigned)((n + 31) / 32)), dim3(32, 32), 0, (const float2*)hs.p, tv, tgt, lse, nll, loss, counters + 1, (int)n, (int)pairs);
}

int launch_head_loss_backward(const float* x, const float* w, const float* targets, i64 ignore, const float* lse, const float* g, float* gx, float* gw,
                              i64 n, i64 d, i64 v) {
  Temp hx, hk, hw, hz, ht;
  i64 piece = kPieceBytes / (4 * n) / 256 * 256;
  if (piece < 256) piece = 256;
  const i64 pieces = (v + piece - 1) / piece;
  piece = ((v + pieces - 1) / pieces + 255) / 256 * 256;
  if (piece > v) piece = v;
  VB_TRY(scratch_alloc(split16_bytes(n, d, true), &hx.p));
  if (gw) VB_TRY(scratch_alloc(split16_bytes(n, d), &hk.p));
  VB_TRY(scratch_alloc(split16_bytes(v, d), &hw.p));
  VB_TRY(scratch_alloc(split16_bytes(n, piece), &hz.p));
  VB_TRY(scratch_alloc((size_t)(n + 2 * pieces) * 4 + 16, &ht.p));
  float* coef = (float*)ht.p; int* tgt = (int*)(coef + 4); int* counters = tgt + n;
  const Split16 sx = split16_at(hx.p, n, d, true), sw = split16_at(hw.p, v, d);      // x for the logits, where its rows are the product's,
  const Split16 sk = gw ? split16_at(hk.p, n, d) : sx;                                  // and for dW, which sums over them
  k_targets<<<1, 1024, 0, ctx().stream>>>(targets, n, ignore, v, tgt, g, coef, counters, (int)(2 * pieces), ctx().d_err);
  VB_LAUNCH_CHECK();
  const SplitJob jobs[3] = {{w, sw}, {x, sx, tgt}, {x, sk, tgt}};        // (rows that are left out may hold anything: they must not reach dW)
  VB_TRY(launch_split16(jobs, gw ? 3 : 2));
  for (i64 v0 = 0; v0 < v; v0 += piece, counters += 2) {
    const i64 vc = v - v0 < piece ? v - v0 : piece;
    Split16 wc = sw;                                     // this piece's rows of W
    wc.planes = (uint16_t*)sw.planes + v0 * sw.ld; wc.inv = sw.inv + v0 / 128 * sw.inv_ld; wc.rows = vc;
    Split16 z = split16_at(hz.p, n, vc);
    Product16 f{};
    f.a = Op16{sx, false}; f.b = Op16{wc, false}; f.M = n; f.N = vc; f.K = d;
    f.target = tgt; f.col0 = v0; f.lse = lse; f.grad = z;
    VB_TRY(launch_gemm16(Tile16::LossGrad, &f, 1, counters));
    z.inv = nullptr;
    Product16 b[2] = {};
    int nb = 0;
    if (gx) {
      Product16& q = b[nb++];
      q.a = Op16{z, false}; q.b = Op16{wc, true}; q.M = n; q.N = d; q.K = vc;
      q.out = gx; q.ldo = d; q.add = v0 > 0; q.alpha = coef; q.alpha_host = 1.0f / 16384.0f;
    }
    if (gw) {
      Product16& q = b[nb++];
      q.a = Op16{z, true}; q.b = Op16{sk, true}; q.M = vc; q.N = d; q.K = n;
      q.out = gw + v0 * d; q.ldo = d; q.alpha = coef; q.alpha_host = 1.0f / 16384.0f;
    }
    if (nb) VB_TRY(launch_gemm16(Tile16::Store, b, nb, counters + 1));
  }
  return VB_OK;
}

}  // namespace vb
