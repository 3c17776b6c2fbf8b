// Matrix products on half-precision pairs, three tcgen05.mma kind::f16 products per f32-accurate one.
//
//   out[m, n] = sum over 128-wide runs of k of 2^-(eA + eB) (lo hi' + hi lo' + hi hi')[run]
//
// Persistent, one CTA per SM, 320 threads: warp 0 fetches operand tiles by TMA (no multicast), warp 1 issues the MMAs from one
// thread, warps 2-9 add the finished runs to registers (thread = one row x 128 of the tile's 256 columns) and store the tile.  Stage
// = 64 k values of a 128 x 256 tile, both planes: 96 KB, two stages.  A run of k is one accumulator of 256 tensor-memory columns, two of them
// in flight, so the adding warps work on one while the next is formed; a tile's epilogue hides under the next tile's first
// runs the same way.  Both operands may lie K-major or MN-major in memory: half precision takes either through the same
// 128-byte swizzle, so no operand is ever laid out twice.
#include "gemm16.h"
#include "split16.cuh"

namespace vb {
namespace {
using namespace tc;

constexpr int kThreads = 320, kBM = 128, kBN = 256, kBK = 64, kStages = 2;
constexpr int kAPlane = kBM * kBK * 2, kBPlane = kBN * kBK * 2;               // 16 KB, 32 KB
constexpr int kStage = 2 * kAPlane + 2 * kBPlane;
constexpr int kPitch = 33;                                                    // words of a staged row of 32
constexpr int kStaging = 32 * kPitch * 4;
constexpr int kSmem = 1024 + kStages * kStage + 8 * kStaging + 128;
constexpr float kGradScale = 16384.0f;

// ---- splitting ------------------------------------------------------------------------------------------------------------------
struct SplitDev { const float* x; __half* planes; float* inv; i64 rows, cols, ld, plane; int cb, blocks; bool vec; };
__global__ void __launch_bounds__(256) k_split16(SplitDev j0, SplitDev j1) {
  __shared__ float red[8];
  const bool second = (int)blockIdx.x >= j0.blocks;
  const SplitDev& j = second ? j1 : j0;
  const int blk = second ? (int)blockIdx.x - j0.blocks : (int)blockIdx.x;
  const int rb = blk / j.cb, cbi = blk - rb * j.cb;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const i64 c0 = (i64)cbi * 128 + lane * 4;
  float4 v[16];
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const i64 r = (i64)rb * 128 + i * 8 + wid;
    v[i] = make_float4(0, 0, 0, 0);
    if (r < j.rows && c0 < j.cols) {
      const float* p = j.x + r * j.cols + c0;
      if (j.vec) v[i] = *reinterpret_cast<const float4*>(p);
      else { v[i].x = p[0]; if (c0 + 1 < j.cols) v[i].y = p[1]; if (c0 + 2 < j.cols) v[i].z = p[2]; if (c0 + 3 < j.cols) v[i].w = p[3]; }
    }
    m = fmaxf(m, fmaxf(fmaxf(finite_abs(v[i].x), finite_abs(v[i].y)), fmaxf(finite_abs(v[i].z), finite_abs(v[i].w))));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[wid] = m;
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, red[i]);
  float inv;
  const float s = block_scale(m, &inv);
  if (threadIdx.x == 0) j.inv[blk] = inv;
  if (c0 >= j.ld) return;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const i64 r = (i64)rb * 128 + i * 8 + wid;
    if (r >= j.rows) continue;
    uint2 h, l;
    split2(v[i].x * s, v[i].y * s, &h.x, &l.x);
    split2(v[i].z * s, v[i].w * s, &h.y, &l.y);
    *reinterpret_cast<uint2*>(j.planes + r * j.ld + c0) = h;
    *reinterpret_cast<uint2*>(j.planes + j.plane + r * j.ld + c0) = l;
  }
}

// ---- the product ----------------------------------------------------------------------------------------------------------------
struct OperandDev { CUtensorMap map; const float* inv; int inv_ld; int mn; };
struct ProblemDev {
  OperandDev a, b;
  int M, N, K, tiles_m, tiles;
  float* out; i64 ldo; int add;
  const float* alpha; float alpha_host;
};
struct Params {
  ProblemDev prob[2];
  const int* target; int col0; float2* stats; float* target_value; const float* lse;
  __half* grad; i64 grad_ld, grad_plane;
  int* err;
};
enum { B_FULL = 0, B_EMPTY = B_FULL + kStages, B_RUN = B_EMPTY + kStages, B_RUNFREE = B_RUN + 2, B_COUNT = B_RUNFREE + 2 };

__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

template <Tile16 WHAT>
__global__ void __launch_bounds__(kThreads, 1) k_gemm16(const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint32_t* staging = (uint32_t*)(smem + kStages * kStage);
  uint64_t* bars = (uint64_t*)((uint8_t*)staging + 8 * kStaging);
  uint32_t* tmem_slot = (uint32_t*)(bars + B_COUNT);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) { mbar_init(&bars[B_FULL + i], 1); mbar_init(&bars[B_EMPTY + i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&bars[B_RUN + i], 1); mbar_init(&bars[B_RUNFREE + i], 8); }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int tiles = p.prob[0].tiles + p.prob[1].tiles;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const ProblemDev& q = t < p.prob[0].tiles ? p.prob[0] : p.prob[1];
        const int lt = t < p.prob[0].tiles ? t : t - p.prob[0].tiles;
        const int m0 = (lt % q.tiles_m) * kBM, n0 = (lt / q.tiles_m) * kBN;
        for (int k0 = 0; k0 < q.K; k0 += kBK, ++it) {
          const int st = it % kStages;
          if (it >= kStages && !mbar_wait(&bars[B_EMPTY + st], ((it / kStages) - 1) & 1, abort_flag)) { ok = false; break; }
          uint64_t* full = &bars[B_FULL + st];
          uint8_t* base = smem + st * kStage;
          mbar_arrive_expect_tx(full, kStage);
          for (int pl = 0; pl < 2; ++pl) {
            uint8_t* a = base + pl * kAPlane;
            uint8_t* b = base + 2 * kAPlane + pl * kBPlane;
            if (!q.a.mn) tma_load_3d(a, &q.a.map, full, k0, m0, pl);
            else for (int i = 0; i < kBM / 64; ++i) tma_load_3d(a + i * 8192, &q.a.map, full, m0 + 64 * i, k0, pl);
            if (!q.b.mn) tma_load_3d(b, &q.b.map, full, k0, n0, pl);
            else for (int i = 0; i < kBN / 64; ++i) tma_load_3d(b + i * 8192, &q.b.map, full, n0 + 64 * i, k0, pl);
          }
        }
      }
      if (*abort_flag) {      // give copies already issued a bounded time to land before the CTA exits
        for (int i = 0; i < kStages; ++i) {
          uint32_t addr = smem_u32(&bars[B_FULL + i]), done = 0;
          for (uint32_t n = 0; n < (1u << 14) && !done; ++n)
            asm volatile("{\n\t.reg .pred q;\n\tmbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(done) : "r"(addr), "r"(0u) : "memory");
        }
      }
    }
  } else if (warp == 1) {
    const uint32_t leader = elect_leader();
    uint32_t it = 0, run = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const ProblemDev& q = t < p.prob[0].tiles ? p.prob[0] : p.prob[1];
      const uint32_t idesc = idesc16(kBM, kBN, q.a.mn, q.b.mn);
      const uint64_t step_a = (q.a.mn ? 2048 : 32) >> 4, step_b = (q.b.mn ? 2048 : 32) >> 4;
      for (int k0 = 0; k0 < q.K && ok; k0 += 2 * kBK, ++run) {
        const int acc = run & 1;
        if (run >= 2 && !warp_wait(&bars[B_RUNFREE + acc], ((run >> 1) - 1) & 1, abort_flag)) { ok = false; break; }
        const uint32_t d = tmem + acc * kBN;
        uint32_t on = 0;
        for (int k = k0; k < q.K && k < k0 + 2 * kBK; k += kBK, ++it) {
          const int st = it % kStages;
          if (!warp_wait(&bars[B_FULL + st], (it / kStages) & 1, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint32_t base = smem_u32(smem + st * kStage);
          const uint64_t ah = desc16(base, 8192), al = desc16(base + kAPlane, 8192);
          const uint64_t bh = desc16(base + 2 * kAPlane, 8192), bl = desc16(base + 2 * kAPlane + kBPlane, 8192);
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            mma_f16(leader, d, al + s * step_a, bh + s * step_b, idesc, on);
            on = 1;
            mma_f16(leader, d, ah + s * step_a, bl + s * step_b, idesc, 1);
          }
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_f16(leader, d, ah + s * step_a, bh + s * step_b, idesc, 1);
          commit_by(leader, &bars[B_EMPTY + st]);
        }
        if (ok) commit_by(leader, &bars[B_RUN + acc]);
      }
    }
  } else {
    const int w = warp - 2, quarter = warp & 3, half = w >> 2;
    const int row = quarter * 32 + lane;
    uint32_t* stg = staging + w * 32 * kPitch;
    uint32_t run = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const ProblemDev& q = t < p.prob[0].tiles ? p.prob[0] : p.prob[1];
      const int lt = t < p.prob[0].tiles ? t : t - p.prob[0].tiles;
      const int tm = lt % q.tiles_m, tn = lt / q.tiles_m;
      const int m = tm * kBM + row, n0 = tn * kBN + half * 128;
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
      const int nb = n0 < q.N ? tn * 2 + half : tn * 2;          // (a half tile past the last column has no scale of its own)
      for (int kb = 0; kb * 128 < q.K; ++kb, ++run) {
        float s = 1.0f;
        if (q.a.inv) s = q.a.mn ? q.a.inv[(i64)kb * q.a.inv_ld + tm] : q.a.inv[(i64)tm * q.a.inv_ld + kb];
        if (q.b.inv) s *= q.b.mn ? q.b.inv[(i64)kb * q.b.inv_ld + nb] : q.b.inv[(i64)nb * q.b.inv_ld + kb];
        if (!mbar_wait(&bars[B_RUN + (run & 1)], (run >> 1) & 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint32_t src = tmem + (run & 1) * kBN + half * 128 + ((uint32_t)(quarter * 32) << 16);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          tmem_ld32(src + c * 32, v);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[c * 32 + i] = fmaf(__uint_as_float(v[i]), s, acc[c * 32 + i]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[B_RUNFREE + (run & 1)]);
      }
      if (!ok) break;
      if constexpr (WHAT == Tile16::Store) {
        const float alpha = (q.alpha ? *q.alpha : 1.0f) * q.alpha_host;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 32; ++i) stg[lane * kPitch + i] = __float_as_uint(acc[c * 32 + i] * alpha);
          __syncwarp();
          const int col = n0 + c * 32 + lane;
          const int mrow = tm * kBM + quarter * 32;
          if (col < q.N) {
            float* o = q.out + (i64)mrow * q.ldo + col;
            const int live = q.M - mrow < 32 ? q.M - mrow : 32;
            if (q.add) for (int r = 0; r < live; ++r) o[(i64)r * q.ldo] += __uint_as_float(stg[r * kPitch + lane]);
            else for (int r = 0; r < live; ++r) o[(i64)r * q.ldo] = __uint_as_float(stg[r * kPitch + lane]);
          }
        }
      } else if constexpr (WHAT == Tile16::RowStats) {
        const int live = q.N - n0;                     // columns of this half that exist
        if (m < q.M && live > 0) {
          const int tgt = p.target[m] - p.col0 - n0;
          constexpr float kL2e = 1.4426950408889634f;
          float mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < 128; ++i) {
            if (i == tgt && i < live) p.target_value[m] = acc[i];
            if (i >= live) acc[i] = -INFINITY;
            mx = fmaxf(mx, acc[i]);
          }
          float sum = 0.0f;
          if (mx > -INFINITY) {
            const float off = -mx * kL2e;
#pragma unroll
            for (int i = 0; i < 128; ++i) sum += exp2_fast(fmaf(acc[i], kL2e, off));
          }
          p.stats[(i64)(tn * 2 + half) * q.M + m] = make_float2(mx, sum);
        }
      } else {
        const int tgt0 = m < q.M ? p.target[m] : kNoTarget;
        const int tgt = tgt0 - p.col0 - n0;
        constexpr float kL2e = 1.4426950408889634f;
        const float off = m < q.M ? -p.lse[m] * kL2e + 14.0f : 0.0f;     // 2^14 rides in the exponent
        const bool live_row = tgt0 != kNoTarget;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float d[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = c * 32 + i + e;
              d[e] = exp2_fast(fmaf(acc[j], kL2e, off)) - (j == tgt ? kGradScale : 0.0f);
              if (!live_row || n0 + j >= q.N) d[e] = 0.0f;
            }
            uint32_t h, l;
            split2(d[0], d[1], &h, &l);
            stg[lane * kPitch + i / 2] = h;
            stg[lane * kPitch + 16 + i / 2] = l;
          }
          __syncwarp();
          const int col = n0 + c * 32, mrow = tm * kBM + quarter * 32;
          const int live = q.M - mrow < 32 ? q.M - mrow : 32;
          if (col + 2 * (lane & 15) < p.grad_ld) {
            uint32_t* o = reinterpret_cast<uint32_t*>(p.grad + (lane < 16 ? 0 : p.grad_plane) + (i64)mrow * p.grad_ld + col) + (lane & 15);
            for (int r = 0; r < live; ++r) o[(i64)r * (p.grad_ld / 2)] = stg[r * kPitch + lane];
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.err, ERRBIT_WAIT_TIMEOUT);
}

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

int make_operand(const Op16& o, int box_mn, OperandDev* d) {
  if (!encode_fn()) return set_error(VB_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  cuuint64_t dims[3] = {(cuuint64_t)o.s.cols, (cuuint64_t)o.s.rows, 2}, strides[2] = {(cuuint64_t)o.s.ld * 2, (cuuint64_t)o.s.plane * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)(o.mn ? 64 : box_mn), 1}, estr[3] = {1, 1, 1};
  CUresult r = encode_fn()(&d->map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, o.s.planes, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(VB_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
  d->inv = o.s.inv; d->inv_ld = (int)o.s.inv_ld; d->mn = o.mn;
  return VB_OK;
}

template <Tile16 WHAT>
int launch(const Params& p, int ctas) {
  static bool ready = false;
  if (!ready) {
    VB_CUDA(cudaFuncSetAttribute(k_gemm16<WHAT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    ready = true;
  }
  k_gemm16<WHAT><<<ctas, kThreads, kSmem, ctx().stream>>>(p);
  VB_LAUNCH_CHECK();
  return VB_OK;
}

}  // namespace

Split16 split16_at(void* mem, i64 rows, i64 cols) {
  Split16 s{};
  s.rows = rows; s.cols = cols; s.ld = (cols + 7) / 8 * 8; s.plane = rows * s.ld; s.inv_ld = (cols + 127) / 128;
  s.planes = mem;
  s.inv = reinterpret_cast<float*>(static_cast<uint8_t*>(mem) + ((size_t)(2 * s.plane) * 2 + 15) / 16 * 16);
  return s;
}

int launch_split16(const SplitJob* jobs, int n) {
  SplitDev d[2] = {};
  double bytes = 0.0;
  for (int i = 0; i < n; ++i) {
    const Split16& s = jobs[i].to;
    const i64 blocks = ((s.rows + 127) / 128) * s.inv_ld;
    if (blocks > 0x3fffffff) return set_error(VB_ERR_UNSUPPORTED, "matrix too large to split");
    d[i] = SplitDev{jobs[i].x, (__half*)s.planes, s.inv, s.rows, s.cols, s.ld, s.plane, (int)s.inv_ld, (int)blocks,
                    s.cols % 4 == 0 && (reinterpret_cast<uintptr_t>(jobs[i].x) & 15) == 0};
    bytes += 8.0 * (double)s.rows * (double)s.cols;
  }
  const int blocks = d[0].blocks + d[1].blocks;
  if (blocks == 0) return VB_OK;
  ProfScope prof("split16", bytes);
  k_split16<<<blocks, 256, 0, ctx().stream>>>(d[0], d[1]);
  VB_LAUNCH_CHECK();
  return VB_OK;
}

int launch_gemm16(Tile16 what, const Product16* products, int n) {
  Params p{};
  double flops = 0.0;
  for (int i = 0; i < n; ++i) {
    const Product16& g = products[i];
    ProblemDev& q = p.prob[i];
    const i64 tm = (g.M + kBM - 1) / kBM, tn = (g.N + kBN - 1) / kBN;
    if (g.M > 0x7fffff00 || g.N > 0x7fffff00 || g.K > 0x7fffff00 || tm * tn > 0x3fffffff) return set_error(VB_ERR_UNSUPPORTED, "product too large");
    q.M = (int)g.M; q.N = (int)g.N; q.K = (int)g.K; q.tiles_m = (int)tm; q.tiles = (int)(tm * tn);
    VB_TRY(make_operand(g.a, kBM, &q.a));
    VB_TRY(make_operand(g.b, kBN, &q.b));
    q.out = g.out; q.ldo = g.ldo; q.add = g.add; q.alpha = g.alpha; q.alpha_host = g.alpha_host;
    flops += 2.0 * (double)g.M * (double)g.N * (double)g.K;
  }
  p.target = products[0].target; p.col0 = (int)products[0].col0; p.stats = products[0].stats; p.target_value = products[0].target_value; p.lse = products[0].lse;
  p.grad = (__half*)products[0].grad.planes; p.grad_ld = products[0].grad.ld; p.grad_plane = products[0].grad.plane;
  p.err = ctx().d_err;
  const int tiles = p.prob[0].tiles + p.prob[1].tiles;
  if (tiles == 0) return VB_OK;
  ProfScope prof("gemm16", flops);
  const int ctas = tiles < ctx().sm_count ? tiles : ctx().sm_count;
  switch (what) {
    case Tile16::Store: return launch<Tile16::Store>(p, ctas);
    case Tile16::RowStats: return launch<Tile16::RowStats>(p, ctas);
    default: return launch<Tile16::LossGrad>(p, ctas);
  }
}

}  // namespace vb
