// Matrix products on half-precision pairs, three tcgen05.mma kind::f16 products per f32-accurate one.
//
//   out[m, n] = sum over 128-wide runs of k of 2^-(eA + eB) (lo hi' + hi lo' + hi hi')[run]
//
// Persistent, one CTA per SM, 320 threads: warp 0 takes tiles from a counter and fetches their operands by TMA (no multicast), warp 1
// issues the MMAs, warps 2-9 add the finished runs to registers (thread = one row x 128 of the tile's 256 columns) and store the
// tile, 32 x 32 blocks at a time, by TMA.  Stage
// = 64 k values of a 128 x 256 tile, both planes: 96 KB, two stages.  A run of k is one accumulator of 256 tensor-memory columns, two of them
// in flight, so the adding warps work on one while the next is formed; a tile's epilogue hides under the next tile's first
// runs the same way.  Both operands may lie K-major or MN-major in memory: half precision takes either through the same
// 128-byte swizzle, so no operand is ever laid out twice.  Tensor-bound under the power limit: 8192 x 50304 x 768 (RowStats) 1258 us, 503 TFLOP/s
// useful, 1510 issued at 1.53 GHz; dx and dW of 4097 rows, 1024 x 25152 columns (Store) 989 us, 427 useful.  k_split16 is HBM-bound: 4097 x 1024 and
// 50304 x 1024 in 81 us, 5.5 TB/s read and written.
#include "gemm16.h"
#include "split16.cuh"

namespace vb {
namespace {
using namespace tc;

constexpr int kThreads = 320, kBM = 128, kBN = 256, kBK = 64, kStages = 2, kEpiWarps = 8;
constexpr int kAPlane = kBM * kBK * 2, kBPlane = kBN * kBK * 2;               // 16 KB, 32 KB
constexpr int kStage = 2 * kAPlane + 2 * kBPlane;
constexpr int kStaging = 4096;                                                // a warp's 32 x 32 block: f32, or both planes of halves
constexpr int kExponents = kEpiWarps * 128;                                   // a warp's bytes for 128 columns
constexpr int kSmem = 1024 + kStages * kStage + kEpiWarps * kStaging + kExponents + 256;
static_assert(kSmem <= 227 * 1024, "shared memory");
constexpr float kGradScale = 16384.0f;

// ---- splitting ------------------------------------------------------------------------------------------------------------------
struct SplitDev { const float* x; const int* keep; __half* planes; float* inv; i64 rows, cols, ld, plane, inv_ld; int cb, blocks; bool vec, by_row; };      // (by_row: a scale for 128 columns of a row)
struct SplitJobs { SplitDev job[3]; TargetRows rows; int* err; };
__global__ void __launch_bounds__(256) k_split16(const __grid_constant__ SplitJobs jobs) {
  __shared__ float red[8];
  int blk = blockIdx.x, which = 0;
  while (blk >= jobs.job[which].blocks) blk -= jobs.job[which++].blocks;
  const SplitDev& j = jobs.job[which];
  const int rb = blk / j.cb, cbi = blk - rb * j.cb;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const i64 c0 = (i64)cbi * 128 + lane * 4;
  if (jobs.rows.targets && which == 0 && cbi == 0) {
    const i64 r = (i64)rb * 128 + threadIdx.x;
    if (threadIdx.x < 128 && r < j.rows) jobs.rows.out[r] = read_target(jobs.rows.targets[r], jobs.rows.ignore, jobs.rows.vocab, jobs.err);
    if (rb == 0 && threadIdx.x < jobs.rows.n_zero) jobs.rows.zero[threadIdx.x] = 0;
  }
  float4 v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {      // (a warp has whole rows of the block)
    const i64 r = (i64)rb * 128 + i * 8 + wid;
    v[i] = make_float4(0, 0, 0, 0);
    if (r < j.rows && c0 < j.cols && (!j.keep || j.keep[r] != kNoTarget)) {
      const float* p = j.x + r * j.cols + c0;
      if (j.vec) v[i] = *reinterpret_cast<const float4*>(p);
      else { v[i].x = p[0]; if (c0 + 1 < j.cols) v[i].y = p[1]; if (c0 + 2 < j.cols) v[i].z = p[2]; if (c0 + 3 < j.cols) v[i].w = p[3]; }
    }
  }
  float m = 0.0f, s = 1.0f;
  if (!j.by_row) {
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, fmaxf(fmaxf(finite_abs(v[i].x), finite_abs(v[i].y)), fmaxf(finite_abs(v[i].z), finite_abs(v[i].w))));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red[wid] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fmaxf(m, red[i]);
    float inv;
    s = block_scale(m, &inv);
    if (threadIdx.x == 0) j.inv[rb * j.inv_ld + cbi] = inv;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const i64 r = (i64)rb * 128 + i * 8 + wid;
    if (j.by_row) {
      m = fmaxf(fmaxf(finite_abs(v[i].x), finite_abs(v[i].y)), fmaxf(finite_abs(v[i].z), finite_abs(v[i].w)));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      float inv;
      s = block_scale(m, &inv);
      if (lane == 0 && r < j.rows) j.inv[cbi * j.inv_ld + r] = inv;
    }
    if (r >= j.rows || c0 >= j.ld) continue;
    uint2 h, l;
    split2(v[i].x * s, v[i].y * s, &h.x, &l.x);
    split2(v[i].z * s, v[i].w * s, &h.y, &l.y);
    *reinterpret_cast<uint2*>(j.planes + r * j.ld + c0) = h;
    *reinterpret_cast<uint2*>(j.planes + j.plane + r * j.ld + c0) = l;
  }
}

// ---- the product ----------------------------------------------------------------------------------------------------------------
struct OperandDev { CUtensorMap map; const float* inv; i64 inv_ld; int mn, by_m; };      // by_m: inv is [128 k][m]
struct ProblemDev {
  OperandDev a, b;
  CUtensorMap out_map;                       // Store: f32, where `by_copy`; LossGrad: the planes of grad
  int M, N, K, tiles_m, tiles;               // tiles: of all parts
  int parts, part_k;                         // Store: the sum over k in parts of part_k steps, each a tile of its own in plane `part` of the result
  float* out; i64 ldo; int add, by_copy;
  const float* alpha; float alpha_host;
};
// A tile of a problem: rows, columns, steps of k, part.
struct TileAt { int tm, tn, k0, k1, part; };
__device__ __forceinline__ TileAt tile_at(const ProblemDev& q, int t) {
  TileAt a;
  a.part = t % q.parts; t /= q.parts;
  a.tm = t % q.tiles_m; a.tn = t / q.tiles_m;
  a.k0 = a.part * q.part_k; a.k1 = min(q.K, a.k0 + q.part_k);
  return a;
}
struct Params {
  ProblemDev prob[2];
  const int* target; int col0; float2* stats; float* target_value; const float* lse;
  CUtensorMap col_map; float* col_inv; i64 col_inv_ld; int with_rows, with_cols;      // LossGrad: the planes of grad_by_column and their scales
  int* counter;                              // 0: tiles handed out beyond the first of every CTA
  int* err;
};
enum { B_FULL = 0, B_EMPTY = B_FULL + kStages, B_RUN = B_EMPTY + kStages, B_RUNFREE = B_RUN + 2, B_POST = B_RUNFREE + 2, B_TAKEN = B_POST + 2, B_COLS = B_TAKEN + 2, B_COLSREAD = B_COLS + 2, B_COUNT = B_COLSREAD + 2 };
static_assert(B_COUNT * 8 + 16 <= 256, "barriers");

// (asked for here, looked at when the copies of the tile in hand have been issued)
__device__ __forceinline__ int next_tile(int* counter) {
  int r;
  asm volatile("atom.global.add.s32 %0, [%1], 1;" : "=r"(r) : "l"(counter) : "memory");
  return r;
}
__device__ __forceinline__ void store_block(const CUtensorMap* map, const void* src, int c, int r, int plane) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(smem_u32(src)), "r"(c), "r"(r), "r"(plane) : "memory");
}
__device__ __forceinline__ void add_block(const CUtensorMap* map, const void* src, int c, int r, int plane) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(smem_u32(src)), "r"(c), "r"(r), "r"(plane) : "memory");
}
__device__ __forceinline__ void commit_blocks() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }

// A warp's 32 rows x 128 columns as half planes, 32 x 32 blocks through its staging: 16-byte pieces of a plane's 64-byte row, in the copy
// engine's 64-byte swizzle.  (Ordinary stores, of 64 bytes of a row from the staging or 32 a thread, took LossGrad of
// 4097 rows, 1024 x 25152 columns, then at 648 us with the butterfly below, to 780 and 688; it takes 609.)
__device__ __forceinline__ void store_planes(const CUtensorMap* map, uint8_t* stg, const float (&acc)[128], int n0, int row, int N, int M, int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (lane == 0) tma_store_wait_read();
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint4 h, l;
      split2_finite(acc[c * 32 + 8 * e], acc[c * 32 + 8 * e + 1], &h.x, &l.x);
      split2_finite(acc[c * 32 + 8 * e + 2], acc[c * 32 + 8 * e + 3], &h.y, &l.y);
      split2_finite(acc[c * 32 + 8 * e + 4], acc[c * 32 + 8 * e + 5], &h.z, &l.z);
      split2_finite(acc[c * 32 + 8 * e + 6], acc[c * 32 + 8 * e + 7], &h.w, &l.w);
      const int at = lane * 64 + ((e ^ ((lane >> 1) & 3)) << 4);
      *reinterpret_cast<uint4*>(stg + at) = h;
      *reinterpret_cast<uint4*>(stg + 2048 + at) = l;
    }
    fence_async_smem();
    __syncwarp();
    const int col = n0 + c * 32;
    if (lane == 0 && col < N && row < M) {
      store_block(map, stg, col, row, 0);
      store_block(map, stg + 2048, col, row, 1);
      commit_blocks();
    }
  }
}
// The largest magnitudes of columns 4 lane .. 4 lane + 3 among the warp's rows, as the upper seven bits of their exponents, a byte each (all ones:
// NaN or infinity).  Through the warp's staging, a row of bytes a lane: a butterfly of shuffles over pairs of columns, which take their turns with the
// operands' way through shared memory, cost 6200 cycles a tile, as did 128 reductions by redux.sync; so 1600.
__device__ __forceinline__ uint32_t largest_of_columns(const float (&acc)[128], uint8_t* stg, int lane) {
  if (lane == 0) tma_store_wait_read();
  __syncwarp();
  auto tops = [](const float* x) -> uint32_t {
    const uint32_t a = __byte_perm(__float_as_uint(x[0]), __float_as_uint(x[1]), 0x73), b = __byte_perm(__float_as_uint(x[2]), __float_as_uint(x[3]), 0x73);
    return __byte_perm(a, b, 0x5410) & 0x7f7f7f7fu;
  };
#pragma unroll
  for (int e = 0; e < 8; ++e)
    *reinterpret_cast<uint4*>(stg + lane * 128 + ((e ^ (lane & 7)) << 4)) = make_uint4(tops(acc + 16 * e), tops(acc + 16 * e + 4), tops(acc + 16 * e + 8), tops(acc + 16 * e + 12));
  __syncwarp();
  uint32_t even = 0, odd = 0;
#pragma unroll
  for (int r = 0; r < 32; ++r) {
    const uint32_t x = *reinterpret_cast<const uint32_t*>(stg + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
    even = __vmaxu2(even, x & 0x00ff00ffu); odd = __vmaxu2(odd, x & 0xff00ff00u);
  }
  __syncwarp();
  return even | odd;
}

template <Tile16 WHAT>
__global__ void __launch_bounds__(kThreads, 1) k_gemm16(const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* staging = smem + kStages * kStage;
  uint32_t* exponents = (uint32_t*)(staging + kEpiWarps * kStaging);      // [halves][quarters][32]: a byte for every column
  uint64_t* bars = (uint64_t*)(exponents + kExponents / 4);
  uint32_t* tmem_slot = (uint32_t*)(bars + B_COUNT);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  volatile int* posted = abort_flag + 1;       // [2] tiles handed to the other roles
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) { mbar_init(&bars[B_FULL + i], 1); mbar_init(&bars[B_EMPTY + i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&bars[B_RUN + i], 1); mbar_init(&bars[B_RUNFREE + i], kEpiWarps); mbar_init(&bars[B_POST + i], 1); mbar_init(&bars[B_TAKEN + i], 1 + kEpiWarps); mbar_init(&bars[B_COLS + i], 4); mbar_init(&bars[B_COLSREAD + i], 4); }
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
  if (WHAT == Tile16::RowStats) wait_for_last_kernel();
  const uint32_t tmem = *tmem_slot;
  const int tiles = p.prob[0].tiles + p.prob[1].tiles;
  // the i-th tile of the CTA for a whole warp; false where there are no more (or a wait ran out)
  auto take = [&](uint32_t i, int* t) -> bool {
    const bool ok = warp_wait(&bars[B_POST + (i & 1)], (i >> 1) & 1, abort_flag);
    *t = posted[i & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars[B_TAKEN + (i & 1)]);
    return ok && *t < tiles;
  };

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      int t = blockIdx.x, next = 0;
      for (uint32_t i = 0; ok; ++i, t = (int)gridDim.x + next) {
        if (!mbar_wait(&bars[B_TAKEN + (i & 1)], ((i >> 1) & 1) ^ 1, abort_flag)) break;
        posted[i & 1] = t;
        mbar_arrive(&bars[B_POST + (i & 1)]);
        if (t >= tiles) break;
        next = next_tile(p.counter);
        const ProblemDev& q = t < p.prob[0].tiles ? p.prob[0] : p.prob[1];
        const TileAt at = tile_at(q, t < p.prob[0].tiles ? t : t - p.prob[0].tiles);
        const int m0 = at.tm * kBM, n0 = at.tn * kBN;
        for (int k0 = at.k0; k0 < at.k1; k0 += kBK, ++it) {
          const int st = it % kStages;
          if (it >= kStages && !mbar_wait(&bars[B_EMPTY + st], ((it / kStages) - 1) & 1, abort_flag)) { ok = false; break; }
          uint64_t* full = &bars[B_FULL + st];
          uint8_t* base = smem + st * kStage;
          mbar_arrive_expect_tx(full, kStage);
          for (int pl = 0; pl < 2; ++pl) {
            uint8_t* a = base + pl * kAPlane;
            uint8_t* b = base + 2 * kAPlane + pl * kBPlane;
            if (!q.a.mn) tma_load_3d(a, &q.a.map, full, k0, m0, pl);
            else for (int x = 0; x < kBM / 64; ++x) tma_load_3d(a + x * 8192, &q.a.map, full, m0 + 64 * x, k0, pl);
            if (!q.b.mn) tma_load_3d(b, &q.b.map, full, k0, n0, pl);
            else for (int x = 0; x < kBN / 64; ++x) tma_load_3d(b + x * 8192, &q.b.map, full, n0 + 64 * x, k0, pl);
          }
        }
      }
      if (*abort_flag) let_land(&bars[B_FULL], kStages);
    }
  } else if (warp == 1) {
    const uint32_t leader = elect_leader();
    uint32_t it = 0, run = 0;
    bool ok = true;
    int t;
    for (uint32_t i = 0; ok && take(i, &t); ++i) {
      const ProblemDev& q = t < p.prob[0].tiles ? p.prob[0] : p.prob[1];
      const uint32_t idesc = idesc16(kBM, kBN, q.a.mn, q.b.mn);
      const uint64_t step_a = (q.a.mn ? 2048 : 32) >> 4, step_b = (q.b.mn ? 2048 : 32) >> 4;
      const TileAt at = tile_at(q, t < p.prob[0].tiles ? t : t - p.prob[0].tiles);
      for (int k0 = at.k0; k0 < at.k1 && ok; k0 += 2 * kBK, ++run) {
        const int acc = run & 1;
        if (run >= 2 && !warp_wait(&bars[B_RUNFREE + acc], ((run >> 1) - 1) & 1, abort_flag)) { ok = false; break; }
        const uint32_t d = tmem + acc * kBN;
        uint32_t on = 0;
        for (int k = k0; k < at.k1 && k < k0 + 2 * kBK; k += kBK, ++it) {
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
    uint8_t* stg = staging + w * kStaging;
    uint32_t run = 0;
    bool ok = true;
    int t;
    for (uint32_t i = 0; ok && take(i, &t); ++i) {
      const ProblemDev& q = t < p.prob[0].tiles ? p.prob[0] : p.prob[1];
      const TileAt at = tile_at(q, t < p.prob[0].tiles ? t : t - p.prob[0].tiles);
      const int tm = at.tm, tn = at.tn;
      const int m = tm * kBM + row, n0 = tn * kBN + half * 128;
      int target = kNoTarget;
      float off = 0.0f;
      if (WHAT != Tile16::Store && m < q.M) {
        target = p.target[m];
        if (WHAT == Tile16::LossGrad) off = p.lse[m];
      }
      float acc[128];
#pragma unroll
      for (int c = 0; c < 128; ++c) acc[c] = 0.0f;
      const int nb = n0 < q.N ? tn * 2 + half : tn * 2;          // (a half tile past the last column has no scale of its own)
      auto scale_of = [&](int kb) -> float {
        float s = 1.0f;
        if (q.a.by_m) s = m < q.M ? q.a.inv[kb * q.a.inv_ld + m] : 0.0f;
        else if (q.a.inv) s = q.a.mn ? q.a.inv[(i64)kb * q.a.inv_ld + tm] : q.a.inv[(i64)tm * q.a.inv_ld + kb];
        if (q.b.inv) s *= q.b.mn ? q.b.inv[(i64)kb * q.b.inv_ld + nb] : q.b.inv[(i64)nb * q.b.inv_ld + kb];
        return s;
      };
      float s = scale_of(at.k0 / 128);
      for (int kb = at.k0 / 128; kb * 128 < at.k1; ++kb, ++run) {
        const float s_next = (kb + 1) * 128 < at.k1 ? scale_of(kb + 1) : 0.0f;
        if (!mbar_wait(&bars[B_RUN + (run & 1)], (run >> 1) & 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint32_t src = tmem + (run & 1) * kBN + half * 128 + ((uint32_t)(quarter * 32) << 16);
        const float2 s2 = make_float2(s, s);
#pragma unroll
        for (int c = 0; c < 128; c += 32) {
          uint32_t v[32];
          tmem_ld32(src + c, v);
          wait_for_cols<32>(v);
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 x = fma2(make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), s2, make_float2(acc[c + e], acc[c + e + 1]));
            acc[c + e] = x.x; acc[c + e + 1] = x.y;
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[B_RUNFREE + (run & 1)]);
        s = s_next;
      }
      if (!ok) break;
      constexpr float kL2e = 1.4426950408889634f;
      const int mrow = tm * kBM + quarter * 32;
      if constexpr (WHAT == Tile16::Store) {
        const float alpha = (q.alpha ? *q.alpha : 1.0f) * q.alpha_host;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          // 16-byte pieces of a 128-byte row, in the copy engine's 128-byte swizzle
          if (lane == 0) tma_store_wait_read();
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<float4*>(stg + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                make_float4(acc[c * 32 + 4 * e] * alpha, acc[c * 32 + 4 * e + 1] * alpha, acc[c * 32 + 4 * e + 2] * alpha, acc[c * 32 + 4 * e + 3] * alpha);
          const int col = n0 + c * 32;
          if (q.by_copy) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0 && col < q.N && mrow < q.M) {
              if (q.add) add_block(&q.out_map, stg, col, mrow, 0); else store_block(&q.out_map, stg, col, mrow, at.part);
              commit_blocks();
            }
          } else {
            __syncwarp();
            const int live = q.M - mrow < 32 ? q.M - mrow : 32;
            if (col + lane < q.N) {
              float* o = q.out + (i64)mrow * q.ldo + col + lane;
              for (int r = 0; r < live; ++r) {
                const float x = *reinterpret_cast<const float*>(stg + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
                o[(i64)r * q.ldo] = q.add ? o[(i64)r * q.ldo] + x : x;
              }
            }
          }
        }
      } else if constexpr (WHAT == Tile16::RowStats) {
        const int live = q.N - n0;                     // columns of this half that exist
        if (live > 0) {
          const int tgt = target - p.col0 - n0;
          if (live < 128) {
#pragma unroll
            for (int c = 0; c < 128; ++c) if (c >= live) acc[c] = -INFINITY;
          }
          if (__any_sync(0xffffffffu, tgt >= 0 && tgt < 128 && tgt < live)) {
#pragma unroll
            for (int c = 0; c < 128; ++c) if (c == tgt && c < live) p.target_value[m] = acc[c];
          }
          float mx[4] = {acc[0], acc[1], acc[2], acc[3]};
#pragma unroll
          for (int c = 4; c < 128; ++c) mx[c & 3] = fmaxf(mx[c & 3], acc[c]);
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const float lift = top > -INFINITY ? -top * kL2e : 0.0f;
          const float2 k2 = make_float2(kL2e, kL2e), l2 = make_float2(lift, lift);
          float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
#pragma unroll
          for (int c = 0; c < 128; c += 4) {
            const float2 x = fma2(make_float2(acc[c], acc[c + 1]), k2, l2), y = fma2(make_float2(acc[c + 2], acc[c + 3]), k2, l2);
            sum0 = add2(sum0, make_float2(exp2_fast(x.x), exp2_fast(x.y)));
            sum1 = add2(sum1, make_float2(exp2_fast(y.x), exp2_fast(y.y)));
          }
          sum0 = add2(sum0, sum1);
          if (m < q.M) p.stats[(i64)(tn * 2 + half) * q.M + m] = make_float2(top, sum0.x + sum0.y);
        }
      } else {
        const int tgt = target - p.col0 - n0;
        off = target != kNoTarget ? 14.0f - off * kL2e : -INFINITY;     // (2^14 rides in the exponent; a row without a target is 0: its logits are finite, the row of x was read as 0)
        const float2 k2 = make_float2(kL2e, kL2e), o2 = make_float2(off, off);
#pragma unroll
        for (int c = 0; c < 128; c += 2) {
          const float2 x = fma2(make_float2(acc[c], acc[c + 1]), k2, o2);
          acc[c] = exp2_fast(x.x); acc[c + 1] = exp2_fast(x.y);
        }
        if (__any_sync(0xffffffffu, tgt >= 0 && tgt < 128)) {
#pragma unroll
          for (int c = 0; c < 128; ++c) if (c == tgt) acc[c] -= kGradScale;
        }
        if (q.N - n0 < 128) {
#pragma unroll
          for (int c = 0; c < 128; ++c) if (n0 + c >= q.N) acc[c] = 0.0f;
        }
        // the exponent of the largest of each column among these 32 rows, for the other quarters of the tile's rows
        if (p.with_cols) {
          if (i > 0 && !warp_wait(&bars[B_COLSREAD + half], (i - 1) & 1, abort_flag)) break;      // (the last tile's have been read)
          exponents[(half * 4 + quarter) * 32 + lane] = largest_of_columns(acc, stg, lane);
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars[B_COLS + half]);
        }
        if (p.with_rows) store_planes(&q.out_map, stg, acc, n0, mrow, q.N, q.M, lane);
        if (p.with_cols) {
          if (!warp_wait(&bars[B_COLS + half], i & 1, abort_flag)) break;
          const uint32_t* e = exponents + half * 128 + lane;
          const uint32_t top = __vmaxu4(__vmaxu4(e[0], e[32]), __vmaxu4(e[64], e[96]));
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars[B_COLSREAD + half]);
          uint32_t scale = 0;                // 2^e of the four columns as exponent bytes: the largest comes to lie in [2^13, 2^15); e is not below 0 (NaN), nor above 100
          float inv[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int up = min(max(14 + 127 - (int)((top >> (8 * j) & 127) * 2 + 1), 0), 100);
            scale |= (uint32_t)(127 + up) << (8 * j);
            inv[j] = __uint_as_float((uint32_t)(127 - up) << 23);
          }
          if (quarter == 0 && n0 + 4 * lane < q.N) *reinterpret_cast<float4*>(p.col_inv + tm * p.col_inv_ld + n0 + 4 * lane) = make_float4(inv[0], inv[1], inv[2], inv[3]);
#pragma unroll
          for (int c = 0; c < 128; c += 4) {
            const uint32_t f = __shfl_sync(0xffffffffu, scale, c >> 2);
            acc[c] *= __uint_as_float(f << 23 & 0x7f800000u); acc[c + 1] *= __uint_as_float(f << 15 & 0x7f800000u);
            acc[c + 2] *= __uint_as_float(f << 7 & 0x7f800000u); acc[c + 3] *= __uint_as_float(f >> 1 & 0x7f800000u);
          }
          store_planes(&p.col_map, stg, acc, n0, mrow, q.N, q.M, lane);
        }
      }
    }
    if (WHAT != Tile16::RowStats && lane == 0) tma_store_wait_read();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.err, ERRBIT_WAIT_TIMEOUT);
}

int make_operand(const Op16& o, int box_mn, OperandDev* d) {
  if (!encode_fn()) return set_error(VB_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  cuuint64_t dims[3] = {(cuuint64_t)o.s.cols, (cuuint64_t)o.s.rows, 2}, strides[2] = {(cuuint64_t)o.s.ld * 2, (cuuint64_t)o.s.plane * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)(o.mn ? 64 : box_mn), 1}, estr[3] = {1, 1, 1};
  CUresult r = encode_fn()(&d->map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, o.s.planes, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(VB_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
  d->inv = o.s.inv; d->inv_ld = o.s.inv_ld; d->mn = o.mn; d->by_m = o.s.scale != Scale16::Block;
  return VB_OK;
}

// map of a result for the epilogue's 32 x 32 blocks: f32 rows of `ld` (128-byte swizzle), a plane a part, or the two planes of halves (64-byte swizzle)
int make_result(CUtensorMap* map, void* base, i64 cols, i64 rows, i64 ld, i64 plane, int planes, bool half) {
  const cuuint64_t size = half ? 2 : 4;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes}, strides[2] = {(cuuint64_t)ld * size, (cuuint64_t)plane * size};
  cuuint32_t box[3] = {32, 32, 1}, estr[3] = {1, 1, 1};
  CUresult r = encode_fn()(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, base, dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, half ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(VB_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
  return VB_OK;
}

// the parts of a product added in order
__global__ void __launch_bounds__(256) k_join_parts(const float* __restrict__ part, i64 part_ld, i64 part_step, int parts, float* __restrict__ out, i64 ldo, int M, int N, bool add) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  for (i64 m = blockIdx.y; m < M; m += gridDim.y) {
    const float* p = part + m * part_ld + n;
    float s = add ? out[m * ldo + n] : 0.0f;
    int i = 0;
    for (; i + 4 <= parts; i += 4) {
      const float a = p[i * part_step], b = p[(i + 1) * part_step], c = p[(i + 2) * part_step], d = p[(i + 3) * part_step];
      s = (((s + a) + b) + c) + d;
    }
    for (; i < parts; ++i) s += p[i * part_step];
    out[m * ldo + n] = s;
  }
}

template <Tile16 WHAT>
int launch(const Params& p, int ctas) {
  static bool ready = false;
  if (!ready) {
    VB_CUDA(cudaFuncSetAttribute(k_gemm16<WHAT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    ready = true;
  }
  if (WHAT == Tile16::RowStats) return launch_early(k_gemm16<WHAT>, dim3(ctas), dim3(kThreads), kSmem, p);
  k_gemm16<WHAT><<<ctas, kThreads, kSmem, ctx().stream>>>(p);
  VB_LAUNCH_CHECK();
  return VB_OK;
}

}  // namespace

Split16 split16_at(void* mem, i64 rows, i64 cols, Scale16 scale) {
  Split16 s{};
  s.rows = rows; s.cols = cols; s.ld = (cols + 7) / 8 * 8; s.plane = rows * s.ld; s.scale = scale;
  s.inv_ld = scale == Scale16::Row ? rows : scale == Scale16::Column ? s.ld : (cols + 127) / 128;
  s.planes = mem;
  s.inv = reinterpret_cast<float*>(static_cast<uint8_t*>(mem) + ((size_t)(2 * s.plane) * 2 + 15) / 16 * 16);
  return s;
}

int launch_split16(const SplitJob* jobs, int n, const TargetRows* rows) {
  SplitJobs d{};
  if (rows) d.rows = *rows;
  d.err = ctx().d_err;
  double bytes = 0.0;
  i64 all = 0;
  for (int i = 0; i < n; ++i) {
    const Split16& s = jobs[i].to;
    const i64 cb = (s.cols + 127) / 128, blocks = ((s.rows + 127) / 128) * cb;
    d.job[i] = SplitDev{jobs[i].x, jobs[i].keep, (__half*)s.planes, s.inv, s.rows, s.cols, s.ld, s.plane, s.inv_ld, (int)cb, (int)blocks,
                        s.cols % 4 == 0 && (reinterpret_cast<uintptr_t>(jobs[i].x) & 15) == 0, s.scale == Scale16::Row};
    all += blocks;
    bytes += 8.0 * (double)s.rows * (double)s.cols;
  }
  if (all > 0x7fffffff) return set_error(VB_ERR_UNSUPPORTED, "matrix too large to split");
  if (all == 0) return VB_OK;
  ProfScope prof("split16", bytes);
  k_split16<<<(unsigned)all, 256, 0, ctx().stream>>>(d);
  VB_LAUNCH_CHECK();
  return VB_OK;
}

int launch_gemm16(Tile16 what, const Product16* products, int n, int* counter) {
  Params p{};
  p.counter = counter;
  double flops = 0.0;
  i64 work = 0;                    // runs of 128 k, and three for a tile's epilogue
  for (int i = 0; i < n; ++i) {
    const Product16& g = products[i];
    const i64 tm = (g.M + kBM - 1) / kBM, tn = (g.N + kBN - 1) / kBN;
    if (g.M > 0x7fffff00 || g.N > 0x7fffff00 || g.K > 0x7fffff00 || tm * tn > 0x3fffffff) return set_error(VB_ERR_UNSUPPORTED, "product too large");
    work += tm * tn * ((g.K + 127) / 128 + 3);
  }
  Temp hold[2];
  for (int i = 0; i < n; ++i) {
    const Product16& g = products[i];
    ProblemDev& q = p.prob[i];
    const i64 tm = (g.M + kBM - 1) / kBM, tn = (g.N + kBN - 1) / kBN, runs = (g.K + 127) / 128;
    q.M = (int)g.M; q.N = (int)g.N; q.K = (int)g.K; q.tiles_m = (int)tm;
    // A tile whose sum is longer than an SM's share of the launch is formed in parts of that length, eight runs at least (few rows, width 1024,
    // 50304 columns: dx is four tiles of 393 runs; with 64 rows, forward and gradients 1259 us in one part, 450 so).
    q.parts = 1;
    q.part_k = (int)(runs * 128);
    if (what == Tile16::Store) {
      const i64 share = work / ctx().sm_count > 8 ? work / ctx().sm_count : 8;
      if (runs > share + share / 2) {
        const i64 parts = (runs + share - 1) / share, part_runs = (runs + parts - 1) / parts;
        q.parts = (int)((runs + part_runs - 1) / part_runs);
        q.part_k = (int)(part_runs * 128);
      }
    }
    q.tiles = (int)(tm * tn * q.parts);
    VB_TRY(make_operand(g.a, kBM, &q.a));
    VB_TRY(make_operand(g.b, kBN, &q.b));
    q.out = g.out; q.ldo = g.ldo; q.add = g.add; q.alpha = g.alpha; q.alpha_host = g.alpha_host;
    // (the copy engine stores rows that begin on 16 bytes)
    q.by_copy = what == Tile16::Store && g.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(g.out) & 15) == 0;
    if (q.parts > 1) {
      const i64 ld = (g.N + 3) / 4 * 4;
      VB_TRY(scratch_alloc((size_t)(q.parts * g.M * ld) * sizeof(float), &hold[i].p));
      q.by_copy = 1; q.add = 0;
      VB_TRY(make_result(&q.out_map, hold[i].p, g.N, g.M, ld, g.M * ld, q.parts, false));
    } else if (q.by_copy) VB_TRY(make_result(&q.out_map, g.out, g.N, g.M, g.ldo, g.ldo * g.M, 1, false));
    if (what == Tile16::LossGrad) {
      const Split16 &y = g.grad, &z = g.grad_by_column;
      p.with_rows = y.planes != nullptr; p.with_cols = z.planes != nullptr; p.col_inv = z.inv; p.col_inv_ld = z.inv_ld;
      if (p.with_rows) VB_TRY(make_result(&q.out_map, y.planes, g.N, g.M, y.ld, y.plane, 2, true));
      if (p.with_cols) VB_TRY(make_result(&p.col_map, z.planes, g.N, g.M, z.ld, z.plane, 2, true));
    }
    flops += 2.0 * (double)g.M * (double)g.N * (double)g.K;
  }
  p.target = products[0].target; p.col0 = (int)products[0].col0; p.stats = products[0].stats; p.target_value = products[0].target_value; p.lse = products[0].lse;
  p.err = ctx().d_err;
  const int tiles = p.prob[0].tiles + p.prob[1].tiles;
  if (tiles == 0) return VB_OK;
  ProfScope prof("gemm16", flops);
  const int ctas = tiles < ctx().sm_count ? tiles : ctx().sm_count;
  switch (what) {
    case Tile16::Store: VB_TRY(launch<Tile16::Store>(p, ctas)); break;
    case Tile16::RowStats: VB_TRY(launch<Tile16::RowStats>(p, ctas)); break;
    default: VB_TRY(launch<Tile16::LossGrad>(p, ctas));
  }
  for (int i = 0; i < n; ++i) {
    const Product16& g = products[i];
    if (p.prob[i].parts == 1) continue;
    const i64 ld = (g.N + 3) / 4 * 4;
    k_join_parts<<<dim3((unsigned)((g.N + 255) / 256), (unsigned)(g.M < 4096 ? g.M : 4096)), 256, 0, ctx().stream>>>((const float*)hold[i].p, ld, g.M * ld, p.prob[i].parts, g.out, g.ldo,
                                                                                                                   (int)g.M, (int)g.N, g.add);
    VB_LAUNCH_CHECK();
  }
  return VB_OK;
}

}  // namespace vb
