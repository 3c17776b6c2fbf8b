// The extern "C" entry points of the decoder-training operators: norm and rotation of queries and keys, causal attention over
// packed segments, and the vocabulary projection with its cross entropy.  None of them is a `BackendOps` field of the reference
// (its layers use learned positions, equal heads, padded batches and a separate projection and loss, crates/vearo-nn/src/lib.rs:584-621,
// 741-793); they stand beside vb_layernorm, vb_fused_attention and vb_cross_entropy for models that need them.
#include "common.h"
#include "head_loss.h"
#include "qk_norm_rope.h"
#include "segment_attention.h"
#include <cmath>

using namespace vb;

namespace {

// The library's device for the length of a call, whatever the calling thread had current.
struct OnDevice {
  int before = -1;
  OnDevice() { if (ctx().ready && cudaGetDevice(&before) == cudaSuccess && before != ctx().device) cudaSetDevice(ctx().device); }
  ~OnDevice() { if (ctx().ready && before >= 0 && before != ctx().device) cudaSetDevice(before); }
};
// Outputs of a call that may still fail: the caller's descriptors are written by done(), after the last look at the inputs' (which may be
// the same descriptors); without it what has been allocated is given back.
struct Outputs {
  vb_tensor fresh[6], *to[6];
  int n = 0;
  int add(vb_tensor* out, int rank, const i64* dims, float** p) {
    VB_TRY(new_output(&fresh[n], rank, dims));
    to[n] = out;
    return slot_ptr(fresh[n++].slot, p);
  }
  void done() { for (int i = 0; i < n; ++i) *to[i] = fresh[i]; n = 0; }
  ~Outputs() { for (int i = 0; i < n; ++i) slot_release(fresh[i].slot, nullptr); }
};
// The arena hands scratch and outputs of one call to the next, which a replay of a captured call would not know of.
int common_checks(const char* who) {
  if (!ctx().ready) return set_error(VB_ERR_NOT_INIT, "vb_init has not been called");
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  VB_CUDA(cudaStreamIsCapturing(ctx().stream, &st));
  if (st != cudaStreamCaptureStatusNone) return set_error(VB_ERR_UNSUPPORTED, std::string(who) + ": not available while the compute stream is being captured");
  return VB_OK;
}

// [tokens, heads, dk] with contiguous components: the tensor in place, or a copy where its last dimension is strided
int head_view(const vb_tensor* x, HeadView* v, Temp& hold) {
  float* p;
  VB_TRY(tensor_ptr(x, &p));
  const i64 heads = x->dims[1], dk = x->dims[2];
  if (dk == 1 || x->strides[2] == 1) { *v = HeadView{p, x->strides[0], x->strides[1], (int)heads}; return VB_OK; }
  const float* c;
  VB_TRY(contiguous_ptr(x, &c, hold));
  *v = HeadView{c, heads * dk, dk, (int)heads};
  return VB_OK;
}

int rope_checks(const vb_tensor* q, const vb_tensor* k, const vb_tensor* wq, const vb_tensor* wk, const vb_tensor* positions, float theta,
                int rot_dim, float eps, RopeTable* tab) {
  VB_CHECK(q && wq && positions && (k != nullptr) == (wk != nullptr), "q, its weight and positions are needed, and k with its weight or neither");
  VB_CHECK(q->rank == 3 && (!k || k->rank == 3), "queries and keys must be [tokens, heads, head size]");
  const i64 T = q->dims[0], dk = q->dims[2];
  VB_CHECK(T >= 0 && q->dims[1] >= 1 && dk >= 1, "at least one head of at least one component");
  VB_CHECK(!k || (k->dims[0] == T && k->dims[2] == dk && k->dims[1] >= 1), "keys must have the queries' tokens and head size");
  VB_CHECK(wq->rank == 1 && wq->dims[0] == dk && (!wk || (wk->rank == 1 && wk->dims[0] == dk)), "norm weights must be [head size]");
  VB_CHECK(positions->rank == 1 && positions->dims[0] == T, "positions must be [tokens]");
  VB_CHECK(rot_dim >= 0 && rot_dim <= dk && rot_dim % 2 == 0, "rot_dim must be even and at most the head size");
  VB_CHECK(std::isfinite(theta) && theta > 0.0f && std::isfinite(eps) && eps >= 0.0f, "theta must be positive and eps not negative");
  if (dk > 2 * kRopeMaxPairs) return set_error(VB_ERR_UNSUPPORTED, "vb_qk_norm_rope: head sizes up to 512");
  if (T > 0x7fffffff || q->dims[1] + (k ? k->dims[1] : 0) > 65536) return set_error(VB_ERR_UNSUPPORTED, "vb_qk_norm_rope: at most 2^31 - 1 tokens and 65536 heads");
  const double step = rot_dim > 0 ? -2.0 / rot_dim * std::log((double)theta) : 0.0;
  for (int j = 0; j < rot_dim / 2; ++j) tab->rev[j] = std::exp(j * step) / 6.283185307179586476925286766559;
  return VB_OK;
}

int segment_checks(const vb_tensor* q, const vb_tensor* k, const vb_tensor* v, const vb_tensor* starts, float scale, SegShape* s) {
  VB_CHECK(q && k && v && starts, "null tensor");
  VB_CHECK(q->rank == 3 && k->rank == 3 && same_shape(*k, *v), "queries must be [tokens, heads, head size], keys and values alike");
  VB_CHECK(q->dims[0] == k->dims[0] && q->dims[2] == k->dims[2], "keys must have the queries' tokens and head size");
  VB_CHECK(q->dims[1] >= 1 && k->dims[1] >= 1 && q->dims[1] % k->dims[1] == 0, "the number of query heads must be a multiple of the number of key heads");
  VB_CHECK(q->dims[2] >= 1, "head size must be greater than 0");
  VB_CHECK(starts->rank == 1 && starts->dims[0] >= 1, "starts must be [segments + 1]");
  VB_CHECK(std::isfinite(scale) && scale > 0.0f, "scale must be positive");
  if (q->dims[2] > kSegMaxHead) return set_error(VB_ERR_UNSUPPORTED, "vb_segment_attention: head sizes up to 128");
  if (q->dims[0] > (i64)1 << 24 || starts->dims[0] > (i64)1 << 24) return set_error(VB_ERR_UNSUPPORTED, "vb_segment_attention: offsets beyond 2^24 are not whole numbers of f32");
  if (q->dims[1] > 1024) return set_error(VB_ERR_UNSUPPORTED, "vb_segment_attention: at most 1024 query heads");
  *s = SegShape{q->dims[0], (int)q->dims[1], (int)k->dims[1], (int)q->dims[2], scale};
  return VB_OK;
}
int seg_view(const vb_tensor* x, SegHeads* v, Temp& hold) {
  HeadView h;
  VB_TRY(head_view(x, &h, hold));
  *v = SegHeads{h.p, h.st, h.sh};
  return VB_OK;
}

int head_loss_checks(const vb_tensor* x, const vb_tensor* w, const vb_tensor* targets, i64* n) {
  VB_CHECK(x && w && targets, "null tensor");
  VB_CHECK(x->rank >= 2 && w->rank == 2 && targets->rank >= 1, "x must be [.., width], weight [vocabulary, width], targets [..]");
  const i64 d = x->dims[x->rank - 1], v = w->dims[0];
  VB_CHECK(d >= 1 && w->dims[1] == d, "Incompatible dimensions for matmul");
  VB_CHECK(v >= 1, "Vocabulary size must be greater than 0");
  *n = numel(*x) / d;
  VB_CHECK(*n > 0, "Batch size must be greater than 0");
  VB_CHECK(numel(*targets) == *n, "Targets shape must match batch size");
  if (v > (i64)1 << 24) return set_error(VB_ERR_UNSUPPORTED, "vb_linear_cross_entropy: classes beyond 2^24 are not whole numbers of f32");
  if (*n > (i64)1 << 30 || d > (i64)1 << 30) return set_error(VB_ERR_UNSUPPORTED, "vb_linear_cross_entropy: at most 2^30 rows and columns");
  return VB_OK;
}

}  // namespace

extern "C" {

int vb_qk_norm_rope(const vb_tensor* q, const vb_tensor* k, const vb_tensor* wq, const vb_tensor* wk, const vb_tensor* positions, float theta,
                    int rot_dim, int interleaved, float eps, vb_tensor* q_out, vb_tensor* k_out) {
  OnDevice on;
  VB_TRY(common_checks("vb_qk_norm_rope"));
  RopeTable tab;
  VB_TRY(rope_checks(q, k, wq, wk, positions, theta, rot_dim, eps, &tab));
  VB_CHECK(q_out && (!k || k_out), "null output tensor");
  Temp hq, hk, h1, h2, h3;
  HeadView vq{}, vk{};
  const float *pwq, *pwk = nullptr, *pp;
  VB_TRY(head_view(q, &vq, hq));
  if (k) VB_TRY(head_view(k, &vk, hk));
  VB_TRY(contiguous_ptr(wq, &pwq, h1));
  if (wk) VB_TRY(contiguous_ptr(wk, &pwk, h2));
  VB_TRY(contiguous_ptr(positions, &pp, h3));
  Outputs outs;
  float *oq, *ok = nullptr;
  VB_TRY(outs.add(q_out, 3, q->dims, &oq));
  if (k) VB_TRY(outs.add(k_out, 3, k->dims, &ok));
  if (q->dims[0] > 0) VB_TRY(launch_norm_rope(tab, vq, vk, pwq, pwk, pp, oq, ok, q->dims[0], (int)q->dims[2], rot_dim, interleaved != 0, eps));
  outs.done();
  return VB_OK;
}

int vb_qk_norm_rope_backward(const vb_tensor* q, const vb_tensor* k, const vb_tensor* wq, const vb_tensor* wk, const vb_tensor* positions, float theta,
                             int rot_dim, int interleaved, float eps, const vb_tensor* grad_q, const vb_tensor* grad_k, vb_tensor* gq, vb_tensor* gk,
                             vb_tensor* gwq, vb_tensor* gwk) {
  OnDevice on;
  VB_TRY(common_checks("vb_qk_norm_rope_backward"));
  RopeTable tab;
  VB_TRY(rope_checks(q, k, wq, wk, positions, theta, rot_dim, eps, &tab));
  VB_CHECK(grad_q && same_shape(*q, *grad_q) && (k ? grad_k && same_shape(*k, *grad_k) : !grad_k), "gradients must have the shapes of q and k");
  VB_CHECK(gq && gwq && (!k || (gk && gwk)), "null output tensor");
  Temp hq, hk, hgq, hgk, h1, h2, h3;
  HeadView vq{}, vk{}, vgq{}, vgk{};
  const float *pwq, *pwk = nullptr, *pp;
  VB_TRY(head_view(q, &vq, hq));
  VB_TRY(head_view(grad_q, &vgq, hgq));
  if (k) { VB_TRY(head_view(k, &vk, hk)); VB_TRY(head_view(grad_k, &vgk, hgk)); }
  VB_TRY(contiguous_ptr(wq, &pwq, h1));
  if (wk) VB_TRY(contiguous_ptr(wk, &pwk, h2));
  VB_TRY(contiguous_ptr(positions, &pp, h3));
  Outputs outs;
  float *pgq, *pgk = nullptr, *pgwq, *pgwk = nullptr;
  const i64 dk = q->dims[2];
  VB_TRY(outs.add(gq, 3, q->dims, &pgq));
  VB_TRY(outs.add(gwq, 1, &dk, &pgwq));
  if (k) { VB_TRY(outs.add(gk, 3, k->dims, &pgk)); VB_TRY(outs.add(gwk, 1, &dk, &pgwk)); }
  if (q->dims[0] > 0) {
    VB_TRY(launch_norm_rope_backward(tab, vq, vk, vgq, vgk, pwq, pwk, pp, pgq, pgk, pgwq, pgwk, q->dims[0], (int)dk, rot_dim, interleaved != 0, eps));
  } else {
    VB_TRY(launch_fill(pgwq, 0.0f, dk));
    if (k) VB_TRY(launch_fill(pgwk, 0.0f, dk));
  }
  outs.done();
  return VB_OK;
}

int vb_segment_attention(const vb_tensor* q, const vb_tensor* k, const vb_tensor* v, const vb_tensor* starts, float scale, vb_tensor* out, vb_tensor* lse) {
  OnDevice on;
  VB_TRY(common_checks("vb_segment_attention"));
  SegShape s;
  VB_TRY(segment_checks(q, k, v, starts, scale, &s));
  VB_CHECK(out, "null output tensor");
  Temp hq, hk, hv, hs;
  SegHeads vq, vk, vv;
  const float* ps;
  VB_TRY(seg_view(q, &vq, hq)); VB_TRY(seg_view(k, &vk, hk)); VB_TRY(seg_view(v, &vv, hv));
  VB_TRY(contiguous_ptr(starts, &ps, hs));
  Outputs outs;
  float *po, *pl = nullptr;
  const i64 ld[2] = {s.hq, s.T};
  VB_TRY(outs.add(out, 3, q->dims, &po));
  if (lse) VB_TRY(outs.add(lse, 2, ld, &pl));
  if (s.T == 0) VB_TRY(launch_check_offsets(ps, starts->dims[0] - 1));
  else VB_TRY(launch_segment_attention(s, vq, vk, vv, ps, starts->dims[0] - 1, po, pl));
  outs.done();
  return VB_OK;
}

int vb_segment_attention_backward(const vb_tensor* q, const vb_tensor* k, const vb_tensor* v, const vb_tensor* starts, float scale, const vb_tensor* out,
                                  const vb_tensor* lse, const vb_tensor* grad_out, vb_tensor* dq, vb_tensor* dk, vb_tensor* dv) {
  OnDevice on;
  VB_TRY(common_checks("vb_segment_attention_backward"));
  SegShape s;
  VB_TRY(segment_checks(q, k, v, starts, scale, &s));
  VB_CHECK(out && lse && grad_out && same_shape(*q, *out) && same_shape(*q, *grad_out), "out and grad_out must have the shape of q");
  VB_CHECK(lse->rank == 2 && lse->dims[0] == s.hq && lse->dims[1] == s.T, "lse must be [heads, tokens]");
  VB_CHECK(dq && dk && dv, "null output tensor");
  Temp hq, hk, hv, hs, ho, hl, hg;
  SegHeads vq, vk, vv, vo, vg;
  const float *ps, *pl;
  VB_TRY(seg_view(q, &vq, hq)); VB_TRY(seg_view(k, &vk, hk)); VB_TRY(seg_view(v, &vv, hv)); VB_TRY(seg_view(out, &vo, ho)); VB_TRY(seg_view(grad_out, &vg, hg));
  VB_TRY(contiguous_ptr(starts, &ps, hs)); VB_TRY(contiguous_ptr(lse, &pl, hl));
  Outputs outs;
  float *pdq, *pdk, *pdv;
  VB_TRY(outs.add(dq, 3, q->dims, &pdq)); VB_TRY(outs.add(dk, 3, k->dims, &pdk)); VB_TRY(outs.add(dv, 3, v->dims, &pdv));
  if (s.T == 0) VB_TRY(launch_check_offsets(ps, starts->dims[0] - 1));
  else VB_TRY(launch_segment_attention_backward(s, vq, vk, vv, ps, starts->dims[0] - 1, vo, pl, vg, pdq, pdk, pdv));
  outs.done();
  return VB_OK;
}

int vb_linear_cross_entropy(const vb_tensor* x, const vb_tensor* weight, const vb_tensor* targets, int64_t ignore_index, vb_tensor* loss, vb_tensor* lse) {
  OnDevice on;
  VB_TRY(common_checks("vb_linear_cross_entropy"));
  i64 n;
  VB_TRY(head_loss_checks(x, weight, targets, &n));
  VB_CHECK(loss, "null output tensor");
  Temp hx, hw, ht, hl;
  const float *px, *pw, *pt;
  VB_TRY(contiguous_ptr(x, &px, hx)); VB_TRY(contiguous_ptr(weight, &pw, hw)); VB_TRY(contiguous_ptr(targets, &pt, ht));
  Outputs outs;
  float *ploss, *plse;
  const i64 one = 1;
  VB_TRY(outs.add(loss, 1, &one, &ploss));
  if (lse) VB_TRY(outs.add(lse, 1, &n, &plse));
  else { VB_TRY(scratch_alloc((size_t)n * sizeof(float), &hl.p)); plse = (float*)hl.p; }
  VB_TRY(launch_head_loss(px, pw, pt, ignore_index, ploss, plse, n, weight->dims[1], weight->dims[0]));
  outs.done();
  return VB_OK;
}

int vb_linear_cross_entropy_backward(const vb_tensor* x, const vb_tensor* weight, const vb_tensor* targets, int64_t ignore_index, const vb_tensor* lse,
                                     const vb_tensor* grad_out, vb_tensor* gx, vb_tensor* gw) {
  OnDevice on;
  VB_TRY(common_checks("vb_linear_cross_entropy_backward"));
  i64 n;
  VB_TRY(head_loss_checks(x, weight, targets, &n));
  VB_CHECK(lse && grad_out && numel(*lse) == n, "lse must be [rows]");
  VB_CHECK(numel(*grad_out) == 1, "grad_out must be a scalar");
  Temp hx, hw, ht, hl;
  const float *px, *pw, *pt, *pl;
  float* pg;
  VB_TRY(contiguous_ptr(x, &px, hx)); VB_TRY(contiguous_ptr(weight, &pw, hw)); VB_TRY(contiguous_ptr(targets, &pt, ht)); VB_TRY(contiguous_ptr(lse, &pl, hl));
  VB_TRY(tensor_ptr(grad_out, &pg));
  Outputs outs;
  float *pgx = nullptr, *pgw = nullptr;
  if (gx) VB_TRY(outs.add(gx, x->rank, x->dims, &pgx));
  if (gw) VB_TRY(outs.add(gw, 2, weight->dims, &pgw));
  if (gx || gw) VB_TRY(launch_head_loss_backward(px, pw, pt, ignore_index, pl, pg, pgx, pgw, n, weight->dims[1], weight->dims[0]));
  outs.done();
  return VB_OK;
}

}  // extern "C"
