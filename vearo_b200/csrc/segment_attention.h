// Launchers of segment_attention.cu: causal attention with grouped heads over packed segments.
#pragma once
#include "common.h"

namespace vb {

constexpr int kSegMaxHead = 128;
struct SegHeads { const float* p; i64 st, sh; };           // [T, heads, dk], dk contiguous
struct SegShape { i64 T; int hq, hk, dk; float scale; };

// starts: n + 1 offsets.  The first call is for T = 0, the others for T > 0.
int launch_check_offsets(const float* starts, i64 n);
// out [T, hq, dk] contiguous, lse [hq, T].
int launch_segment_attention(const SegShape& s, const SegHeads& q, const SegHeads& k, const SegHeads& v, const float* starts, i64 n, float* out, float* lse);
int launch_segment_attention_backward(const SegShape& s, const SegHeads& q, const SegHeads& k, const SegHeads& v, const float* starts, i64 n,
                                      const SegHeads& out, const float* lse, const SegHeads& g, float* dq, float* dk, float* dv);

}  // namespace vb
