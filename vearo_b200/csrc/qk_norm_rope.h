// Launchers of qk_norm_rope.cu.
#pragma once
#include "common.h"

namespace vb {

constexpr int kRopeMaxPairs = 256;       // rotated pairs of a head: 2 KB of kernel parameters
struct RopeTable { double rev[kRopeMaxPairs]; };                          // turns per position of each pair: theta^(-2j / rot) / (2 pi)
struct HeadView { const float* p; i64 st, sh; int heads; };              // [tokens, heads, dk], dk contiguous; p null: absent

int launch_norm_rope(const RopeTable& tab, const HeadView& q, const HeadView& k, const float* wq, const float* wk, const float* pos,
                     float* oq, float* ok, i64 tokens, int dk, int rot, bool inter, float eps);
int launch_norm_rope_backward(const RopeTable& tab, const HeadView& q, const HeadView& k, const HeadView& gq, const HeadView& gk, const float* wq,
                              const float* wk, const float* pos, float* dq, float* dkeys, float* gwq, float* gwk, i64 tokens, int dk, int rot, bool inter,
                              float eps);

}  // namespace vb
