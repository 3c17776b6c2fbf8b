// Launchers of head_loss.cu: x [n, d], w [v, d], targets [n], all contiguous.
#pragma once
#include "common.h"

namespace vb {

int launch_head_loss(const float* x, const float* w, const float* targets, i64 ignore, float* loss, float* lse, i64 n, i64 d, i64 v);
// gx, gw: null where not wanted
int launch_head_loss_backward(const float* x, const float* w, const float* targets, i64 ignore, const float* lse, const float* g, float* gx, float* gw,
                              i64 n, i64 d, i64 v);

}  // namespace vb
