// layer_norm_train.hpp — which lanes hold a row of the training layer norm
// (layer_norm.hip, layer_norm_grad.hip).
#pragma once

#include "lane_groups.hpp"
#include "rows.hpp"

namespace {

// (G lanes of a row, NV vectors of 16 bytes a lane), by the vectors they hold. A row goes to the first that holds it:
// its elements stay in registers from the one read to the one write, at most 32 of a 16-bit dtype a lane. Three
// vectors for half a wave are there because two for a whole one would leave a quarter of the lanes of
// every second instruction without work.
#define LN_GROUPS(X)                                                                                                \
  X(1, 1) X(2, 1) X(4, 1) X(8, 1) X(16, 1) X(32, 1) X(64, 1) X(32, 3) X(64, 2) X(64, 3) X(64, 4) X(256, 2) X(256, 3) \
  X(256, 4) X(512, 3) X(512, 4)
// The forward pass, which holds a row once, has one more.
#define LN_GROUPS_FORWARD(X) LN_GROUPS(X) X(1024, 4)
// The most vectors that registers hold; longer rows are walked again. (With four of 1024 lanes, of which a unit
// has registers for 128 each, the gradient keeps values in scratch memory: [2000,20000] bfloat16 454 us, 97 by walking.)
constexpr int LN_VECTORS = 4096, LN_VECTORS_GRAD = 2048;

constexpr int ln_threads(int g) { return g > 256 ? g : 256; }

}  // namespace
