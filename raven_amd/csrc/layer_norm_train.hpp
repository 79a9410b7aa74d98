// layer_norm_train.hpp — which lanes hold a row of the training layer norm
// (layer_norm.hip, layer_norm_grad.hip).
#pragma once

#include "lane_groups.hpp"
#include "rows.hpp"

namespace {

// (G lanes of a row, NV vectors of 16 bytes a lane), by the vectors they hold. A row goes to the first that holds it:
// its elements stay in registers from the one read to the one write, at most 32 of a 16-bit dtype a lane.
#define LN_GROUPS_SHORT(X) X(1, 1) X(2, 1) X(4, 1) X(8, 1) X(16, 1) X(32, 1) X(64, 1)
#define LN_GROUPS_LONG(X) X(64, 2) X(64, 3) X(64, 4) X(256, 2) X(256, 3) X(256, 4) X(512, 3) X(512, 4)
// The forward pass, which holds a row once, has three vectors of half a wave, where two of a whole one leave a quarter of its
// lanes without work ([8192,768] bfloat16 6.4 us, 7.2), and rows of up to 64 KB.
#define LN_GROUPS_FORWARD(X) LN_GROUPS_SHORT(X) X(32, 3) LN_GROUPS_LONG(X) X(1024, 4)
// The gradient has not the registers: three vectors leave room for half of the waves (12.7 us, 12.2 with two of a wave).
#define LN_GROUPS_GRAD(X) LN_GROUPS_SHORT(X) LN_GROUPS_LONG(X)
#define LN_GROUPS_GRAD_WORDS(X) X(1024, 3) X(1024, 4)  // of dtypes whose vectors have at most four elements
// The most vectors that registers hold; longer rows are walked again. In sixteen waves a lane has 128 registers: rows of float32 and
// float64 stay in them ([2013,16000] float32 150 us by walking, 89), with 24 or 32 elements of a 16-bit dtype values would go
// to scratch memory ([2000,20000] bfloat16 95 by walking, 111).
constexpr int LN_VECTORS = 4096;
constexpr int ln_vectors_grad(int element_size) { return element_size < 4 ? 2048 : 4096; }

constexpr int ln_threads(int g) { return g > 256 ? g : 256; }

}  // namespace
