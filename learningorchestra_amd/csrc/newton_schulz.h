// What the bindings and the kernels of newton_schulz.hip share.
#pragma once

#include <hip/hip_runtime.h>

namespace lo {

constexpr int kNsChunk = 8192;  // elements a block of the elementwise passes

struct NsMat {
  long src;        // first element in the input
  long ws;         // first half of its workspace
  int rows, cols;  // as stored
  int mp, np;      // short and long side, padded to whole tiles
  int part;        // first of its partial sums
  int chunks;      // how many
  float gain;      // factor on the learning rate
};

// A group of matrices, by a table (mats, *_starts with count + 1 prefix sums)
// or, without one, count equal matrices spaced by the steps.
struct NsGroup {
  const NsMat* mats;
  const int *chunk_starts, *split_starts, *tri_starts, *rect_starts;
  int count, tile;
  NsMat one;
  long src_step, ws_step, part_step;
  long chunks, splits, tris, rects;                   // of one of them
  long all_chunks, all_splits, all_tris, all_rects;  // of the group
  void* ws;
  double* parts;
};

// grad of the input's type; mom (fp32) or null
struct NsInput {
  const void* grad;
  float* mom;
  float gscale, mu;
  int nesterov;
};

// out of the input's type, or the parameters to update
struct NsOutput {
  void* out;
  float* master;
  void* mirror;
  float lr, keep;
};

// one step's coefficients and the powers of two that X, A, B and the next X
// are stored with
struct NsStep {
  float a, b, c;
  float sx, sa, sb, sn;
};

void launch_newton_schulz(const NsGroup& g, int dtype, const NsInput& in,
                          const NsStep* st, int n, float eps,
                          const NsOutput& out, hipStream_t s);

}  // namespace lo
