// What the bindings and the kernels of newton_schulz.hip share.
#pragma once

#include <hip/hip_runtime.h>

namespace lo {

constexpr int kNsChunk = 8192;  // elements a block of the momentum pass

// the products of a step: A = X X^T, C = a + b A + c A A^T, X' = C X
enum { NS_GRAM, NS_POLY, NS_APPLY, NS_KINDS };

// how a product's tiles are shared out: the first `whole` take one block each,
// the others `splits` blocks, each a part of the sum
struct NsTiles {
  int tile;  // 32, 64 or 128
  int whole, splits;
};

struct NsMat {
  long src;        // first element in the input
  long ws;         // first half of its workspace
  int rows, cols;  // as stored
  int mp, np;      // short and long side, padded to whole tiles
  int sum;         // first of its partial norms
  int chunks;      // how many
  float gain;      // factor on the learning rate
  NsTiles kind[NS_KINDS];
};

// a block's matrix and its place in it
struct NsBlock {
  int mat, at;
};

// all that a block of a product has to know: one 64-byte line
struct alignas(64) NsTask {
  long ws;    // the matrix's workspace
  long part;  // a split tile's partial sums (floats)
  int mat, tile, mp, np;
  int ti, tj;  // tile row and column
  int k0, k1;  // steps of 32 of the sum
  int slice, splits;
  int slot;  // a split tile's counter
};

// A group of matrices, by tables (mats; blocks of the momentum pass and of the
// split; tasks of the products) or, without them, count equal matrices spaced
// by the steps.
struct NsGroup {
  const NsMat* mats;
  const NsBlock *chunk_blocks, *split_blocks;
  const NsTask* tasks[NS_KINDS];
  int count;
  NsMat one;
  long src_step, ws_step, part_step;
  int sum_step, slot_step;
  int chunks, splits, kinds[NS_KINDS];               // blocks of one of them
  int tile[NS_KINDS];  // the tiles' size, 0 where sizes differ
  long all_chunks, all_splits, all_kinds[NS_KINDS];  // of the group
  void* ws;
  double* sums;
  float* parts;
  unsigned* slots;  // arrivals at a split tile, zero between calls
  int all_slots;
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

// one step's coefficients and the powers of two that X, A, C and the next X
// are stored with
struct NsStep {
  float a, b, c;
  float sx, sa, sc, sn;
};

constexpr int kNsSmallSteps = 32;  // of one ns_small_kernel

// all of the group's matrices fit a block (ns_fit_block): `shortest` and
// `longest` are the largest of their short and of their long sides;
// n <= kNsSmallSteps
void launch_newton_schulz_small(const NsGroup& g, int shortest, int longest,
                                int dtype, const NsInput& in, const NsStep* st,
                                int n, float eps, const NsOutput& out,
                                hipStream_t s);

void launch_newton_schulz(const NsGroup& g, int dtype, const NsInput& in,
                          const NsStep* st, int n, float eps,
                          const NsOutput& out, hipStream_t s);

}  // namespace lo
