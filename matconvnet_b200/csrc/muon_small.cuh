// The Newton-Schulz steps of small matrices, all of them in one launch (muon_small.cu).
#pragma once
#include "common.cuh"

namespace vlb {

constexpr int kSmallMost = 16;        // matrices in one launch
constexpr int kSmallSteps = 16;
constexpr int kSmallSide = 128, kSmallLong = 2048;

// u / (sqrt(sum of parts) + epsilon) goes through the steps; w -= rate * the result.  u and w: rows x cols floats, rows one after the other.
struct SmallMatrix { float* w; float const* u; double const* parts; int partCount, rows, cols; float rate; };

struct SmallSteps {
  int count;
  double epsilon;
  float a, b, c;
  int x[kSmallSteps + 1], gram[kSmallSteps], poly[kSmallSteps];      // scale exponents of the halves: of X before each step, of A and of b*A + c*A*A
};

// Fits: at most kSmallSide rows or columns, at most kSmallLong of the other, at most kSmallSteps steps.
bool small_fits(int rows, int cols, int steps);

int small_matrices(vlb_ctx* ctx, SmallMatrix const* m, int count, SmallSteps const& steps);

}  // namespace vlb
