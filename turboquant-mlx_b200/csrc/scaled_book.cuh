// 16-bit codebooks of the tensor-core decode kernels (host side).
#pragma once

#include <stdint.h>

namespace tq {

// 16-bit floats hold 11 bits; rounding the centroids directly would leave a fixed relative error of up to 2^-12 on each.
// A common factor beta in [1, 2) is searched so that every beta * c lands (almost) on a 16-bit value; 1 / beta is
// applied in 32 bits.
struct ScaledBook {
  uint16_t c16[16];      // beta * c as f16 bits
  float beta;
  bool good;             // every centroid within 2^-13 of its value (a codebook with wild levels may have no such factor)
};
// The search takes 0.5 to 3 ms of host time; results are kept by value (the n centroids), not by address.
ScaledBook scaled_book(const float* c, int n);

}  // namespace tq
