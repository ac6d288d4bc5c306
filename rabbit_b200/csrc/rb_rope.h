// rb_rope.h -- rotary positions: the frequency table of a rope object as the
// kernels take it (by value, in the launch's parameters) and the angle.
#pragma once
#include <stdint.h>

#include "../../include/rabbit_cuda.h"

namespace rb {

constexpr int kRopeMaxPairs = 256;

struct RopeTab {
    double turns[kRopeMaxPairs];  // rotations per position of each pair: f_i / 2 pi
    double mag;                   // magnitude of the rotated channels
    int rot, layout;
};

// The table of `r`, and its head_dim.
const RopeTab &rope_tab(const rabbit_cuda_rope *r, int *head_dim);

#ifdef __CUDACC__
// (cos, sin) of position * f in 64 bits. The whole turns are taken out of the
// product before the sine, with the product's rounding error added back, so
// the error does not grow beyond that of f itself (2^-53 of the angle).
__device__ __forceinline__ double2 rope_cs(int pos, double turns) {
    const double p = pos, t = p * turns;
    const double r = (t - rint(t)) + fma(p, turns, -t);
    double2 cs;
    sincospi(2.0 * r, &cs.y, &cs.x);
    return cs;
}
#endif

}  // namespace rb
