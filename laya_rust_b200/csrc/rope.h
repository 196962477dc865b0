// Rotary positions: frequencies, their stretching and the device kernels.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/laya_ops.h"

namespace laya {

// Stretches n = rot / 2 frequencies (radians per position) in place; returns
// the factor on cos and sin.  Throws OpError on bad parameters.
float rope_stretch(double* freqs, int rot, const laya_rope_scaling* s);

// f radians per position as a 64-bit fixed-point fraction of a turn per
// position: position * result (mod 2^64) is the angle, whole turns dropped.
uint64_t rope_turns(double f);
// What it takes: finite, of magnitude at most 2^20.
bool rope_freq_fits(double f);

// cosb/sinb[p][j] = mscale cos/sin(p * freqs[j]) for p < positions, j < n
// (n <= 32), the tables the Wqkv epilogue reads.
cudaError_t launch_rope_table(const double* freqs, int n, float mscale, int positions, float* cosb, float* sinb,
                              cudaStream_t s);

}  // namespace laya
