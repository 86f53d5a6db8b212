// What the dense attention kernels' running softmax shares: when a row's reference is renewed, and where
// it lies, by the type that the weights are multiplied in.
#pragma once

#include "common.cuh"

namespace mzb {

// A row's sum and output are rescaled only when its maximum has grown by more than 2^GROW, so weights are at most
// 2^GROW.  bf16 has fp32's range.  f16 ends at 2^16 and rounds what lies below 2^-14 to multiples of 2^-24: beside one
// key with nearly all of the weight (a sink), the weights of a long context would lose their digits or vanish, so
// the reference lies 2^8 below the maximum (weights of at most 2^15, rounded to multiples of 2^-32 of the largest).
// Maxima from 2^23 on, where fp32 counts in whole numbers and less, are the reference themselves; GROW = 7 is
// rounded to 8 there at most.
template <int DT>
struct Running {
  static constexpr float GROW = DT == MZB_F16 ? 7.0f : 8.0f;
  // exponent (log2) that the weights of a row with maximum m are relative to: -inf while no score is above it, and
  // 0 in that place for the weights themselves
  static __device__ __forceinline__ float relative(float m) {
    if constexpr (DT == MZB_F16) return fabsf(m) < 8388608.0f ? m - 8.0f : m;
    else return m;
  }
  static __device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.0f : relative(m); }
};

}  // namespace mzb
