// The argmax order and its wave reduction, shared by the greedy token selection
// (sample.hip) and the logits step (logits.hip): the larger value, NaN above
// every number, ties to the smaller index.
#pragma once
#include "common.h"

namespace rwkv7mi {

// (va, ia) better than (vb, ib)
__device__ __forceinline__ bool am_better(float va, int64_t ia, float vb, int64_t ib) {
  const bool na = va != va, nb = vb != vb;
  if (na || nb) return na && (!nb || ia < ib);
  return va > vb || (va == vb && ia < ib);
}

__device__ __forceinline__ bool am_better(float va, int ia, float vb, int ib) {
  const bool na = va != va, nb = vb != vb;
  if (na || nb) return na && (!nb || ia < ib);
  return va > vb || (va == vb && ia < ib);
}

__device__ __forceinline__ void am_wave_best(float& bv, int& bi) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float ov = __shfl_xor(bv, o, 64);
    const int oi = __shfl_xor(bi, o, 64);
    if (am_better(ov, oi, bv, bi)) {
      bv = ov;
      bi = oi;
    }
  }
}

}  // namespace rwkv7mi
