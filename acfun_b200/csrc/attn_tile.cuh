// attn_tile.cuh — what the two attention kernels share: the keys a tile of packed rows can see,
// the range in which softmax weights are kept, and fp16 packing.
#pragma once
#include "attn.cuh"

namespace acf {

// Weights are kept within fp16's upper range, so that keys far below the largest keep their bits:
// a row's offset m is set so that its largest weight is 2^kTop, and moves when one would pass
// 2^kMost.
constexpr float kTop = 7.0f, kMost = 15.0f;

// The keys [lo, hi) that some row of packed rows [r0, r0 + nr) sees, and the steps of `step` keys
// (first, n) that cover them.
struct KeyRange {
  int first, n, lo, hi;
};
__device__ __forceinline__ KeyRange key_range(const AttnArgs& a, const SeqView& sv, int r0, int nr, int step) {
  const int t_first = r0 / a.group, t_last = (r0 + nr - 1) / a.group;
  const int pos0 = sv.len - sv.n;  // position of new token 0 (negative: it sees nothing)
  const int hi = a.causal ? max(0, min(sv.len, pos0 + t_last + 1)) : sv.len;
  const int lo = a.window > 0 ? max(0, pos0 + t_first - a.window + 1) : 0;
  KeyRange k;
  k.lo = lo, k.hi = hi;
  k.first = lo / step;
  k.n = hi > lo ? (hi + step - 1) / step - k.first : 0;
  return k;
}

// The power of two that brings a row whose largest element is `top` below 1, and its inverse.  A row
// with an infinity or NaN is left as it is.
struct Pow2 {
  float down, up;
};
__device__ __forceinline__ Pow2 row_pow2(float top) {
  const int biased = (int)(__float_as_uint(top) >> 23);  // 0: zero or subnormal, 255: not finite
  const int ex = biased == 255 ? 0 : min(max(biased - 126, -100), 126);
  return {__uint_as_float((uint32_t)(127 - ex) << 23), __uint_as_float((uint32_t)(127 + ex) << 23)};
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace acf
