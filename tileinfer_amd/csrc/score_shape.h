// Shaped attention scores, in exp2 units: s = scale (q . k), capped by cap tanh(s / cap), less slope * distance.
#pragma once

#include "decode_common.h"

namespace ti {

constexpr float kLog2e = 1.4426950408889634f;

// Factors of a call. The cap is cap tanh(y) = cap (1 - 2 / (1 + e^2y)), one exponential and one reciprocal, with an
// absolute error of about cap * 1e-7 (the two units' last bits; at most 5e-6 for a cap of 50), and exact limits for
// scores that leave 32 bits.
struct ScoreShape {
  float scale_log2;  // scale log2 e
  float cap_in;      // 2 scale log2 e / cap
  float cap_log2;    // cap log2 e; 0: no cap
};

__device__ __forceinline__ float capped(float dot, const ScoreShape& s) {
  const float r = __builtin_amdgcn_rcpf(1.f + fast_exp2(dot * s.cap_in));
  return fmaf(-2.f * s.cap_log2, r, s.cap_log2);
}

// A cap beyond this would cost the scores more than their last bits (see above); one below it, or a scale far above
// it, leaves 32 bits.
constexpr float kMaxCap = 1e4f, kMinCap = 1e-3f;

inline bool shape_ok(float scale, float cap) {
  return scale > 0.f && scale <= kMaxScale && (cap == 0.f || (cap >= kMinCap && cap <= kMaxCap && scale / cap <= kMaxScale));
}

inline ScoreShape score_shape(float scale, float cap) {
  ScoreShape s{};
  s.scale_log2 = scale * kLog2e;
  if (cap > 0.f) {
    s.cap_in = 2.f * kLog2e * (scale / cap);
    s.cap_log2 = cap * kLog2e;
  }
  return s;
}

}  // namespace ti
