// Shaped attention scores, in exp2 units: s = scale (q . k), capped by cap tanh(s / cap), less slope * distance.
#pragma once

#include "decode_common.h"

namespace ti {

constexpr float kLog2e = 1.4426950408889634f;

// Factors of a call. The cap is cap tanh(y) = cap (1 - 2 / (1 + e^2y)), one exponential and one reciprocal, with exact
// limits for scores that leave 32 bits. The difference cancels near y = 0 and leaves an absolute error of about
// cap * 1e-7 (the two units' last bits), 5e-6 for a cap of 50.
struct ScoreShape {
  float scale_log2;  // scale log2 e
  float cap_in;      // 2 scale log2 e / cap
  float cap_log2;    // cap log2 e; 0: no cap
};

// How a kernel's scores are capped.
enum : int { kNoCap, kCap, kWideCap };

__device__ __forceinline__ float capped(float dot, const ScoreShape& s) {
  const float r = __builtin_amdgcn_rcpf(1.f + fast_exp2(dot * s.cap_in));
  return fmaf(-2.f * s.cap_log2, r, s.cap_log2);
}

// Caps beyond this (an error of 2.6e-5, a twentieth of half an fp16 step of a weight) take the form below: a call with a
// cap of 1e4 would have scores of any size off by 1e-3. It costs ten more instructions a score (2,048 queries in a window
// of 4,096 with 24/4 heads of 256 and a cap of 1,000 318 us against 260 by the difference; a step of 32 x 16,384 tokens
// the same).
constexpr float kCloseCap = 256.f;

// |y| < 1/2: y (945 + 105 y^2 + y^4) / (945 + 420 y^2 + 15 y^4), from the continued fraction of tanh, off by less than
// 2^-24 of it, so that the error is a few last bits of the capped score. Beyond, the difference above keeps its bits.
__device__ __forceinline__ float capped_wide(float dot, const ScoreShape& s) {
  const float y = dot * s.cap_in * (0.5f / kLog2e), y2 = y * y;
  const float near = dot * s.scale_log2 * fmaf(y2, y2 + 105.f, 945.f) *
                     __builtin_amdgcn_rcpf(fmaf(y2, fmaf(y2, 15.f, 420.f), 945.f));
  const float far = capped(dot, s);
  return fabsf(y) < 0.5f ? near : far;
}

// Caps that the calls take. A smaller one, or a scale far above it, leaves 32 bits.
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
inline int cap_of(const ScoreShape& s) {
  return s.cap_log2 == 0.f ? kNoCap : s.cap_log2 <= kCloseCap * kLog2e ? kCap : kWideCap;
}

}  // namespace ti
