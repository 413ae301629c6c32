// Score modifications shared by the decode and prefill attention kernels that
// carry them (attn_decode_mod.cu, attn_prefill_mod.cu).
//
// For a query at position p and a key at position j, with s = q . k:
//   x = scale * s;  x = c * tanh(x / c)  (cap);  x = x - slope * |p - j|  (distance bias)
// and the key is visible iff lo <= j < hi.  The kernels keep x in base 2
// (times log2 e), where the softmax needs one ex2 per score.
#pragma once
#include <cmath>
#include <cstdint>

namespace krt {

struct ScoreMod {
  float mul;         // scale * log2(e)
  float cap2;        // cap * log2(e), 0 = no cap
  float cap_in;      // 2 * log2(e) * scale / cap: ex2(s * cap_in) = e^(2 x / c)
  const float* slopes;  // [n_heads] or NULL
  int window;        // 0 = none
};

inline ScoreMod make_score_mod(float scale, float softcap, const float* slopes, int window) {
  constexpr float kLog2e = 1.4426950408889634f;
  ScoreMod m;
  const float sc = scale > 0.f ? scale : 0.08838834764831845f;  // 1 / sqrt(128)
  m.mul = sc * kLog2e;
  m.cap2 = softcap * kLog2e;
  m.cap_in = softcap > 0.f ? 2.f * kLog2e * sc / softcap : 0.f;
  m.slopes = slopes;
  m.window = window;
  return m;
}

constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// s -> cap2 * tanh(scale * s / c) = cap2 - 2 cap2 / (1 + e^(2 x / c)).  The
// form saturates without overflow checks (ex2 = inf gives +cap, 0 gives -cap)
// and is off by about 2e-7 * cap2 near zero (one rounding each of 1 + e and of
// the difference), where the hardware tanh would be off by 5e-4 * cap2: more
// than the bf16 rounding of the weights at a cap of 50.
__device__ __forceinline__ float cap_score(float s, float cap_in, float cap2) {
  const float e = ex2(s * cap_in);
  return fmaf(-2.f * cap2, rcp_approx(1.f + e), cap2);
}

}  // namespace krt
