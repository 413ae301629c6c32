// Score modifications shared by the decode and prefill attention kernels that
// carry them (attn_decode_mod.cu, attn_prefill_mod.cu).
//
// For a query at position p and a key at position j, with s = q . k:
//   x = scale * s;  x = c * tanh(x / c)  (cap);  x = x - slope * |p - j|  (distance bias)
// and the key is visible iff lo <= j < hi.  The kernels keep x in base 2
// (times log2 e), where the softmax needs one ex2 per score.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "qkv_paged.cuh"

namespace krt {

// Workspaces of both attentions: status word and prompt queue in the header,
// then decode's counters, then partial results.  What must be zero between
// calls (queue, counters) lies at the same place for every call, of either
// kind and of any size, and partial results never reach it: one buffer serves
// all calls that follow one another.
constexpr int kModCounters = 16384;  // (sequence, KV head) pairs; calls of more zero their own
constexpr size_t kModCountersAt = kWsHeaderBytes;
constexpr size_t kModPartsAt = kModCountersAt + kModCounters * 4;

struct ScoreMod {
  float mul;         // scale * log2(e)
  float cap2;        // cap * log2(e), 0 = no cap
  float cap_in;      // 2 * log2(e) * scale / cap: ex2(s * cap_in) = e^(2 x / c)
  const float* slopes;  // [n_heads] or NULL
  int window;        // 0 = none
  int wide_cap;      // decode: small scores take the cap's polynomial
  // cap by polynomial while |s| <= poly_max: x = s * P(s^2), see cap_poly
  float2 poly[5];    // each coefficient twice: operands of packed multiply-adds
  float poly_max;    // negative: never
};

inline ScoreMod make_score_mod(float scale, float softcap, const float* slopes, int window) {
  constexpr float kLog2e = 1.4426950408889634f;
  ScoreMod m;
  const float sc = scale > 0.f ? scale : 0.08838834764831845f;  // 1 / sqrt(128)
  m.mul = sc * kLog2e;
  m.cap2 = (float)std::min((double)softcap * kLog2e, 1.5e38);
  m.cap_in = softcap > 0.f ? std::min(2.f * kLog2e * sc / softcap, 1e38f) : 0.f;
  m.slopes = slopes;
  m.window = window;
  m.wide_cap = 0;
  m.poly_max = -1.f;
  for (int k = 0; k < 5; ++k) m.poly[k] = make_float2(0.f, 0.f);
  if (softcap > 0.f) {
    // cap2 * tanh(u), u = a s, as an odd polynomial in s: coefficients of u^(2k+1)
    // times cap2 a^(2k+1) (cap2 a = mul).  cap_poly's where their powers of a keep
    // within the range of a float.  For a larger cap (a softcap of 884 at the usual
    // scale) the scores that matter are small beside it: the series of tanh, whose
    // next term is below 1e-8 of the first up to u_max.
    static const double fit[5] = {0.9999985098838806, -0.33326974511146545, 0.13257454335689545, -0.05019525811076164,
                                  0.013194185681641102};
    static const double series[3] = {1.0, -1.0 / 3, 2.0 / 15};
    const double a = (double)sc / softcap;
    const bool fitted = a > 1e-4 && a < 1e3 && softcap < 1e6f;
    const int terms = fitted ? 5 : a > 1e-9 ? 3 : a > 1e-18 ? 2 : 1;
    const double u_max = fitted ? 0.7 : terms == 3 ? 0.05 : terms == 2 ? 1e-3 : 1e-4;
    if (a < 1e3) {
      double f = fitted ? a * m.cap2 : (double)m.mul;
      for (int k = 0; k < terms; ++k, f *= a * a) {
        const float c = (float)((fitted ? fit : series)[k] * f);
        m.poly[k] = make_float2(c, c);
      }
      m.poly_max = (float)std::min(u_max / a, 1e18);  // its square is a float too
    }
  }
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
// and is off by about 2e-7 * cap2, also near zero (one rounding each of 1 + e
// and of the difference), where the hardware tanh would be off by 5e-4 * cap2:
// more than the bf16 rounding of the weights at a cap of 50.
__device__ __forceinline__ float cap_score(float s, float cap_in, float cap2) {
  const float e = ex2(s * cap_in);
  return fmaf(-2.f * cap2, rcp_approx(1.f + e), cap2);
}

// ---- two floats in one 64-bit register: one issue slot for two multiply-adds
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair_of(const float2& v) { return *reinterpret_cast<const f32x2*>(&v); }
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// P(w), w = s^2, of cap2 * tanh(scale s / c) = s * P(s^2) for |u| = |scale s /
// c| <= 0.7: the degree-4 polynomial in u^2 with the smallest largest error of
// u * P(u^2) against tanh(u) there (fitted by reweighted least squares), off
// by at most 9.94e-8, and 1.5e-6 of tanh(u).  Scores beyond that take cap_score;
// a cap outside the coefficients' range takes tanh's series (make_score_mod).
// Five multiply-adds and no special-function operation, of which the softmax
// needs all: tanh by ex2 and rcp would triple them.
__device__ __forceinline__ f32x2 cap_poly(f32x2 w, const f32x2* c) {
  return fma2(fma2(fma2(fma2(c[4], w, c[3]), w, c[2]), w, c[1]), w, c[0]);
}
// The capped score of s, one value.
__device__ __forceinline__ float cap_at(float s, const float2* c) {
  const float w = s * s;
  return s * fmaf(fmaf(fmaf(fmaf(c[4].x, w, c[3].x), w, c[2].x), w, c[1].x), w, c[0].x);
}

}  // namespace krt
