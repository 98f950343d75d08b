// The 4-bit cache format, shared by everything that writes it (kv4.cu, attention_q4.cu, prefill_gemm.cu, w8a8.cu).
//
// A head vector is rounded to bf16 (what the bf16 cache would hold), clamped to +-32752 with NaN as 0, and cut into groups of
// 64 dims. Per group: lo = fp16(min), step = fp16((max - lo) / 15), code = clamp(rint((x - lo) / step), 0, 15), 0 where step
// is 0; x ~ lo + code * step, and x is within half a step of that. fp16 holds a bf16 value as it is down to 2^-14, so lo is
// exact, and a step that is off by 2^-11 of itself moves the fifteenth code by less than a hundredth of a step. Below 2^-14
// fp16 numbers are 2^-24 apart: a lo there is off by up to 2^-25, a step by as much, fifteen times over at the top, and together
// that is up to 2^-21 more. The clamp keeps max - min inside fp16. 64 dims share a (step, lo) pair of 4 bytes: 4.5 bits a value.
// A vector's codes are D / 2 bytes, dim 2i in the low half of byte i; its pairs are D / 64 half2 {step, lo}.
#pragma once
#include "common.cuh"

namespace b200dec_detail {

constexpr float KV4_LIMIT = 32752.f;

// x as the format sees it, for values already rounded to bf16
DEVI float kv4_clamp(float x) { return x != x ? 0.f : fminf(fmaxf(x, -KV4_LIMIT), KV4_LIMIT); }

struct Kv4Group {
  float lo, step, inv;
  uint32_t word;  // half2 {step, lo}
};
DEVI Kv4Group kv4_group(float mn, float mx) {
  Kv4Group g;
  const __half lo = __float2half_rn(mn);
  g.lo = __half2float(lo);
  const __half step = __float2half_rn(__fdiv_rn(mx - g.lo, 15.f));
  g.step = __half2float(step);
  g.inv = g.step > 0.f ? __frcp_rn(g.step) : 0.f;
  g.word = (uint32_t)__half_as_ushort(step) | ((uint32_t)__half_as_ushort(lo) << 16);
  return g;
}

// rint((x - lo) / step) clamped to 0..15, as if the quotient were exact: the product with the reciprocal is off by a few
// 2^-23, so its rounding can only be wrong beside a half; the remainder d - c * step is exact (c has 4 bits, step 11), and
// against half a step it decides, ties to even. (x - lo itself is exact for bf16 x and fp16 lo unless one is 2^13 times
// smaller than the other; then the difference is correctly rounded.)
DEVI int kv4_code(float x, const Kv4Group& g) {
  const float d = x - g.lo;
  float c = fminf(fmaxf(rintf(d * g.inv), 0.f), 15.f);
  const float e2 = 2.f * __fmaf_rn(-c, g.step, d);
  const bool odd = ((int)c & 1) != 0;
  if (e2 > g.step || (e2 == g.step && odd)) c += 1.f;
  if (-e2 > g.step || (-e2 == g.step && odd)) c -= 1.f;
  return g.step > 0.f ? (int)fminf(fmaxf(c, 0.f), 15.f) : 0;
}
// Largest and smallest of bf16 pairs; a NaN stays one.
DEVI uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmax2_nan(reinterpret_cast<const __nv_bfloat162&>(a), reinterpret_cast<const __nv_bfloat162&>(b));
  return reinterpret_cast<const uint32_t&>(m);
}
DEVI uint32_t min_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmin2_nan(reinterpret_cast<const __nv_bfloat162&>(a), reinterpret_cast<const __nv_bfloat162&>(b));
  return reinterpret_cast<const uint32_t&>(m);
}
// Nothing to clamp, and no NaN among what the extremes are of.
DEVI bool kv4_tame(float mn, float mx) { return mx <= KV4_LIMIT && mn >= -KV4_LIMIT; }

// N values' codes the long way, in little code: the first is taken, the rest move up (no index into registers).
template <int N, bool CLAMP>
DEVI void kv4_codes_slow(const float* v, const Kv4Group& g, uint32_t* words) {
  float x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = v[i];
  uint32_t w[N / 8];
#pragma unroll
  for (int i = 0; i < N / 8; ++i) w[i] = 0;
#pragma unroll 1
  for (int i = 0; i < N; ++i) {
    const uint32_t code = kv4_code(CLAMP ? kv4_clamp(x[0]) : x[0], g);
#pragma unroll
    for (int j = 0; j + 1 < N; ++j) x[j] = x[j + 1];
    // the words move on by four bits, a new code coming in at the top: after N of them each is in its place
#pragma unroll
    for (int j = 0; j < N / 8; ++j) w[j] = __funnelshift_r(w[j], j + 1 < N / 8 ? w[j + 1] : code, 4);
  }
#pragma unroll
  for (int i = 0; i < N / 8; ++i) words[i] = w[i];
}

// The group's pair and 8 of its values' codes, of values that are finite and within the limit, where |lo| <= 512 steps and the step
// is a normal fp16 number (else false: the caller takes kv4_code for each). Then 0 <= x - lo + step / 2 and (x - lo) / step <=
// 15.01, so nothing has to be clamped, and only a quotient within 2^-17 of a half needs the exact remainder. Adding 1.5 * 2^23
// rounds to an integer, which the sum's low bits are.
DEVI bool kv4_plain(const Kv4Group& g) { return g.step >= 6.103515625e-05f && fabsf(g.lo) <= 512.f * g.step; }
// COMPACT: that in a loop instead of straight-line code (a kernel of few warps waits for its instructions; one of many does not).
template <bool COMPACT>
DEVI uint32_t kv4_codes8(const float (&x)[8], const Kv4Group& g) {
  constexpr float MAGIC = 12582912.f;  // 0x4b400000
  uint32_t w = 0;
  float near = 0.f;
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    const float d = x[i] - g.lo, t = __fmaf_rn(d, g.inv, MAGIC);
    near = fmaxf(near, fabsf(__fmaf_rn(d, g.inv, MAGIC - t)));
    w = w * 16u + __float_as_uint(t);
  }
  w -= 0x4b400000u * 0x11111111u;
  if (near > 0.5f - 7.62939453e-06f) {
    if constexpr (COMPACT) {
      kv4_codes_slow<8, false>(x, g, &w);
    } else {
      w = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) w |= (uint32_t)kv4_code(x[i], g) << (4 * i);
    }
  }
  return w;
}
DEVI float kv4_value(int code, float step, float lo) { return __fmaf_rn((float)code, step, lo); }

}  // namespace b200dec_detail
