// Stores of a head vector's values into int8 and 4-bit slot caches, from a thread that holds 64 of them (the epilogues of
// prefill_gemm.cu and w8a8.cu).
#pragma once
#include "kv4.cuh"

namespace b200dec_detail {

// the reference's int8 cache format for 64 values already rounded to bf16, given the vector's absmax
DEVI void store_q8_64(const float (&f)[64], float mx, int8_t* dst) {
  const float sc = mx > 0.f ? __fdiv_rn(mx, 127.f) : 1.f, inv = __fdiv_rn(1.f, sc);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int q = __float2int_rn(fminf(fmaxf(__fmul_rn(f[16 * c + i], inv), -127.f), 127.f));
      w[i >> 2] |= (uint32_t)(q & 0xff) << ((i & 3) * 8);
    }
    *reinterpret_cast<uint4*>(dst + 16 * c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// 4 bits. The extremes of 32 values after rounding to bf16, on top of those in hi and lo (pairs; `first`: there are none yet).
DEVI void extremes_32(const float* v, bool first, uint32_t& hi, uint32_t& lo) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    const uint32_t w = pack_bf16(v[i], v[i + 1]);
    hi = first && i == 0 ? w : max_bf16x2(hi, w), lo = first && i == 0 ? w : min_bf16x2(lo, w);
  }
}
DEVI void extremes_of(uint32_t hi, uint32_t lo, float& mn, float& mx) {
  // a NaN in either half has to come through
  const uint32_t m = max_bf16x2(hi, hi >> 16 | hi << 16), n = min_bf16x2(lo, lo >> 16 | lo << 16);
  mx = bf16_lo(m), mn = bf16_lo(n);
}
// ... and with the clamp, where that is needed
DEVI void extremes_32_clamped(const float* v, float& mn, float& mx) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float x = kv4_clamp(__bfloat162float(__float2bfloat16_rn(v[i])));
    mn = fminf(mn, x), mx = fmaxf(mx, x);
  }
}
// the codes of 32 values of a group; tame: its values need no clamp
DEVI void store_q4_32(const float* v, const Kv4Group& g, bool tame, uint8_t* codes) {
  uint32_t w[4] = {0, 0, 0, 0};
  if (tame && kv4_plain(g)) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const uint32_t b = pack_bf16(v[8 * c + i], v[8 * c + i + 1]);
        x[i] = bf16_lo(b), x[i + 1] = bf16_hi(b);
      }
      w[c] = kv4_codes8<true>(x, g);
    }
  } else {
    float x[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = __bfloat162float(__float2bfloat16_rn(v[i]));
    kv4_codes_slow<32, true>(x, g, w);
  }
  *reinterpret_cast<uint4*>(codes) = make_uint4(w[0], w[1], w[2], w[3]);
}
// int8 for 32 values already rounded to bf16, whose vector's scale is known.
DEVI void store_q8_32(const float (&f)[32], float inv, int8_t* dst) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int q = __float2int_rn(fminf(fmaxf(__fmul_rn(f[16 * c + i], inv), -127.f), 127.f));
      w[i >> 2] |= (uint32_t)(q & 0xff) << ((i & 3) * 8);
    }
    *reinterpret_cast<uint4*>(dst + 16 * c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
}  // namespace b200dec_detail
