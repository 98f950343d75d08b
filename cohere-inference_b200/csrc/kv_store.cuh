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

// 64 values, which are one group of the 4-bit format: its codes and its pair
DEVI void store_q4_64(const float (&v)[64], uint8_t* codes, uint32_t* pair) {
  float mn = INFINITY, mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const float x = kv4_clamp(__bfloat162float(__float2bfloat16_rn(v[i])));
    mn = fminf(mn, x), mx = fmaxf(mx, x);
  }
  const Kv4Group g = kv4_group(mn, mx);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 32; ++i)
      w[i >> 3] |= (uint32_t)kv4_code(kv4_clamp(__bfloat162float(__float2bfloat16_rn(v[32 * c + i]))), g) << ((i & 7) * 4);
    *reinterpret_cast<uint4*>(codes + 16 * c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  *pair = g.word;
}

// The same for 32 values already rounded to bf16, whose vector's or group's scale is known.
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
DEVI void store_q4_32(const float (&f)[32], const Kv4Group& g, uint8_t* codes) {
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 32; ++i) w[i >> 3] |= (uint32_t)kv4_code(kv4_clamp(f[i]), g) << ((i & 7) * 4);
  *reinterpret_cast<uint4*>(codes) = make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace b200dec_detail
