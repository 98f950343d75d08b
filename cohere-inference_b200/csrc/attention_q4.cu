// Attention of one new token per row over a 4-bit slot cache (format: kv4.cuh).
//
//   score_j = step_j * (q . code_j) + lo_j * sum(q),  out = sum_j (p_j step_j) code_j + sum_j p_j lo_j,  per group of 64 dims.
//
// With 36 bytes per 64 dims the memory's share of a key is small: at the copy rate an SM has about 400 lane operations for the
// 128 values of a key and its value, which unpacking, multiplying and adding on the fp32 units take as well. So both products
// run on the tensor cores' warp instruction, m16n8k16 on fp16 operands with fp32 sums, exactly:
//   * a code in the low four bits of a half is the (subnormal) number code * 2^-24, in the next four code * 2^-20: one AND per
//     two codes makes an operand register, and the factor 16 between neighbouring dims goes into the other side;
//   * the other operand goes in as a fixed-point number cut into digits, one column of the instruction each (one query would
//     need one of its eight columns): the query as two digits of 11 bits, the weights p * step as four of 8 bits, raw bytes
//     that are subnormal halves too. Products of codes and digits are integers and so are their sums, exact in fp32 as long as
//     they stay below 2^24 (FOLD blocks); the columns are put together at the end. Nothing is rounded between the
//     fixed-point operand and that sum.
// (With a high and a low half of fp16 instead of digits the fp32 output of 24 rows of up to 32 771 keys was 8.4e-7 off, now
// 1.1e-7. e4m3 operands, on which bytes 0..15 are linear too, take a conversion per register on this chip: 1.2 times the
// instructions.) tcgen05 would need the codes as 8- or 16-bit tiles in shared memory: for a single query that staging costs
// more than the multiply.
//
// A warp takes blocks of 32 keys through a ring of its own in shared memory (cp.async, no barrier but the warp's): what is in
// flight does not sit in registers, and the next blocks come in while one is multiplied. Lane (g, t) = (lane / 4, lane % 4)
// owns key 8 t + g of the block in the softmax. Keys are the rows of the first product: lane (g, t) takes 8 bytes (16 dims) of
// the keys 8 i + g. Dims are the rows of the second: lane (g, t) takes the words of dims 8 g .. 8 g + 7 of the keys 8 t .. 8 t + 7
// and puts pairs of keys side by side; the weights' digits change places among the eight lanes of one t.
#include "kv4.cuh"

using namespace b200dec_detail;

namespace {

constexpr int NTHREADS = 128, WARPS = NTHREADS / 32, BLOCK_KEYS = 32;
constexpr int MAX_SPLITS = 128, MIN_CHUNK = 64, LONG_CHUNK = 2048;
constexpr int FOLD = 128;  // blocks of a warp after which its sums are put away: 4096 keys * 255 * 15 < 2^24
constexpr float LOWEST = -3.3e38f;  // below every finite score, and finite: the difference of two is no NaN

DEVI float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
DEVI float warp_max(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
DEVI void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
DEVI float half_lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xffff))); }
DEVI float half_hi(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }
template <int D>
struct Ring {
  static constexpr int G = D / 64, STAGES = D == 64 ? 3 : 2, CODES = BLOCK_KEYS * D / 2, PAIRS = BLOCK_KEYS * G * 4;
  static constexpr int STAGE = 2 * CODES + 2 * PAIRS, BYTES = WARPS * STAGES * STAGE;
};
// 4 or 8 bytes
template <int N>
DEVI void cp_async_small(void* smem, const void* gmem) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_addr_u32(smem)), "l"(gmem), "n"(N) : "memory");
}

constexpr uint32_t EVEN = 0x000f000fu, ODD = 0x00f000f0u;
constexpr float TWO24 = 16777216.f, TWO48 = TWO24 * TWO24;

// Among the eight lanes g of one t, each with a word of four digits (bytes): the digits g % 4 of the lanes 0-3 in x, of the
// lanes 4-7 in y.
DEVI void turn_digits(uint32_t w, int g, uint32_t& x, uint32_t& y) {
  uint32_t p = __shfl_xor_sync(0xffffffffu, w, 8);
  w = __byte_perm(w, p, (g & 2) ? 0x3276u : 0x5410u);  // own half first where g's bit is clear, last where it is set
  p = __shfl_xor_sync(0xffffffffu, w, 4);
  w = __byte_perm(w, p, (g & 1) ? 0x3715u : 0x6240u);
  p = __shfl_xor_sync(0xffffffffu, w, 16);
  x = (g & 4) ? p : w, y = (g & 4) ? w : p;
}

struct Q4Args {
  const int* active;
  const float* q;  // (rows, ldq)
  uint8_t* k;      // (slots + 1, H, cap, D / 2)
  uint8_t* v;
  uint32_t* km;    // (slots + 1, H, cap, D / 64) {step, lo}
  uint32_t* vm;
  const int* n;
  const int* sched;
  void* out;
  float* part;
  int* count;
  int* status;
  int ldq, H, cap, slots, out_kind, chunk;
  float scale_log2;
};

// 2^(bits - 1 - e) for a largest magnitude of 2^e or more and less than 2^(e + 1): the factor to a fixed-point number below
// 2^bits. A power of two; the exponent is kept where the factor and what is divided by it stay normal.
DEVI float to_fixed(float amax, int bits) {
  const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -90), 100);
  return amax > 0.f ? __uint_as_float((uint32_t)(126 + bits - e) << 23) : 1.f;
}

// The row's new key or value (a warp, D / 32 dims a lane): rounded to bf16, its codes and pairs into the cache, its bf16
// values into x.
template <int D>
DEVI void append(const float* src, uint8_t* codes, uint32_t* pairs, int lane, float (&x)[D / 32]) {
  constexpr int N = D / 32;
  float mn = INFINITY, mx = -INFINITY, y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = __bfloat162float(__float2bfloat16_rn(__ldcg(src + lane * N + i)));
    y[i] = kv4_clamp(x[i]);
    mn = fminf(mn, y[i]), mx = fmaxf(mx, y[i]);
  }
#pragma unroll
  for (int o = 1; o < 64 / N; o <<= 1) {
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  const Kv4Group g = kv4_group(mn, mx);
#pragma unroll
  for (int i = 0; i < N; i += 2)
    codes[(lane * N + i) / 2] = (uint8_t)(kv4_code(y[i], g) | (kv4_code(y[i + 1], g) << 4));
  if (lane % (64 / N) == 0) pairs[lane * N / 64] = g.word;
}

// WPI: warps of a (row, head); a CTA takes 4 / WPI neighbouring heads of a row.
template <int D, bool SELF, int WPI>
__global__ void __launch_bounds__(NTHREADS) attention_q4_kernel(const Q4Args p) {
  constexpr int G = D / 64, ITEMS = WARPS / WPI, SETS = WARPS + ITEMS;  // groups of a vector; partial sets: the warps' and the new keys'
  __shared__ float s_m[SETS], s_l[SETS], s_acc[SETS][D];
  __shared__ int s_last[ITEMS];
  __shared__ __align__(16) __half s_q[ITEMS][2][D];  // the queries' digits
  __shared__ float s_sum[ITEMS][3][D / 32];          // of 32 dims each: the query, its high and its low digits
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int it = warp / WPI, wi = warp % WPI, gt = wi * 32 + lane;  // the warp's item in the CTA, its place there, the thread's
  const bool live = (int)blockIdx.y * ITEMS + it < p.H;             // the last CTA of a row may have heads to spare
  const int h = min((int)blockIdx.y * ITEMS + it, p.H - 1);
  pdl_wait();

  // the row, its slot and its number of cached keys; out of range: clamped and reported
  int r, s, n;
  if (p.sched) {
    const int4 e = __ldcg(reinterpret_cast<const int4*>(p.sched) + blockIdx.z);
    r = e.x, s = e.y, n = e.z;
  } else {
    r = blockIdx.z;
  }
  const float* qrow = p.q + (size_t)r * p.ldq + h * D;
  float x[D / 32];  // the query does not depend on the slot: on its way first
#pragma unroll
  for (int i = 0; i < D / 32; ++i) x[i] = __ldcg(qrow + 32 * i + lane);
  if (!p.sched) {
    s = p.active[r];
    const bool report = tid == 0 && blockIdx.y == 0 && blockIdx.x == 0;
    if (s < 0 || s > p.slots) {
      if (report) atomicOr(p.status, B200DEC_ST_SLOT_RANGE);
      s = p.slots;
    }
    n = p.n[s];
    const int most = SELF ? p.cap - 1 : p.cap;
    if (n < 0 || n > most) {
      if (report) atomicOr(p.status, SELF ? B200DEC_ST_POS_RANGE : B200DEC_ST_FRAMES_RANGE);
      n = max(0, min(n, most));
    }
  }
  const int chunks = max(1, (n + p.chunk - 1) / p.chunk);
  if ((int)blockIdx.x >= chunks) return;
  const int start = blockIdx.x * p.chunk, end = live ? min(n, start + p.chunk) : start;
  const bool with_new = SELF && blockIdx.x == 0;
  const size_t vec0 = ((size_t)s * p.H + h) * p.cap;

  // this warp's ring: a stage is a block's key codes, value codes, key pairs, value pairs
  using R = Ring<D>;
  extern __shared__ __align__(16) uint8_t dyn_smem[];
  uint8_t* ring = dyn_smem + warp * R::STAGES * R::STAGE;
  const int first = start + wi * BLOCK_KEYS, stride = WPI * BLOCK_KEYS;
  // Keys lie in a stage as they come; values in rows 4 (key % 8) + key / 8, so that the four t of a step read neighbouring rows.
  // Vectors of 64 bytes have their halves swapped where bit 1 of the row is set: then no bank is asked for twice either.
  constexpr int PARTS = D / 32, KEYS = 32 / PARTS;  // 16-byte pieces of a vector; keys of a warp-wide copy
  const int key = lane / PARTS, piece = lane % PARTS;
  const uint8_t* kc = p.k + (vec0 + first) * (D / 2) + 16 * lane;
  const uint8_t* vc = p.v + (vec0 + first) * (D / 2) + 16 * lane;
  const uint32_t* kp_at = p.km + (vec0 + first + lane) * G;
  const uint32_t* vp_at = p.vm + (vec0 + first + lane) * G;
  const int k_to = key * (D / 2) + 16 * (D == 128 ? piece ^ (key & 2) : piece);
  const int v_to = ((key & 7) * 4 + (key >> 3)) * (D / 2);
  const auto fetch = [&](int i) {  // block i of this warp, called in order; what lies past the end is not fetched, and counts for nothing
    const int left = end - (first + i * stride);
    uint8_t* st = ring + i % R::STAGES * R::STAGE;
#pragma unroll
    for (int j = 0; j < PARTS; ++j)
      if (key + KEYS * j < left) {
        // row of the value: KEYS j / 8 further; its bit 1 is that of j where vectors have 64 bytes
        cp_async16(st + k_to + j * 512, kc + j * 512);
        cp_async16(st + R::CODES + v_to + KEYS * j / 8 * (D / 2) + 16 * (D == 128 ? piece ^ (j & 2) : piece), vc + j * 512);
      }
    if (lane < left) {
      cp_async_small<4 * G>(st + 2 * R::CODES + lane * 4 * G, kp_at);
      cp_async_small<4 * G>(st + 2 * R::CODES + R::PAIRS + lane * 4 * G, vp_at);
    }
    kc += stride * (D / 2), vc += stride * (D / 2), kp_at += stride * G, vp_at += stride * G;
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < R::STAGES - 1; ++i) fetch(i);  // before anything waits for the query

  // The query in log2 units as the first product's B operand: a fixed-point number of 22 bits, its high digit in the even
  // columns and its low one in the odd. Register b of step ks holds two dims of the lane's word ks / 2: those whose codes are in
  // bits 0-3 (b = 0) or 4-7 (b = 1) of its low (ks even) or high byte pair. The CTA cuts it up once, a dim per thread, in that
  // order. A code's part of a score is taken relative to 7.5, the middle of the codes: `off` is what 7.5 for every code would
  // add, taken off before anything rounds.
  uint32_t qb[G][4][2];
  float qsum[G], off_hi[G], off_lo[G], unit;
  {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) amax = fmaxf(amax, fabsf(x[i]));
    amax = warp_max(amax) * fabsf(p.scale_log2);
    const float f = to_fixed(amax, 22);
    unit = TWO24 / f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      if (i % WPI != wi) continue;
      const int d = 32 * i + lane, at = (d & ~7) + 2 * (d & 3) + ((d >> 2) & 1);  // dims d and d + 4 of a word side by side
      const float v = rintf(x[i] * p.scale_log2 * f);                             // |v| <= 2^22
      const float hi = rintf(v * 0.00048828125f), lo = v - 2048.f * hi;           // |hi| <= 2^11, |lo| <= 2^10
      const float sc = (d & 1) ? 0.0625f : 1.f;
      s_q[it][0][at] = __float2half_rn(hi * sc), s_q[it][1][at] = __float2half_rn(lo * sc);
      const float s0 = warp_sum(x[i]), s1 = warp_sum(hi), s2 = warp_sum(lo);
      if (lane == 0) s_sum[it][0][i] = s0, s_sum[it][1][i] = s1, s_sum[it][2][i] = s2;
    }
    if constexpr (WPI == 1) __syncwarp();
    else __syncthreads();
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      qsum[gr] = (s_sum[it][0][2 * gr] + s_sum[it][0][2 * gr + 1]) * p.scale_log2;
      off_hi[gr] = (s_sum[it][1][2 * gr] + s_sum[it][1][2 * gr + 1]) * (7.5f / TWO24);
      off_lo[gr] = (s_sum[it][2][2 * gr] + s_sum[it][2][2 * gr + 1]) * (7.5f / TWO24);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint4 q = *reinterpret_cast<const uint4*>(&s_q[it][g & 1][64 * gr + 16 * t + 8 * w]);
        qb[gr][2 * w][0] = q.x, qb[gr][2 * w][1] = q.y, qb[gr][2 * w + 1][0] = q.z, qb[gr][2 * w + 1][1] = q.w;
      }
    }
  }

  float m = LOWEST, l = 0.f, acc[G][4][4], lo_sum[G], vf[G];
  uint32_t vtop[G];  // bits of the largest value step so far, a power of two: the weights are scaled by vf = 2^31 / it
#pragma unroll
  for (int gr = 0; gr < G; ++gr) {
    lo_sum[gr] = 0.f, vtop[gr] = 0, vf[gr] = 1.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[gr][i][c] = 0.f;
  }

  // The warp's (max, sum, output) set in shared memory: what it has so far, added to what is there already; and a new start.
  bool folded = false;
  const auto fold = [&] {
    const float sum = warp_sum(l), top = folded ? fmaxf(s_m[warp], m) : m;
    const float was = folded ? ex2(s_m[warp] - top) : 0.f, now = ex2(m - top), l0 = folded ? s_l[warp] : 0.f;
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      // columns 2 t and 2 t + 1 are the digits 0, 1 (t even) or 2, 3: units of 2^-48 times 256^digit
      const float add = warp_sum(lo_sum[gr]), u0 = TWO48 / vf[gr] * ((t & 1) ? 65536.f : 1.f), u1 = 256.f * u0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float a = acc[gr][j][0] * u0 + acc[gr][j][1] * u1, b = (acc[gr][j][2] * u0 + acc[gr][j][3] * u1) * 0.0625f;
        a += __shfl_xor_sync(0xffffffffu, a, 1), b += __shfl_xor_sync(0xffffffffu, b, 1);
        if (t == j) {
          float* o = &s_acc[warp][64 * gr + 8 * g + 2 * j];
          o[0] = (a + add) * now + (folded ? o[0] * was : 0.f), o[1] = (b + add) * now + (folded ? o[1] * was : 0.f);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[gr][j][c] = 0.f;
      }
      lo_sum[gr] = 0.f;
    }
    __syncwarp();  // every lane has read the set's maximum and sum
    if (lane == 0) s_m[warp] = top, s_l[warp] = sum * now + l0 * was;
    __syncwarp();
    l = 0.f, m = LOWEST, folded = true;
  };
  for (int i = 0, k0 = first; k0 < end; ++i, k0 += stride) {
    cp_async_wait_group<R::STAGES - 2>();
    __syncwarp();  // the other lanes' pieces are there, and everyone is done with the stage that is filled next
    fetch(i + R::STAGES - 1);
    const uint8_t* st = ring + i % R::STAGES * R::STAGE;
    const int own = 8 * t + g;
    const bool ok = k0 + own < end;
    uint32_t kp[G], vp[G];
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      kp[gr] = reinterpret_cast<const uint32_t*>(st + 2 * R::CODES)[own * G + gr];
      vp[gr] = ok ? reinterpret_cast<const uint32_t*>(st + 2 * R::CODES + R::PAIRS)[own * G + gr] : 0;
    }

    // scores: two tiles of 16 keys per group
    float sc = 0.f;
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      float c[2][4] = {};
#pragma unroll
      for (int pr = 0; pr < 2; ++pr) {
        const int at = (16 * pr + g) * (D / 2) + 32 * (D == 128 ? gr ^ ((g >> 1) & 1) : gr) + 8 * t;
        const uint2 lo = *reinterpret_cast<const uint2*>(st + at), hi = *reinterpret_cast<const uint2*>(st + at + 8 * (D / 2));
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          uint32_t a = ks < 2 ? lo.x : lo.y, b = ks < 2 ? hi.x : hi.y;
          if (ks & 1) a >>= 8, b >>= 8;
          mma16816(c[pr], a & EVEN, b & EVEN, a & ODD, b & ODD, qb[gr][ks][0], qb[gr][ks][1]);
        }
      }
      const float h0 = (t & 1) ? c[0][2] : c[0][0], h1 = (t & 1) ? c[1][2] : c[1][0];
      const float l0 = (t & 1) ? c[0][3] : c[0][1], l1 = (t & 1) ? c[1][3] : c[1][1];
      const float dot = __fmaf_rn(2048.f, ((t & 2) ? h1 : h0) - off_hi[gr], ((t & 2) ? l1 : l0) - off_lo[gr]);
      const float step = half_lo(kp[gr]);
      sc += step * (unit * dot) + __fmaf_rn(7.5f, step, half_hi(kp[gr])) * qsum[gr];
    }
    sc = ok ? sc : -INFINITY;

    // the warp's running maximum, and the range of the weights p * step; both warp-uniform
    const float top = warp_max(sc);
    bool raise = top > m;
    uint32_t vt[G];
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      vt[gr] = __reduce_max_sync(0xffffffffu, __float_as_uint(half_lo(vp[gr])) & 0x7f800000u);
      raise |= vt[gr] > vtop[gr];
    }
    if (raise) {
      // the reference is a whole number, so that the sums are scaled by powers of two and stay what they are
      const float mn = fmaxf(m, ceilf(top)), a = ex2(m - mn);
      m = mn, l *= a;
#pragma unroll
      for (int gr = 0; gr < G; ++gr) {
        float f = a;
        if (vt[gr] > vtop[gr]) {
          const float now = to_fixed(__uint_as_float(vt[gr]), 32);
          f *= vtop[gr] ? now / vf[gr] : 0.f;  // nothing but zeros was added before the first step above zero
          vtop[gr] = vt[gr], vf[gr] = now;
        }
        lo_sum[gr] *= a;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[gr][i][c] *= f;
      }
    }
    const float e = ex2(sc - m);
    l += e;
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      lo_sum[gr] += e * half_hi(vp[gr]);
      uint32_t x, y;  // the weights' digits g % 4, of the keys 8 t + 0..3 and 8 t + 4..7
      turn_digits(__float2uint_rn(e * half_lo(vp[gr]) * vf[gr]), g, x, y);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const uint32_t d = ks ? y : x, b0 = __byte_perm(d, 0, 0x4140), b1 = __byte_perm(d, 0, 0x4342);
        const uint8_t* vs = st + R::CODES + (16 * ks + t) * (D / 2) + 4 * g + 32 * (D == 128 ? gr ^ ((t >> 1) & 1) : gr);
        const auto word = [&](int j) { return *reinterpret_cast<const uint32_t*>(vs + 4 * j * (D / 2)); };
        const uint32_t v0 = word(0), v1 = word(1), v2 = word(2), v3 = word(3);
        // bytes 0, 1 then 2, 3 of a key pair side by side: dims 0-3 and 4-7 of the lane's eight
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const uint32_t u = __byte_perm(v0, v1, hf ? 0x7632u : 0x5410u), v = __byte_perm(v2, v3, hf ? 0x7632u : 0x5410u);
          mma16816(acc[gr][2 * hf], u & EVEN, u & ODD, v & EVEN, v & ODD, b0, b1);
          mma16816(acc[gr][2 * hf + 1], u >> 8 & EVEN, u >> 8 & ODD, v >> 8 & EVEN, v >> 8 & ODD, b0, b1);
        }
      }
    }
    if (i % FOLD == FOLD - 1) fold();
  }
  fold();

  if (SELF && with_new && live) {
    // the new key and value, each by a warp where there are two: into the cache, and as a set of their own with the bf16 values
    constexpr int N = D / 32;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      if (kv % WPI != wi) continue;
      float y[N];
      append<D>(qrow + (size_t)(1 + kv) * p.H * D, (kv ? p.v : p.k) + (vec0 + n) * (D / 2), (kv ? p.vm : p.km) + (vec0 + n) * G, lane, y);
      if (kv == 0) {
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) d += __ldcg(qrow + lane * N + i) * y[i];
        d = warp_sum(d) * p.scale_log2;
        if (lane == 0) s_m[WARPS + it] = d, s_l[WARPS + it] = 1.f;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) s_acc[WARPS + it][lane * N + i] = y[i];
      }
    }
  }
  pdl_trigger();  // late: a grid that started earlier would take registers from the stream
  if constexpr (WPI == 1) __syncwarp();
  else __syncthreads();
  // the item's sets: dims gt, gt + 32 WPI, ... of its threads
  constexpr int ND = (D + 32 * WPI - 1) / (32 * WPI);
  float M = LOWEST, L = 0.f, O[ND] = {};
  {
    const int sets = with_new ? WPI + 1 : WPI;
    const auto set = [&](int i) { return i < WPI ? it * WPI + i : WARPS + it; };
    for (int i = 0; i < sets; ++i) M = fmaxf(M, s_m[set(i)]);
    for (int i = 0; i < sets; ++i) {
      const float w = ex2(s_m[set(i)] - M);
      L += w * s_l[set(i)];
#pragma unroll
      for (int k = 0; k < ND; ++k)
        if (gt + 32 * WPI * k < D) O[k] += w * s_acc[set(i)][gt + 32 * WPI * k];
    }
  }
  const auto store = [&](const float (&o)[ND], float sum) {
#pragma unroll
    for (int k = 0; k < ND; ++k) {
      const int d = gt + 32 * WPI * k;
      if (d >= D || !live) continue;
      const float val = sum > 0.f || sum != sum ? o[k] / sum : 0.f;  // no key at all: zeros
      const size_t at = ((size_t)r * p.H + h) * D + d;
      if (p.out_kind == B200DEC_OUT_F16) reinterpret_cast<__half*>(p.out)[at] = __float2half_rn(clamp_h(val));
      else reinterpret_cast<float*>(p.out)[at] = val;
    }
  };
  if (chunks == 1) {
    store(O, L);
    return;
  }
  // a row in several chunks: partials to the workspace, the last CTA of the (row, head) to arrive merges them
  const int item = r * p.H + h;
  if (live) {
    float* part = p.part + ((size_t)item * gridDim.x + blockIdx.x) * (D + 2);
#pragma unroll
    for (int k = 0; k < ND; ++k)
      if (gt + 32 * WPI * k < D) part[gt + 32 * WPI * k] = O[k];
    if (gt == 0) part[D] = M, part[D + 1] = L;
  }
  __threadfence();
  __syncthreads();
  if (gt == 0) s_last[it] = live && atomicAdd(p.count + item, 1) == chunks - 1;
  __syncthreads();
  if (!s_last[it]) return;
  __threadfence();
  const float* pb = p.part + (size_t)item * gridDim.x * (D + 2);
  M = LOWEST, L = 0.f;
  for (int i = 0; i < chunks; ++i) M = fmaxf(M, __ldcg(pb + i * (D + 2) + D));
#pragma unroll
  for (int k = 0; k < ND; ++k) O[k] = 0.f;
  for (int i = 0; i < chunks; ++i) {
    const float w = ex2(__ldcg(pb + i * (D + 2) + D) - M);
    L += w * __ldcg(pb + i * (D + 2) + D + 1);
#pragma unroll
    for (int k = 0; k < ND; ++k)
      if (gt + 32 * WPI * k < D) O[k] += w * __ldcg(pb + i * (D + 2) + gt + 32 * WPI * k);
  }
  store(O, L);
  if (gt == 0) p.count[item] = 0;
}

template <int D, bool SELF, int WPI>
cudaError_t launch_wpi(int splits, int rows, cudaStream_t st, int pdl, const Q4Args& p) {
  static_assert(Ring<D>::BYTES <= 40 * 1024, "with the static arrays below 48 KB: no attribute to set");
  const dim3 grid(splits, (p.H + WARPS / WPI - 1) / (WARPS / WPI), rows);
  return launch_kernel(attention_q4_kernel<D, SELF, WPI>, grid, dim3(NTHREADS), Ring<D>::BYTES, st, 0, pdl, p);
}

template <int D, bool SELF>
cudaError_t launch_q4(int splits, int rows, cudaStream_t st, int pdl, const Q4Args& p) {
  // Warps of a (row, head). Many short rows are bound by what every item costs before and after its keys (query, merge), which
  // fewer warps share; long rows and few ones by what is in flight. us with 1 / 2 / 4 warps: 2048 items of 0-457 keys (64 dims)
  // 19.0 / 20.4 / 25.8, 1024 of 50-375 keys 10.7 / 10.1 / 12.3, 8 items of 217 keys (128 dims) 10.7 / 9.5 / 8.4, 192 items of
  // up to 32 771 keys (128 dims, in chunks) 135 / 104 / 97.
  const int64_t items = (int64_t)rows * p.H;
  const int wpi = splits > 1 || p.cap > 2048 || items < 512 ? 4 : items < 1400 || p.cap > 1024 ? 2 : 1;
  if (wpi == 1) return launch_wpi<D, SELF, 1>(splits, rows, st, pdl, p);
  if (wpi == 2) return launch_wpi<D, SELF, 2>(splits, rows, st, pdl, p);
  return launch_wpi<D, SELF, 4>(splits, rows, st, pdl, p);
}

// CTAs a (row, head) may be cut into over a cache of cap keys: enough for every SM to hold several, and on a long axis as many
// as keep a CTA at LONG_CHUNK keys, so that rows of unlike lengths even out
int q4_splits(int rows, int heads, int cap) {
  const int64_t items = (int64_t)rows * heads;
  int64_t s = (4 * 148 + items - 1) / items;
  if (s < cap / LONG_CHUNK) s = cap / LONG_CHUNK;
  if (s > cap / MIN_CHUNK) s = cap / MIN_CHUNK;
  return (int)(s < 1 ? 1 : s > MAX_SPLITS ? MAX_SPLITS : s);
}

}  // namespace

extern "C" {

int64_t b200dec_attention_q4_scratch_floats(int rows, int heads, int head_dim, int cap) {
  if (rows < 1 || heads < 1 || head_dim < 1 || cap < 1) return 0;
  return (int64_t)rows * heads * q4_splits(rows, heads, cap) * (head_dim + 2);
}

int b200dec_attention_q4(int self, const int32_t* active, const float* q, int ldq, void* kcache, void* vcache, void* kpairs,
                         void* vpairs, const int32_t* n, const int32_t* sched, int slots, int heads, int head_dim, int cap,
                         float scale, void* out, int out_kind, int rows, float* part, int32_t* count, int32_t* status, int pdl,
                         void* stream) {
  B200_REQUIRE(q && kcache && vcache && kpairs && vpairs && out && (sched || (active && n && status)), "attention_q4: null pointer");
  B200_REQUIRE((part == nullptr) == (count == nullptr), "attention_q4: the workspace and its counters go together");
  B200_REQUIRE(head_dim == 64 || head_dim == 128, "attention_q4: head_dim %d (64 or 128)", head_dim);
  B200_REQUIRE(rows >= 1 && rows <= 65535 && heads >= 1 && heads <= 65535 && cap >= 1 && cap <= 1 << 30 && slots >= 0,
               "attention_q4: rows %d heads %d cap %d slots %d", rows, heads, cap, slots);
  B200_REQUIRE((int64_t)rows * heads <= 1 << 26, "attention_q4: %d rows x %d heads", rows, heads);
  B200_REQUIRE(ldq >= (self ? 3 : 1) * heads * head_dim && ldq % 4 == 0 && ((uintptr_t)q & 15) == 0,
               "attention_q4: ldq %d (rows of %d floats, 16-byte aligned)", ldq, (self ? 3 : 1) * heads * head_dim);
  B200_REQUIRE((((uintptr_t)kcache | (uintptr_t)vcache) & 15) == 0 && ((uintptr_t)kpairs | (uintptr_t)vpairs) % (head_dim / 16) == 0 &&
                   (!sched || ((uintptr_t)sched & 15) == 0), "attention_q4: alignment");
  B200_REQUIRE(out_kind == B200DEC_OUT_F16 || out_kind == B200DEC_OUT_F32, "attention_q4: out_kind %d", out_kind);
  B200_REQUIRE((uintptr_t)out % (out_kind == B200DEC_OUT_F16 ? 2 : 4) == 0, "attention_q4: alignment of out");
  Q4Args p{active, q, (uint8_t*)kcache, (uint8_t*)vcache, (uint32_t*)kpairs, (uint32_t*)vpairs, n, sched, out, part, count, status,
           ldq, heads, cap, slots, out_kind, cap, scale * 1.4426950408889634f};
  const int splits = part ? q4_splits(rows, heads, cap) : 1;
  p.chunk = ((cap + splits - 1) / splits + BLOCK_KEYS - 1) / BLOCK_KEYS * BLOCK_KEYS;
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = head_dim == 64 ? self ? launch_q4<64, true>(splits, rows, st, pdl, p) : launch_q4<64, false>(splits, rows, st, pdl, p)
                        : self ? launch_q4<128, true>(splits, rows, st, pdl, p) : launch_q4<128, false>(splits, rows, st, pdl, p);
  if (e != cudaSuccess) return fail(B200DEC_ECUDA, "attention_q4 launch: %s", cudaGetErrorString(e));
  return 0;
}

}  // extern "C"
