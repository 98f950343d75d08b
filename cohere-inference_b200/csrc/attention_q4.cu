// Attention of one new token per row over a 4-bit slot cache (format: kv4.cuh).
//
// With 36 bytes per 64 dims the memory's share of a key is small, and a kernel that unpacks and multiplies on the fp32 units
// spends more time on instructions than the memory needs (about 400 lane operations per key of 64 dims are there per key at
// the copy rate; unpacking, multiplying and adding 128 values takes as many). So both products run on the tensor cores' warp
// instruction (m16n8k16, fp16 in, fp32 out), whose operands come out of the packed words nearly for free: a nibble in
// bits 0-3 of a half is the number code * 2^-24, one in bits 4-7 is code * 2^-20, both exact (subnormal) halves, so one AND
// per two values makes an operand register. One query per row would leave seven of the eight columns idle; instead the
// even columns hold the high half of an fp32 operand and the odd ones the low half (x = hi + lo to 22 bits), so scores and
// outputs keep fp32's accuracy and nothing is rounded to 16 bits. tcgen05 would need the codes as 8 or 16-bit
// tiles in shared memory: for a single query that staging costs more than the multiply.
//
// score_j = step_j * (q . code_j) + lo_j * sum(q),  out = sum_j (p_j step_j) code_j + sum_j p_j lo_j,  per group of 64 dims.
//
// A warp takes blocks of 32 keys; lane (g, t) = (lane / 4, lane % 4) owns key 8 t + g of the block in the softmax. Keys are
// the rows of the first product: lane (g, t) loads 8 bytes (16 dims) of the keys 8 i + g. Dims are the rows of the second:
// lane (g, t) loads the words of dims 8 g .. 8 g + 7 of the keys t + 4 i, and pairs of keys are merged byte by byte.
#include "kv4.cuh"

using namespace b200dec_detail;

namespace {

constexpr int NTHREADS = 128, WARPS = NTHREADS / 32, BLOCK_KEYS = 32;
constexpr int MAX_SPLITS = 128, MIN_CHUNK = 64, LONG_CHUNK = 1024;
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
DEVI uint32_t pack_halves(__half a, __half b) { return (uint32_t)__half_as_ushort(a) | ((uint32_t)__half_as_ushort(b) << 16); }

constexpr uint32_t EVEN = 0x000f000fu, ODD = 0x00f000f0u;
constexpr float TWO24 = 16777216.f;

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

// 2^(12 - e) for a largest magnitude of 2^e: the operand then lies in fp16's upper range, its low half included. Powers of two
// only; the exponent is kept where both the factor and its use as a divisor stay normal.
DEVI float to_fp16_range(float amax) {
  const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -100), 100);
  return amax > 0.f ? __uint_as_float((uint32_t)(127 + 12 - e) << 23) : 1.f;
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

template <int D, bool SELF>
__global__ void __launch_bounds__(NTHREADS) attention_q4_kernel(const Q4Args p) {
  constexpr int G = D / 64, SETS = WARPS + 1;  // groups of a vector; partial sets: the warps' and the new key's
  __shared__ float s_m[SETS], s_l[SETS], s_acc[SETS][D];
  __shared__ int s_last;
  const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  pdl_wait();

  // the row, its slot and its number of cached keys; out of range: clamped and reported
  int r, s, n;
  if (p.sched) {
    const int4 e = __ldcg(reinterpret_cast<const int4*>(p.sched) + blockIdx.z);
    r = e.x, s = e.y, n = e.z;
  } else {
    r = blockIdx.z, s = p.active[r];
    const bool report = tid == 0 && h == 0 && blockIdx.x == 0;
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
  const int start = blockIdx.x * p.chunk, end = min(n, start + p.chunk);
  const bool with_new = SELF && blockIdx.x == 0;
  const size_t vec0 = ((size_t)s * p.H + h) * p.cap;
  const float* qrow = p.q + (size_t)r * p.ldq + h * D;

  // the query in log2 units as the first product's B operand: register b of k-step ks of a group holds two dims of the
  // lane's word ks / 2, those in bits 0-3 (b = 0) or 4-7 (b = 1) of its low (ks even) or high byte pair
  uint32_t qb[G][4][2];
  float unscale, qsum[G];
  {
    float amax = 0.f;
    for (int d = lane; d < D; d += 32) amax = fmaxf(amax, fabsf(__ldcg(qrow + d)));
    amax = warp_max(amax) * fabsf(p.scale_log2);
    const float f = to_fp16_range(amax), to = f * p.scale_log2;
    unscale = TWO24 / f;
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      float x[16], sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 a = ld_cg_f4(qrow + 64 * gr + 16 * t + 4 * i);
        x[4 * i] = a.x, x[4 * i + 1] = a.y, x[4 * i + 2] = a.z, x[4 * i + 3] = a.w;
        sum += (a.x + a.y) + (a.z + a.w);
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      qsum[gr] = sum * p.scale_log2;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int d = 8 * (ks >> 1) + 2 * (ks & 1) + b;  // nibbles d % 8 and d % 8 + 4 of the word
          const float u = x[d] * to * (b ? 0.0625f : 1.f), w = x[d + 4] * to * (b ? 0.0625f : 1.f);
          const __half uh = __float2half_rn(u), wh = __float2half_rn(w);
          const __half ul = __float2half_rn(u - __half2float(uh)), wl = __float2half_rn(w - __half2float(wh));
          qb[gr][ks][b] = (g & 1) ? pack_halves(ul, wl) : pack_halves(uh, wh);
        }
    }
  }

  float m = LOWEST, l = 0.f, acc[G][4][4], lo_sum[G], vf[G];
  uint32_t vtop[G];  // bits of the largest value step so far, a power of two: the weights are scaled by vf = 2^14 / it
#pragma unroll
  for (int gr = 0; gr < G; ++gr) {
    lo_sum[gr] = 0.f, vtop[gr] = 0, vf[gr] = 1.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[gr][i][c] = 0.f;
  }

  const uint8_t* kb = p.k + vec0 * (D / 2) + 8 * t;
  const uint8_t* vb = p.v + vec0 * (D / 2) + 4 * g;
  for (int k0 = start + warp * BLOCK_KEYS; k0 < end; k0 += WARPS * BLOCK_KEYS) {
    // everything the block needs, before any of it is used
    uint2 kw[4][G];
    uint32_t vw[8][G], kp[G], vp[G];
    const int own = k0 + 8 * t + g;
    const bool ok = own < end;
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      kp[gr] = ok ? ld_stream4(p.km + (vec0 + own) * G + gr) : 0;
      vp[gr] = ok ? ld_stream4(p.vm + (vec0 + own) * G + gr) : 0;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int gr = 0; gr < G; ++gr)
        kw[i][gr] = k0 + 8 * i + g < end ? ld_stream8(kb + (size_t)(k0 + 8 * i + g) * (D / 2) + 32 * gr) : make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int gr = 0; gr < G; ++gr)
        vw[i][gr] = k0 + 4 * i + t < end ? ld_stream4(vb + (size_t)(k0 + 4 * i + t) * (D / 2) + 32 * gr) : 0;

    // scores: two tiles of 16 keys per group
    float sc = 0.f;
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      float c[2][4] = {};
#pragma unroll
      for (int pr = 0; pr < 2; ++pr)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const uint2 lo = kw[2 * pr][gr], hi = kw[2 * pr + 1][gr];
          uint32_t a = ks < 2 ? lo.x : lo.y, b = ks < 2 ? hi.x : hi.y;
          if (ks & 1) a >>= 8, b >>= 8;
          mma16816(c[pr], a & EVEN, b & EVEN, a & ODD, b & ODD, qb[gr][ks][0], qb[gr][ks][1]);
        }
      const float d0 = (t & 1) ? c[0][2] + c[0][3] : c[0][0] + c[0][1];
      const float d1 = (t & 1) ? c[1][2] + c[1][3] : c[1][0] + c[1][1];
      sc += half_lo(kp[gr]) * (unscale * ((t & 2) ? d1 : d0)) + half_hi(kp[gr]) * qsum[gr];
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
      const float mn = fmaxf(m, top), a = ex2(m - mn);
      m = mn, l *= a;
#pragma unroll
      for (int gr = 0; gr < G; ++gr) {
        float f = a;
        if (vt[gr] > vtop[gr]) {
          const float now = to_fp16_range(__uint_as_float(vt[gr]));
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
      const float w = e * half_lo(vp[gr]) * vf[gr];
      const __half wh = __float2half_rn(w), wl = __float2half_rn(w - __half2float(wh));
      const uint32_t both = pack_halves(wh, wl);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {  // 16 keys each: t, t + 4 | t + 8, t + 12 of the tile
        const uint32_t w0 = __shfl_sync(0xffffffffu, both, 4 * t + 2 * ks), w1 = __shfl_sync(0xffffffffu, both, 4 * t + 16 + 2 * ks);
        const uint32_t w2 = __shfl_sync(0xffffffffu, both, 4 * t + 2 * ks + 1);
        const uint32_t w3 = __shfl_sync(0xffffffffu, both, 4 * t + 16 + 2 * ks + 1);
        const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
        const uint32_t b0 = __byte_perm(w0, w1, sel), b1 = __byte_perm(w2, w3, sel);
        const uint32_t v0 = vw[4 * ks][gr], v1 = vw[4 * ks + 1][gr], v2 = vw[4 * ks + 2][gr], v3 = vw[4 * ks + 3][gr];
        // bytes 0, 1 then 2, 3 of a key pair side by side: dims 0-3 and 4-7 of the lane's eight
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const uint32_t x = __byte_perm(v0, v1, hf ? 0x7632u : 0x5410u), y = __byte_perm(v2, v3, hf ? 0x7632u : 0x5410u);
          mma16816(acc[gr][2 * hf], x & EVEN, x & ODD, y & EVEN, y & ODD, b0, b1);
          mma16816(acc[gr][2 * hf + 1], (x >> 8) & EVEN, (x >> 8) & ODD, (y >> 8) & EVEN, (y >> 8) & ODD, b0, b1);
        }
      }
    }
  }

  // one (max, sum, output) set per warp
  l = warp_sum(l);
#pragma unroll
  for (int gr = 0; gr < G; ++gr) {
    const float add = warp_sum(lo_sum[gr]), f = TWO24 / vf[gr];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (t == i) {
        s_acc[warp][64 * gr + 8 * g + 2 * i] = (acc[gr][i][0] + acc[gr][i][1]) * f + add;
        s_acc[warp][64 * gr + 8 * g + 2 * i + 1] = (acc[gr][i][2] + acc[gr][i][3]) * (f * 0.0625f) + add;
      }
  }
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
  if (SELF && with_new) {
    // the new key and value, each by a warp: into the cache, and as a set of their own with the bf16 values
    constexpr int N = D / 32;
    if (warp < 2) {
      const float* src = qrow + (size_t)(1 + warp) * p.H * D;
      float x[N];
      append<D>(src, (warp ? p.v : p.k) + (vec0 + n) * (D / 2), (warp ? p.vm : p.km) + (vec0 + n) * G, lane, x);
      if (warp == 0) {
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) d += __ldcg(qrow + lane * N + i) * x[i];
        d = warp_sum(d) * p.scale_log2;
        if (lane == 0) s_m[WARPS] = d, s_l[WARPS] = 1.f;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) s_acc[WARPS][lane * N + i] = x[i];
      }
    }
  }
  pdl_trigger();  // late: a grid that started earlier would take registers from the stream
  __syncthreads();
  const int sets = with_new ? SETS : WARPS;
  float M = LOWEST, L = 0.f, O = 0.f;
  if (tid < D) {
    for (int i = 0; i < sets; ++i) M = fmaxf(M, s_m[i]);
    for (int i = 0; i < sets; ++i) {
      const float w = ex2(s_m[i] - M);
      L += w * s_l[i], O += w * s_acc[i][tid];
    }
  }
  const auto store = [&](float o, float sum) {
    const float val = sum > 0.f || sum != sum ? o / sum : 0.f;  // no key at all: zeros
    const size_t at = ((size_t)r * p.H + h) * D + tid;
    if (p.out_kind == B200DEC_OUT_F16) reinterpret_cast<__half*>(p.out)[at] = __float2half_rn(clamp_h(val));
    else reinterpret_cast<float*>(p.out)[at] = val;
  };
  if (chunks == 1) {
    if (tid < D) store(O, L);
    return;
  }
  // a row in several chunks: partials to the workspace, the last CTA of the (row, head) to arrive merges them
  const int item = r * p.H + h;
  float* part = p.part + ((size_t)item * gridDim.x + blockIdx.x) * (D + 2);
  if (tid < D) part[tid] = O;
  if (tid == 0) part[D] = M, part[D + 1] = L;
  __threadfence();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(p.count + item, 1) == chunks - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  if (tid < D) {
    const float* pb = p.part + (size_t)item * gridDim.x * (D + 2);
    float MM = LOWEST;
    for (int i = 0; i < chunks; ++i) MM = fmaxf(MM, __ldcg(pb + i * (D + 2) + D));
    float LL = 0.f, OO = 0.f;
    for (int i = 0; i < chunks; ++i) {
      const float w = ex2(__ldcg(pb + i * (D + 2) + D) - MM);
      LL += w * __ldcg(pb + i * (D + 2) + D + 1);
      OO += w * __ldcg(pb + i * (D + 2) + tid);
    }
    store(OO, LL);
  }
  if (tid == 0) p.count[item] = 0;
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
  B200_REQUIRE(ldq >= (self ? 3 : 1) * heads * head_dim && ldq % 4 == 0 && ((uintptr_t)q & 15) == 0,
               "attention_q4: ldq %d (rows of %d floats, 16-byte aligned)", ldq, (self ? 3 : 1) * heads * head_dim);
  B200_REQUIRE((((uintptr_t)kcache | (uintptr_t)vcache) & 15) == 0 && (((uintptr_t)kpairs | (uintptr_t)vpairs) & 3) == 0 &&
                   (!sched || ((uintptr_t)sched & 15) == 0), "attention_q4: alignment");
  B200_REQUIRE(out_kind == B200DEC_OUT_F16 || out_kind == B200DEC_OUT_F32, "attention_q4: out_kind %d", out_kind);
  Q4Args p{active, q, (uint8_t*)kcache, (uint8_t*)vcache, (uint32_t*)kpairs, (uint32_t*)vpairs, n, sched, out, part, count, status,
           ldq, heads, cap, slots, out_kind, cap, scale * 1.4426950408889634f};
  const int splits = part ? q4_splits(rows, heads, cap) : 1;
  p.chunk = ((cap + splits - 1) / splits + BLOCK_KEYS - 1) / BLOCK_KEYS * BLOCK_KEYS;
  const dim3 grid(splits, heads, rows);
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e =
      head_dim == 64 ? self ? launch_kernel(attention_q4_kernel<64, true>, grid, dim3(NTHREADS), 0, st, 0, pdl, p)
                            : launch_kernel(attention_q4_kernel<64, false>, grid, dim3(NTHREADS), 0, st, 0, pdl, p)
      : self ? launch_kernel(attention_q4_kernel<128, true>, grid, dim3(NTHREADS), 0, st, 0, pdl, p)
             : launch_kernel(attention_q4_kernel<128, false>, grid, dim3(NTHREADS), 0, st, 0, pdl, p);
  if (e != cudaSuccess) return fail(B200DEC_ECUDA, "attention_q4 launch: %s", cudaGetErrorString(e));
  return 0;
}

}  // extern "C"
