// Rows of keys and values into the 4-bit slot caches, and back (format: kv4.cuh).
//
// One thread per 16 dims on the way in (two 32-byte loads, the group's extremes over four lanes; what a group costs is shared by
// more values than with 8), per 8 on the way back; the first lane of a group stores its (step, lo). A CTA takes a fixed range
// of channels over many rows, so that the channel's (layer, key | value, head) is worked out once. What it has to move is the fp32 rows (8 times the codes); the way in is close to bound by its instructions (23
// a value), the way back by writing. 64 clips, 13 600 rows of 16 384 values: 179 us in (5.7 TB/s; 217 with 8 dims a
// thread), 171 us back (5.9 TB/s).
#include "kv4.cuh"

using namespace b200dec_detail;

namespace {

struct Kv4Args {
  float* kv;  // (nrows, layers * 2 * H * D)
  const int* slot_of;
  const int* frame_of;
  uint32_t* ck;  // (L, S1, H, T, D / 8) words of codes
  uint32_t* cv;
  uint32_t* ckm;  // (L, S1, H, T, D / 64) {step, lo}
  uint32_t* cvm;
  int nrows, L, S1, H, D, T;
};

constexpr int THREADS = 256;

struct f32x8 {
  float v[8];
};
DEVI f32x8 ld_stream32(const float* p) {
  f32x8 r;
  asm volatile("ld.global.nc.L1::no_allocate.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(r.v[0]), "=f"(r.v[1]), "=f"(r.v[2]), "=f"(r.v[3]), "=f"(r.v[4]), "=f"(r.v[5]), "=f"(r.v[6]), "=f"(r.v[7])
               : "l"(p));
  return r;
}
DEVI void st32(float* p, const f32x8& r) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(r.v[0]), "f"(r.v[1]), "f"(r.v[2]), "f"(r.v[3]),
               "f"(r.v[4]), "f"(r.v[5]), "f"(r.v[6]), "f"(r.v[7])
               : "memory");
}

// The thread's DIMS dims of every row: where their codes and pair of slot 0, frame 0 lie, and how far a slot is from the next.
struct Channel {
  uint32_t* codes;
  uint32_t* pair;
  int slot_vecs, code_words, pair_words;  // vectors of a slot; words of a vector
  bool live, first;                       // in the row at all; the first of its group
};
template <int DIMS>
DEVI Channel channel(const Kv4Args& p) {
  const int pieces = p.D / DIMS, chunks = p.L * 2 * p.H * pieces;
  const int c = blockIdx.x * THREADS + threadIdx.x, cc = min(c, chunks - 1);
  const int d = cc % pieces * DIMS, h = (cc / pieces) % p.H, kvi = (cc / (pieces * p.H)) & 1, l = cc / (pieces * p.H * 2);
  const size_t vec = ((size_t)l * p.S1 * p.H + h) * p.T;
  return Channel{(kvi ? p.cv : p.ck) + vec * (p.D / 8) + d / 8, (kvi ? p.cvm : p.ckm) + vec * (p.D / 64) + d / 64, p.H * p.T,
                 p.D / 8, p.D / 64, c < chunks, d % 64 == 0};
}
DEVI int64_t vecs(const Channel& c, int slot, int frame) { return (int64_t)slot * c.slot_vecs + frame; }
DEVI bool inside(const Kv4Args& p, int slot, int frame) { return slot >= 0 && slot < p.S1 && frame >= 0 && frame < p.T; }

__global__ void __launch_bounds__(THREADS, 4) scatter_kv_q4_kernel(const Kv4Args p) {
  const Channel c = channel<16>(p);
  const size_t width = (size_t)p.L * 2 * p.H * p.D, at = (size_t)(blockIdx.x * THREADS + threadIdx.x) * 16;
  struct Row {
    f32x8 x[2];
    int slot, frame;
  };
  const auto load = [&](int row) {
    Row r{};
    r.slot = -1;
    if (row < p.nrows) {
      r.slot = __ldg(p.slot_of + row), r.frame = __ldg(p.frame_of + row);
      if (c.live) r.x[0] = ld_stream32(p.kv + row * width + at), r.x[1] = ld_stream32(p.kv + row * width + at + 8);
    }
    return r;
  };
  Row next = load(blockIdx.y);
  for (int row = blockIdx.y; row < p.nrows; row += gridDim.y) {
    Row r = next;
    next = load(row + gridDim.y);  // on its way while this one is worked on
    if (!inside(p, r.slot, r.frame)) continue;  // the whole CTA
    uint32_t hi = 0, lo = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const uint32_t w = pack_bf16(r.x[k].v[i], r.x[k].v[i + 1]);
        hi = k + i ? max_bf16x2(hi, w) : w, lo = k + i ? min_bf16x2(lo, w) : w;
        r.x[k].v[i] = bf16_lo(w), r.x[k].v[i + 1] = bf16_hi(w);
      }
    // {largest, -smallest} of the 16, then of the group's four threads: both go round in one word
    uint32_t ext = max_bf16x2(__byte_perm(hi, lo ^ 0x80008000u, 0x5410), __byte_perm(hi, lo ^ 0x80008000u, 0x7632));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) ext = max_bf16x2(ext, __shfl_xor_sync(0xffffffffu, ext, o));
    float mx = bf16_lo(ext), mn = -bf16_hi(ext);
    if (__any_sync(0xffffffffu, !kv4_tame(mn, mx))) {  // something to clamp, or a NaN, in some group of the warp
      mn = INFINITY, mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float& x = r.x[k].v[i];
          x = kv4_clamp(x), mn = fminf(mn, x), mx = fmaxf(mx, x);
        }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      }
    }
    if (!c.live) continue;
    const Kv4Group g = kv4_group(mn, mx);
    uint32_t codes[2];
    const bool plain = kv4_plain(g);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (plain) codes[k] = kv4_codes8<false>(r.x[k].v, g);
      else kv4_codes_slow<8, false>(r.x[k].v, g, &codes[k]);
    }
    const int64_t v = vecs(c, r.slot, r.frame);
    *reinterpret_cast<uint2*>(c.codes + v * c.code_words) = make_uint2(codes[0], codes[1]);
    if (c.first) c.pair[v * c.pair_words] = g.word;
  }
}

__global__ void __launch_bounds__(THREADS) gather_kv_q4_kernel(const Kv4Args p) {
  const Channel c = channel<8>(p);
  if (!c.live) return;
  const size_t width = (size_t)p.L * 2 * p.H * p.D, at = (size_t)(blockIdx.x * THREADS + threadIdx.x) * 8;
  for (int row = blockIdx.y; row < p.nrows; row += gridDim.y) {
    const int slot = __ldg(p.slot_of + row), frame = __ldg(p.frame_of + row);
    f32x8 x{};
    if (inside(p, slot, frame)) {
      const int64_t v = vecs(c, slot, frame);
      const uint32_t w = c.codes[v * c.code_words], m = c.pair[v * c.pair_words];
      const float step = __half2float(__ushort_as_half(m & 0xffff)), lo = __half2float(__ushort_as_half(m >> 16));
#pragma unroll
      for (int i = 0; i < 8; ++i) x.v[i] = kv4_value((w >> (4 * i)) & 15, step, lo);
    }
    st32(p.kv + row * width + at, x);
  }
}

int check_kv4(const char* what, const void* kv, const int32_t* slot_of, const int32_t* frame_of, const void* ck, const void* cv,
              const void* ckm, const void* cvm, int nrows, int layers, int slots_plus_1, int heads, int head_dim, int frames) {
  B200_REQUIRE(nrows >= 0, "%s: nrows %d", what, nrows);
  B200_REQUIRE(kv && slot_of && frame_of && ck && cv && ckm && cvm, "%s: null pointer", what);
  B200_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim %d (64 or 128)", what, head_dim);
  B200_REQUIRE(layers >= 1 && slots_plus_1 >= 1 && heads >= 1 && frames >= 1 && (int64_t)layers * 2 * heads * head_dim <= 1 << 28 &&
                   (int64_t)heads * frames <= 1 << 30,
               "%s: layers %d slots %d heads %d frames %d", what, layers, slots_plus_1, heads, frames);
  B200_REQUIRE(((uintptr_t)kv & 31) == 0 && (((uintptr_t)ck | (uintptr_t)cv) & 7) == 0 && (((uintptr_t)ckm | (uintptr_t)cvm) & 3) == 0,
               "%s: alignment (the rows 32 bytes, the codes 8, the pairs 4)", what);
  return 0;
}

dim3 kv4_grid(const Kv4Args& p, int dims) {
  const int x = (p.L * 2 * p.H * (p.D / dims) + THREADS - 1) / THREADS;
  const int y = (148 * 8 * 4 + x - 1) / x;  // about four waves of CTAs
  return dim3(x, p.nrows < y ? p.nrows : y);
}

Kv4Args kv4_args(float* kv, const int32_t* slot_of, const int32_t* frame_of, void* ck, void* cv, void* ckm, void* cvm, int nrows,
                 int layers, int slots_plus_1, int heads, int head_dim, int frames) {
  return Kv4Args{kv, slot_of, frame_of, (uint32_t*)ck, (uint32_t*)cv, (uint32_t*)ckm, (uint32_t*)cvm, nrows, layers, slots_plus_1,
                 heads, head_dim, frames};
}

}  // namespace

extern "C" {

int b200dec_scatter_kv_q4(const float* kv, const int32_t* slot_of, const int32_t* frame_of, void* ck, void* cv, void* ck_pairs,
                          void* cv_pairs, int nrows, int layers, int slots_plus_1, int heads, int head_dim, int frames,
                          void* stream) {
  if (const int rc = check_kv4("scatter_kv_q4", kv, slot_of, frame_of, ck, cv, ck_pairs, cv_pairs, nrows, layers, slots_plus_1,
                               heads, head_dim, frames))
    return rc;
  if (nrows == 0) return 0;
  const Kv4Args p = kv4_args(const_cast<float*>(kv), slot_of, frame_of, ck, cv, ck_pairs, cv_pairs, nrows, layers, slots_plus_1,
                             heads, head_dim, frames);
  scatter_kv_q4_kernel<<<kv4_grid(p, 16), THREADS, 0, (cudaStream_t)stream>>>(p);
  return check_launch("scatter_kv_q4");
}

int b200dec_gather_kv_q4(float* kv, const int32_t* slot_of, const int32_t* frame_of, const void* ck, const void* cv,
                         const void* ck_pairs, const void* cv_pairs, int nrows, int layers, int slots_plus_1, int heads,
                         int head_dim, int frames, void* stream) {
  if (const int rc = check_kv4("gather_kv_q4", kv, slot_of, frame_of, ck, cv, ck_pairs, cv_pairs, nrows, layers, slots_plus_1,
                               heads, head_dim, frames))
    return rc;
  if (nrows == 0) return 0;
  const Kv4Args p = kv4_args(kv, slot_of, frame_of, const_cast<void*>(ck), const_cast<void*>(cv), const_cast<void*>(ck_pairs),
                             const_cast<void*>(cv_pairs), nrows, layers, slots_plus_1, heads, head_dim, frames);
  gather_kv_q4_kernel<<<kv4_grid(p, 8), THREADS, 0, (cudaStream_t)stream>>>(p);
  return check_launch("gather_kv_q4");
}

}  // extern "C"
