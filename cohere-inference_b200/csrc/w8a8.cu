// A product of 8-bit integers on the fifth-generation tensor cores: y = act((q_x q_w^T) * s_x * s_w + bias), q_x quantised per row as
// the rows come, q_w and s_w per channel at init time. The result goes to fp32, fp16 or bf16 rows, or straight into the slot
// caches (the cross-attention prefill in 8 bits).
//
// Both operands lie in global memory as the images of their shared-memory tiles (rows of 128 bytes = 128 k, 128-byte swizzle), so a
// pipeline stage is two plain cp.async.bulk copies. tcgen05.mma kind::i8 multiplies M 128 x N TN x K 32 into 32-bit integer
// accumulators in tensor memory: the sums are exact, and every later operation rounds once.
//   * persistent CTAs walk the (channel tile, row tile) list: warp 0 feeds the ring, warp 1 issues the MMAs into one of two
//     accumulators, warps 2-17 drain the other: four warps per 32 lanes, each a quarter of the tile's columns. Per k the MMA is
//     twice as fast as with 16-bit operands, so the epilogue decides, and what decides it is latency: 13 600 x 1024 x 16 384 to bf16
//     took 591 us with four warps, 258-274 with eight, 218-240 with sixteen and turned stores (k = 128: 232 with eight, 147 with
//     sixteen); the products alone take 135 us (the slope from k = 1024 to 2048).
//     Pairs of CTAs (cta_group::2), which copy a third less, were slower: 390 us per 1024 of k.
//   * channel scales and biases of a tile go to shared memory once, as pairs, and are read back as broadcasts.
//   * rows leave in runs of 64 bytes; rows that are not 16-byte aligned through a transposition in shared memory.
// Every mbarrier wait is bounded; a wait that runs out sets B200DEC_ST_TIMEOUT, the roles fall through, copies in flight are
// awaited (bounded) and tensor memory is released.
#include <type_traits>

#include "kv_store.cuh"
#include "umma.cuh"

using namespace b200dec_detail;

namespace {

constexpr int BM = UMMA_BM, BN = UMMA_BN, MAX_K8 = 131072;  // 127 * 127 * k stays below 2^31
constexpr int MAX_MN = 1 << 30;
constexpr int EPI_WARPS = 16, NTHREADS = 64 + 32 * EPI_WARPS;

template <int TN>
struct Tile {
  static constexpr int B_STAGE = TN * 128, STAGE_BYTES = A_STAGE + B_STAGE, STAGES = TN == 256 ? 4 : TN == 128 ? 5 : 7;
  static constexpr int TR_COLS = TN == 256 ? 8 : 16, TR_LD = TR_COLS + 1;  // columns of rows turned in shared memory at a time
  static constexpr int PARTS = TN / 32 < 4 ? TN / 32 : 4;                  // of the columns, a warp each per 32 lanes
  static constexpr int PAIRS = STAGES * STAGE_BYTES, TR = PAIRS + 2 * TN * 8;  // {scale, bias} per column and accumulator
  static constexpr int SMEM_BYTES = TR + EPI_WARPS * 32 * TR_LD * 4 + 1024;     // slack to align the base to a swizzle atom
  static constexpr int TMEM_COLS = 2 * TN;
  // signed 8-bit x signed 8-bit -> 32-bit, both operands K-major, M = 128, N = TN
  static constexpr uint32_t IDESC =
      (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
};

struct W8Args {
  const unsigned char* a;  // rows: [m tile][K / 128][16 KB]
  const unsigned char* w;  // weights: [n / 256][K / 128][32 KB]
  const float* a_scale;    // (M)
  const float* w_scale;    // (N)
  const float* bias;       // (N) or null
  int M, N, NKB;           // NKB: blocks of 128 k
  int mode;                // 1 bf16 caches, 2 int8 caches, 3 4-bit caches, 4 rows
  int act;
  void* out;               // mode 4: (M, ldo) of out_kind
  int64_t ldo;
  int out_kind;
  const int4* pieces;      // modes 1-3: (n_pieces) {first row, frames, slot, 0}, first rows ascending from 0
  int n_pieces;
  void* ck;
  void* cv;
  float* cks;
  float* cvs;
  int S1, H, D, T;         // caches (layers, S1, H, T, D)
  int* status;
};

DEVI void umma_i8(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
DEVI void epi_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(32 * EPI_WARPS) : "memory"); }

DEVI float relu(float x) {  // NaN stays NaN (fmaxf would make it 0)
  float y;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(x));
  return y;
}
DEVI float activate(float x, int act) {
  if (act == B200DEC_ACT_RELU) return relu(x);
  if (act == B200DEC_ACT_GELU) return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
  return x;
}

// two fp32 operations in one instruction
DEVI uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
DEVI void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
DEVI uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
DEVI uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 32 sums of a row -> values: sum * (row scale * channel scale) + bias; ws, bs: the columns' scales and biases
DEVI void finish32(const uint32_t (&e)[32], float (&v)[32], const float* ws, const float* bs, float sa, int act) {
  const uint64_t s2 = pack2(sa, sa);
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(ws + i), b = *reinterpret_cast<const ulonglong2*>(bs + i);
    unpack2(fma2(pack2(__int2float_rn((int)e[i]), __int2float_rn((int)e[i + 1])), mul2(s2, w.x), b.x), v[i], v[i + 1]);
    unpack2(fma2(pack2(__int2float_rn((int)e[i + 2]), __int2float_rn((int)e[i + 3])), mul2(s2, w.y), b.y), v[i + 2], v[i + 3]);
  }
  if (act != B200DEC_ACT_NONE) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = activate(v[i], act);
  }
}

// Among four neighbouring lanes, each with four pieces of 16 bytes: piece j of lane i becomes piece i of lane j.
DEVI void turn_pieces(uint32_t (&p)[4][4], int lane) {
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const bool high = lane & o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j & o) continue;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, high ? p[j][c] : p[j + o][c], o);
        p[j][c] = high ? got : p[j][c], p[j + o][c] = high ? p[j + o][c] : got;
      }
    }
  }
}

template <class T>
DEVI T out_value(float x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}
DEVI uint32_t pair_of(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return reinterpret_cast<const uint32_t&>(h);
}
DEVI uint32_t pair_of(float a, float b, __nv_bfloat16) { return pack_bf16(a, b); }
// 32 columns of the warp's 32 rows (a row per thread) from row m0 on, column n0 on, into T rows
template <class T, int TR_COLS>
DEVI void store_rows(const W8Args& p, const float (&v)[32], int m0, int n0, int lane, bool wide, float* tr) {
  constexpr int TR_LD = TR_COLS + 1, ROWS = 32 / TR_COLS;
  T* out = reinterpret_cast<T*>(p.out);
  if (wide && n0 + 32 <= p.N) {
    // 64 bytes of a row at a time: four lanes turn theirs, so that a store instruction covers runs of 64 bytes of eight rows (a
    // thread per row wrote 32 rows' single sectors: 267 us for 13 600 x 1024 x 16 384, 240 this way)
    constexpr int PER = 16 / (int)sizeof(T);  // values of a piece
#pragma unroll
    for (int c = 0; c < 32; c += 4 * PER) {
      uint32_t w[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (sizeof(T) == 4) w[j][i] = __float_as_uint(v[c + PER * j + i]);
          else w[j][i] = pair_of(v[c + PER * j + 2 * i], v[c + PER * j + 2 * i + 1], T());
        }
      turn_pieces(w, lane);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = m0 + (lane & ~3) + j;
        if (m < p.M)
          *reinterpret_cast<uint4*>(out + (size_t)m * p.ldo + n0 + c + PER * (lane & 3)) = make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]);
      }
    }
    return;
  }
  // TR_COLS columns at a time through shared memory: a store instruction then covers runs of that many columns
#pragma unroll
  for (int c = 0; c < 32; c += TR_COLS) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < TR_COLS; ++i) tr[lane * TR_LD + i] = v[c + i];
    __syncwarp();
    const int col = n0 + c + lane % TR_COLS;
    if (col < p.N) {
#pragma unroll 4
      for (int r = lane / TR_COLS; r < 32; r += ROWS)
        if (m0 + r < p.M) out[(size_t)(m0 + r) * p.ldo + col] = out_value<T>(tr[r * TR_LD + lane % TR_COLS]);
    }
  }
}

template <int TN>
__global__ void __launch_bounds__(NTHREADS, 1) w8a8_kernel(const W8Args p) {
  using Cfg = Tile<TN>;
  constexpr int STAGES = Cfg::STAGES, STAGE_BYTES = Cfg::STAGE_BYTES, B_STAGE = Cfg::B_STAGE;
  extern __shared__ unsigned char dyn_smem[];
  unsigned char* smem = dyn_smem + ((1024 - (smem_u32(dyn_smem) & 1023)) & 1023);
  __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], tfull[2], tempty[2];
  __shared__ uint32_t tmem_base;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int MT = (p.M + BM - 1) / BM, NT = (p.N + TN - 1) / TN, NKB = p.NKB;
  const int64_t tiles = (int64_t)MT * NT;
  const auto weights = [&](int nt, int kb) {
    const int n0 = nt * TN;
    return p.w + ((size_t)(n0 / BN) * NKB + kb) * B_BLOCK + n0 % BN / TN * B_STAGE;
  };

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&tfull[i], 1), mbar_init(&tempty[i], EPI_WARPS);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    // the first tile's weights are nobody's output: on their way before the wait for the kernel that quantises the rows
    for (int kb = 0; kb < min(NKB, STAGES); ++kb) {
      mbar_expect_tx(&full[kb], STAGE_BYTES);
      bulk_load(smem + kb * STAGE_BYTES + A_STAGE, weights(blockIdx.x / MT, kb), B_STAGE, &full[kb]);
    }
  }
  pdl_wait();  // ahead of the allocation, so that no CTA sits on tensor memory while it waits
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                 "n"(Cfg::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_d = tmem_base;
  pdl_trigger();

  if (warp == 0) {
    // ---- producer: two bulk copies per stage ----------------------------------------------------------------------------
    if (lane == 0) {
      bool ok = true;
      uint32_t it = 0;
      for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
        const int mt = (int)(tile % MT), nt = (int)(tile / MT);
        for (int kb = 0; kb < NKB; ++kb, ++it) {
          const int s = it % STAGES;
          unsigned char* st = smem + s * STAGE_BYTES;
          if (it >= (uint32_t)min(NKB, STAGES)) {
            ok = mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1);
            if (!ok) break;
            mbar_expect_tx(&full[s], STAGE_BYTES);
            bulk_load(st + A_STAGE, weights(nt, kb), B_STAGE, &full[s]);
          }
          bulk_load(st, p.a + ((size_t)mt * NKB + kb) * A_STAGE, A_STAGE, &full[s]);
        }
      }
      if (!ok) {
        atomicOr(p.status, B200DEC_ST_TIMEOUT);
        // the copies already issued must land before this CTA's shared memory is given away
        const uint32_t issued = it < (uint32_t)STAGES ? it : (uint32_t)STAGES;
        for (uint32_t i = 0; i < issued; ++i) {
          const uint32_t jt = it - 1 - i;
          mbar_wait(&full[jt % STAGES], (jt / STAGES) & 1);
        }
      }
    }
  } else if (warp == 1) {
    // ---- MMA issue: one lane --------------------------------------------------------------------------------------------
    if (lane == 0) {
      bool ok = true;
      uint32_t it = 0, tc = 0;
      for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++tc) {
        const uint32_t buf = tc & 1;
        ok = mbar_wait(&tempty[buf], ((tc >> 1) & 1) ^ 1);  // the epilogue has drained this accumulator
        if (!ok) break;
        tc_fence_after();
        const uint32_t acc = tmem_d + buf * TN;
        for (int kb = 0; kb < NKB; ++kb, ++it) {
          const int s = it % STAGES;
          ok = mbar_wait(&full[s], (it / STAGES) & 1);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a0 = smem_u32(smem + s * STAGE_BYTES), b0 = a0 + A_STAGE;
#pragma unroll
          for (int k = 0; k < 4; ++k)  // 32 k = 32 bytes each
            umma_i8(acc, umma_desc(a0 + k * 32), umma_desc(b0 + k * 32), Cfg::IDESC, (kb | k) != 0);
          umma_commit(&empty[s]);  // the stage is free once these MMAs have read it
        }
        if (ok) umma_commit(&tfull[buf]);
      }
      if (!ok) atomicOr(p.status, B200DEC_ST_TIMEOUT);
    }
  } else {
    // ---- epilogue: warp w reads tensor-memory lanes 32 (w % 4) .. + 31, the columns' part (w - 2) / 4 -----------------------
    const int q = warp & 3, row = q * 32 + lane, part = (warp - 2) >> 2, et = tid - 64;
    // rows: every part a warp of its own; caches: two parts, so that a head's 128 channels are one thread's
    const int parts = p.mode == 4 ? Cfg::PARTS : 2, cols = TN / parts;
    float* tr = reinterpret_cast<float*>(smem + Cfg::TR) + (warp - 2) * 32 * Cfg::TR_LD;
    const int size = p.out_kind == B200DEC_T_F32 ? 4 : 2;
    const bool wide = ((uintptr_t)p.out & 15) == 0 && p.ldo * size % 16 == 0;
    bool ok = true;
    uint32_t tc = 0;
    // what a tile needs from global memory is fetched a tile ahead: this thread's column's {scale, bias}, its row's scale
    static_assert(TN <= 32 * EPI_WARPS, "one column per epilogue thread");
    float2 pair_next;
    float sa_next;
    const auto fetch = [&](int64_t tile) {
      const int m = (int)(tile % MT) * BM + row, n = (int)(tile / MT) * TN + et;
      const bool has = tile < tiles && et < TN && n < p.N;
      pair_next = make_float2(has ? __ldg(p.w_scale + n) : 0.f, has && p.bias ? __ldg(p.bias + n) : 0.f);
      sa_next = tile < tiles && m < p.M ? __ldg(p.a_scale + m) : 0.f;
    };
    fetch(blockIdx.x);
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++tc) {  // after a time-out too: all meet at the barriers
      const int mt = (int)(tile % MT), nt = (int)(tile / MT), buf = tc & 1;
      const int m = mt * BM + row;
      // the pairs go into the buffer of two tiles ago, which every warp has left (it passed the barrier of the tile between)
      float* pairs = reinterpret_cast<float*>(smem + Cfg::PAIRS) + buf * 2 * TN;  // TN scales, TN biases
      if (et < TN) pairs[et] = pair_next.x, pairs[TN + et] = pair_next.y;
      const float sa = sa_next;
      fetch(tile + gridDim.x);
      int slot = -1, frame = 0;
      if (p.mode != 4 && m < p.M) {  // the piece that holds row m: the last one that starts at or before it
        int lo = 0, hi = p.n_pieces - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (__ldg(&p.pieces[mid].x) <= m) lo = mid;
          else hi = mid - 1;
        }
        const int4 pc = __ldg(&p.pieces[lo]);
        frame = m - pc.x;
        if (frame >= 0 && frame < pc.y && frame < p.T && pc.z >= 0 && pc.z < p.S1) slot = pc.z;
      }
      epi_barrier();
      if (ok) ok = mbar_wait(&tfull[buf], (tc >> 1) & 1);
      if (!ok) continue;
      tc_fence_after();
      const uint32_t acc = tmem_d + buf * TN + part * cols + ((uint32_t)(q * 32) << 16);
      const float* ws = pairs + part * cols;
      const float* bs = ws + TN;
      const int n0 = nt * TN + part * cols;
      const auto load = [&](int c, float (&v)[32], int act) {  // columns c .. c + 31 of the part
        uint32_t e[32];
        __syncwarp();  // a collective load: rows without a slot may have gone ahead
        tmem_ld32(acc + c, e);
        tmem_wait();
        finish32(e, v, ws + c, bs + c, sa, act);
      };
      float v[32];
      if (p.mode == 4) {
        if (part < parts)
#pragma unroll 1
          for (int c = 0; c < TN / Cfg::PARTS && n0 + c < p.N; c += 32) {
            load(c, v, p.act);
            const int m0 = mt * BM + q * 32;
            if (p.out_kind == B200DEC_T_F32) store_rows<float, Cfg::TR_COLS>(p, v, m0, n0 + c, lane, wide, tr);
            else if (p.out_kind == B200DEC_T_F16) store_rows<__half, Cfg::TR_COLS>(p, v, m0, n0 + c, lane, wide, tr);
            else store_rows<__nv_bfloat16, Cfg::TR_COLS>(p, v, m0, n0 + c, lane, wide, tr);
          }
      } else if constexpr (TN == BN) {
        // caches: a group of 64 channels, or a head's D for int8, at a time; channel n = ((layer * 2 + k|v) * H + head) * D + d.
        // Its values go by twice, for its extremes and to be stored.
        const int span = p.mode == 2 ? p.D : 64;
#pragma unroll 1
        for (int c = 0; c < cols && part < parts; c += span) {
          const int n = n0 + c, hd = p.H * p.D, l = n / (2 * hd), kvi = (n / hd) & 1, h = (n % hd) / p.D, d0 = n % p.D;
          const size_t vec = slot < 0 ? 0 : ((((size_t)l * p.S1 + slot) * p.H + h) * p.T + frame);
          char* cache = reinterpret_cast<char*>(kvi ? p.cv : p.ck);
          float mn = 0.f, mx = 0.f;
          bool tame = true;
          if (p.mode != 1) {
            uint32_t hi = 0, lo = 0;
#pragma unroll 1
            for (int i = 0; i < span; i += 32) {
              load(c + i, v, B200DEC_ACT_NONE);
              if (p.mode == 3) extremes_32(v, i == 0, hi, lo);
              else {
#pragma unroll
                for (int j = 0; j < 32; ++j) mx = fmaxf(mx, fabsf(__bfloat162float(__float2bfloat16_rn(v[j]))));
              }
            }
            if (p.mode == 3) {
              extremes_of(hi, lo, mn, mx);
              tame = kv4_tame(mn, mx);
              if (__any_sync(0xffffffffu, !tame)) {  // some row of the warp: all of them again, the loads are the warp's
                mn = INFINITY, mx = -INFINITY;
#pragma unroll 1
                for (int i = 0; i < span; i += 32) {
                  load(c + i, v, B200DEC_ACT_NONE);
                  extremes_32_clamped(v, mn, mx);
                }
              }
            }
          }
          const float s8 = p.mode == 2 && mx > 0.f ? __fdiv_rn(mx, 127.f) : 1.f, inv8 = __fdiv_rn(1.f, s8);
          const Kv4Group g = kv4_group(mn, mx);
#pragma unroll 1
          for (int i = 0; i < span; i += 32) {
            load(c + i, v, B200DEC_ACT_NONE);
            if (slot >= 0) {
              const size_t at = vec * p.D + d0 + i;
              if (p.mode == 1) {
#pragma unroll
                for (int j = 0; j < 32; j += 8)
                  *reinterpret_cast<uint4*>(cache + (at + j) * 2) = make_uint4(pack_bf16(v[j], v[j + 1]), pack_bf16(v[j + 2], v[j + 3]),
                                                                               pack_bf16(v[j + 4], v[j + 5]), pack_bf16(v[j + 6], v[j + 7]));
              } else if (p.mode == 2) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = __bfloat162float(__float2bfloat16_rn(v[j]));
                store_q8_32(v, inv8, reinterpret_cast<int8_t*>(cache) + at);
              } else {
                store_q4_32(v, g, tame, reinterpret_cast<uint8_t*>(cache) + at / 2);
              }
            }
          }
          if (slot >= 0 && p.mode == 2) (kvi ? p.cvs : p.cks)[vec] = s8;
          if (slot >= 0 && p.mode == 3) reinterpret_cast<uint32_t*>(kvi ? p.cvs : p.cks)[(vec * p.D + d0) / 64] = g.word;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[buf]);
    }
    if (!ok && lane == 0) atomicOr(p.status, B200DEC_ST_TIMEOUT);
  }
  // ---- release the tensor memory: after every warp is done with it -----------------------------------------------------
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_d), "n"(Cfg::TMEM_COLS) : "memory");
  }
}

// ---- 8-bit operands --------------------------------------------------------------------------------------------------------
// Rows -> 8-bit integers with one scale a row: s = max(max |x|, 1e-12) / 127, q = rint(x / s), both as if the quotients were
// exact: the product with the reciprocal is off by a few 2^-23 of it, so only its rounding beside a half can be wrong, and
// the remainder x - q s (exact: a multiple of ulp(s) / 2 below 2^24 of them) decides there. A row with an infinity or NaN gets
// scale NaN: its results are NaN. One warp a row; rows of up to 1024 values stay in registers between the largest magnitude
// and the codes, longer ones are read again.
template <class X>
DEVI float row_value(X x) {
  if constexpr (std::is_same<X, float>::value) return x;
  else if constexpr (std::is_same<X, __half>::value) return __half2float(x);
  else return __bfloat162float(x);
}

// This lane's 16 of the 512 values from c on of a row of k, zeros past its end: loads of A bytes, neighbouring lanes side by side.
template <class X, int A>
DEVI void load_16(const X* row, int c, int k, int lane, float (&f)[16]) {
  constexpr int V = A / (int)sizeof(X);
#pragma unroll
  for (int j = 0; j < 16 / V; ++j) {
    const int at = c + (lane + 32 * j) * V;
    if (V > 1 && at + V <= k) {
      X x[V];
      if constexpr (A == 16) *reinterpret_cast<uint4*>(x) = __ldg(reinterpret_cast<const uint4*>(row + at));
      else if constexpr (A == 8) *reinterpret_cast<uint2*>(x) = __ldg(reinterpret_cast<const uint2*>(row + at));
      else *reinterpret_cast<uint32_t*>(x) = __ldg(reinterpret_cast<const uint32_t*>(row + at));
#pragma unroll
      for (int i = 0; i < V; ++i) f[j * V + i] = row_value(x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) f[j * V + i] = at + i < k ? row_value(row[at + i]) : 0.f;
    }
  }
}

DEVI int code8(float x, float s, float inv) {
  float c = fminf(fmaxf(rintf(x * inv), -127.f), 127.f);
  const float e2 = 2.f * __fmaf_rn(-c, s, x);
  const bool odd = ((int)c & 1) != 0;
  if (e2 > s || (e2 == s && odd)) c += 1.f;
  if (-e2 > s || (-e2 == s && odd)) c -= 1.f;
  return (int)fminf(fmaxf(c, -127.f), 127.f);
}

// The same for 16 values: adding 1.5 * 2^23 rounds the product, whose low byte is the code then (two's complement); only where one
// of them is within 2^-15 of a half, four times what the reciprocal can be off, does the remainder decide.
DEVI void codes16(const float (&x)[16], float s, float inv, uint8_t (&q)[16]) {
  constexpr float MAGIC = 12582912.f;
  float near = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float t = __fmaf_rn(x[i], inv, MAGIC);
    near = fmaxf(near, fabsf(__fmaf_rn(x[i], inv, MAGIC - t)));
    q[i] = (uint8_t)__float_as_uint(t);
  }
  if (near > 0.5f - 3.0517578e-05f) {
#pragma unroll
    for (int i = 0; i < 16; ++i) q[i] = (uint8_t)code8(x[i], s, inv);
  }
}

template <class X, int A>
__global__ void __launch_bounds__(256) pack_rows_i8_kernel(const X* __restrict__ x, int m, int k, int64_t ldx,
                                                           unsigned char* __restrict__ image, float* __restrict__ scale) {
  constexpr int V = A / (int)sizeof(X), KEPT = 2;  // 512 values each
  __shared__ __align__(16) uint8_t s_codes[8][512];
  const int warp = threadIdx.x >> 5, row = blockIdx.x * 8 + warp, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  if (row >= m) return;  // the rows that fill the last tile up are never stored: whatever the image holds there does no harm
  const X* src = x + row * ldx;
  uint32_t top = 0;  // largest magnitude by its bits, so that a NaN is the largest
  float kept[KEPT][16];
#pragma unroll
  for (int i = 0; i < KEPT; ++i) load_16<X, A>(src, 512 * i, k, lane, kept[i]);
#pragma unroll
  for (int i = 0; i < KEPT; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(kept[i][j]) & 0x7fffffffu);
  for (int c = 512 * KEPT; c < k; c += 512) {
    float f[16];
    load_16<X, A>(src, c, k, lane, f);
#pragma unroll
    for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  const float s = top < 0x7f800000u ? __fdiv_rn(fmaxf(__uint_as_float(top), 1e-12f), 127.f) : __uint_as_float(0x7fffffffu);
  const float inv = __frcp_rn(s);
  if (lane == 0) scale[row] = s;
  const int kp = (k + 127) / 128 * 128;
  unsigned char* tile = image + (size_t)(row / BM) * (kp / 128) * A_STAGE;
  const auto put = [&](int c, const float (&f)[16]) {  // 512 codes through shared memory into pieces of 16
    uint8_t* codes = s_codes[warp];
    __syncwarp();
    uint8_t q[16];
    codes16(f, s, inv, q);
#pragma unroll
    for (int j = 0; j < 16 / V; ++j) {
      uint8_t* to = codes + (lane + 32 * j) * V;
      if constexpr (V >= 4) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
          const uint8_t* b = q + j * V + i;
          *reinterpret_cast<uint32_t*>(to + i) = b[0] | b[1] << 8 | b[2] << 16 | (uint32_t)b[3] << 24;
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) to[i] = q[j * V + i];
      }
    }
    __syncwarp();
    const int at = c + 16 * lane;
    if (at < kp)
      *reinterpret_cast<uint4*>(tile + (size_t)(at / 128) * A_STAGE + swz(row % BM, (at % 128) / 16)) =
          *reinterpret_cast<const uint4*>(codes + 16 * lane);
  };
#pragma unroll
  for (int i = 0; i < KEPT; ++i)
    if (512 * i < kp) put(512 * i, kept[i]);
  for (int c = 512 * KEPT; c < kp; c += 512) {
    float f[16];
    load_16<X, A>(src, c, k, lane, f);
    put(c, f);
  }
}

// int8 weights (n, k) row-major -> [n / 256][k / 128][256 rows x 128 B, swizzled], zeros where n or k end; a thread per 16 bytes
__global__ void tile_weight_i8_kernel(const int8_t* __restrict__ q, int n, int k, unsigned char* __restrict__ out) {
  const int np = (n + BN - 1) / BN * BN, kp = (k + 127) / 128 * 128, cpr = kp / 16;
  const size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (size_t)np * cpr) return;
  const int r = (int)(i / cpr), c = (int)(i % cpr);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (r < n && c * 16 + j < k) w[j >> 2] |= (uint32_t)(uint8_t)q[(size_t)r * k + c * 16 + j] << ((j & 3) * 8);
  *reinterpret_cast<uint4*>(out + ((size_t)(r / BN) * (kp / 128) + c / 8) * B_BLOCK + swz(r % BN, c % 8)) =
      make_uint4(w[0], w[1], w[2], w[3]);
}

// The widest loads that the rows' addresses and distance allow.
template <class X>
cudaError_t launch_pack_i8(const void* x, int m, int k, int64_t ldx, void* image, float* scale, cudaStream_t st) {
  const uint64_t at = (uintptr_t)x | (m == 1 ? 0 : (uint64_t)ldx * sizeof(X));
  const dim3 grid((m + 7) / 8);
  const auto go = [&](auto kern) { kern<<<grid, 256, 0, st>>>((const X*)x, m, k, ldx, (unsigned char*)image, scale); };
  if (at % 16 == 0) go(pack_rows_i8_kernel<X, 16>);
  else if (at % 8 == 0) go(pack_rows_i8_kernel<X, 8>);
  else if (at % 4 == 0) go(pack_rows_i8_kernel<X, 4>);
  else if constexpr (sizeof(X) == 2) go(pack_rows_i8_kernel<X, 2>);
  return cudaGetLastError();
}

template <int TN>
int launch_tile(const W8Args& a, int sms, cudaStream_t stream) {
  constexpr int BYTES = Tile<TN>::SMEM_BYTES;
  cudaError_t e = cudaFuncSetAttribute(w8a8_kernel<TN>, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
  if (e != cudaSuccess) return fail(B200DEC_ECUDA, "w8a8: smem attribute: %s", cudaGetErrorString(e));
  const int64_t tiles = (int64_t)((a.M + BM - 1) / BM) * ((a.N + TN - 1) / TN);
  e = launch_kernel(w8a8_kernel<TN>, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(NTHREADS), BYTES, stream, 0, true, a);
  if (e != cudaSuccess) return fail(B200DEC_ECUDA, "w8a8 launch: %s", cudaGetErrorString(e));
  return 0;
}

// The narrowest tile with which the tiles still are one wave, else the widest: the wide one copies least per product.
int launch(const W8Args& a, cudaStream_t stream) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t mt = (a.M + BM - 1) / BM;
  if (a.mode == 4 && mt * ((a.N + 63) / 64) <= sms) return launch_tile<64>(a, sms, stream);
  if (a.mode == 4 && mt * ((a.N + 127) / 128) <= sms) return launch_tile<128>(a, sms, stream);
  return launch_tile<256>(a, sms, stream);
}

}  // namespace

extern "C" {

int64_t b200dec_w8a8_rows_bytes(int m, int k) {
  if (m < 0 || m > MAX_MN || k <= 0 || k > MAX_K8) return -1;
  return (int64_t)((m + BM - 1) / BM) * BM * ((k + 127) / 128 * 128);
}

int64_t b200dec_w8a8_weight_bytes(int n, int k) {
  if (n <= 0 || n > MAX_MN || k <= 0 || k > MAX_K8) return -1;
  return (int64_t)((n + BN - 1) / BN) * BN * ((k + 127) / 128 * 128);
}

int b200dec_w8a8_pack_rows(const void* x, int kind, int m, int k, int64_t ldx, void* image, float* scale, void* stream) {
  B200_REQUIRE(x && image && scale, "w8a8_pack_rows: null pointer");
  B200_REQUIRE(m >= 1 && m <= MAX_MN && k >= 1 && k <= MAX_K8 && (m == 1 || ldx >= k), "w8a8_pack_rows: m %d k %d ldx %lld", m, k, (long long)ldx);
  B200_REQUIRE(kind == B200DEC_T_F32 || kind == B200DEC_T_F16 || kind == B200DEC_T_BF16, "w8a8_pack_rows: kind %d", kind);
  B200_REQUIRE(((uintptr_t)image & 1023) == 0 && (uintptr_t)x % (kind == B200DEC_T_F32 ? 4 : 2) == 0,
               "w8a8_pack_rows: alignment (the image 1 KB)");
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = kind == B200DEC_T_F32   ? launch_pack_i8<float>(x, m, k, ldx, image, scale, st)
                        : kind == B200DEC_T_F16 ? launch_pack_i8<__half>(x, m, k, ldx, image, scale, st)
                                                : launch_pack_i8<__nv_bfloat16>(x, m, k, ldx, image, scale, st);
  if (e != cudaSuccess) return fail(B200DEC_ECUDA, "w8a8_pack_rows launch: %s", cudaGetErrorString(e));
  return 0;
}

int b200dec_w8a8_tile_weight(const int8_t* q, int n, int k, void* image, void* stream) {
  B200_REQUIRE(q && image && n >= 1 && n <= MAX_MN && k >= 1 && k <= MAX_K8 && ((uintptr_t)image & 1023) == 0,
               "w8a8_tile_weight: (%d, %d) into a 1 KB aligned image", n, k);
  const size_t total = (size_t)b200dec_w8a8_weight_bytes(n, k) / 16;
  tile_weight_i8_kernel<<<(unsigned)((total + 255) / 256), 256, 0, (cudaStream_t)stream>>>(q, n, k, (unsigned char*)image);
  return check_launch("w8a8_tile_weight");
}

int b200dec_w8a8_linear(const void* rows_image, const float* row_scale, int m, int k, const void* weight_image,
                        const float* w_scale, const float* bias, int n, int act, void* out, int out_kind, int64_t ldo,
                        int32_t* status, void* stream) {
  B200_REQUIRE(rows_image && row_scale && weight_image && w_scale && out && status, "w8a8_linear: null pointer");
  B200_REQUIRE(m >= 1 && m <= MAX_MN && n >= 1 && n <= MAX_MN && k >= 1 && k <= MAX_K8 && (m == 1 || ldo >= n), "w8a8_linear: m %d k %d n %d ldo %lld", m, k, n,
               (long long)ldo);
  B200_REQUIRE(out_kind == B200DEC_T_F32 || out_kind == B200DEC_T_F16 || out_kind == B200DEC_T_BF16, "w8a8_linear: out_kind %d", out_kind);
  B200_REQUIRE(act == B200DEC_ACT_NONE || act == B200DEC_ACT_RELU || act == B200DEC_ACT_GELU, "w8a8_linear: act %d", act);
  B200_REQUIRE((((uintptr_t)rows_image | (uintptr_t)weight_image) & 1023) == 0 && (((uintptr_t)w_scale | (uintptr_t)bias) & 15) == 0 &&
                   (uintptr_t)out % (out_kind == B200DEC_T_F32 ? 4 : 2) == 0,
               "w8a8_linear: alignment (images 1 KB, channel scales and bias 16 bytes)");
  W8Args a{};
  a.a = (const unsigned char*)rows_image, a.w = (const unsigned char*)weight_image, a.bias = bias;
  a.M = m, a.N = n, a.NKB = (k + 127) / 128, a.mode = 4, a.status = status;
  a.a_scale = row_scale, a.w_scale = w_scale, a.out = out, a.ldo = ldo, a.out_kind = out_kind, a.act = act;
  return launch(a, (cudaStream_t)stream);
}

int b200dec_w8a8_prefill(const void* rows_image, const float* row_scale, int m, int k, const void* weight_image,
                         const float* w_scale, const float* bias, int n, int mode, const int32_t* pieces, int n_pieces, void* ck,
                         void* cv, void* ck_scale, void* cv_scale, int layers, int slots_plus_1, int heads, int head_dim, int frames,
                         int32_t* status, void* stream) {
  B200_REQUIRE(rows_image && row_scale && weight_image && w_scale && status, "w8a8_prefill: null pointer");
  B200_REQUIRE(m >= 1 && m <= MAX_MN && k >= 1 && k <= MAX_K8 && mode >= 1 && mode <= 3, "w8a8_prefill: m %d k %d mode %d", m, k, mode);
  B200_REQUIRE(pieces && n_pieces >= 1 && ck && cv && (mode == 1 || (ck_scale && cv_scale)), "w8a8_prefill: pieces and caches");
  B200_REQUIRE((((uintptr_t)rows_image | (uintptr_t)weight_image) & 1023) == 0 &&
                   (((uintptr_t)w_scale | (uintptr_t)bias | (uintptr_t)pieces | (uintptr_t)ck | (uintptr_t)cv) & 15) == 0 &&
                   (mode == 1 || (((uintptr_t)ck_scale | (uintptr_t)cv_scale) & 3) == 0),
               "w8a8_prefill: alignment (images 1 KB, the caches' scales or pairs 4 bytes, the rest 16)");
  B200_REQUIRE((head_dim == 64 || head_dim == 128) && layers >= 1 && heads >= 1 && slots_plus_1 >= 1 && frames >= 1 &&
                   (int64_t)n == (int64_t)layers * 2 * heads * head_dim && n % BN == 0,
               "w8a8_prefill: n %d != layers %d x 2 x heads %d x head_dim %d (a multiple of 256)", n, layers, heads, head_dim);
  W8Args a{};
  a.a = (const unsigned char*)rows_image, a.w = (const unsigned char*)weight_image, a.bias = bias;
  a.M = m, a.N = n, a.NKB = (k + 127) / 128, a.mode = mode, a.status = status, a.a_scale = row_scale, a.w_scale = w_scale;
  a.pieces = (const int4*)pieces, a.n_pieces = n_pieces, a.ck = ck, a.cv = cv, a.cks = (float*)ck_scale, a.cvs = (float*)cv_scale;
  a.S1 = slots_plus_1, a.H = heads, a.D = head_dim, a.T = frames;
  return launch(a, (cudaStream_t)stream);
}

}  // extern "C"
