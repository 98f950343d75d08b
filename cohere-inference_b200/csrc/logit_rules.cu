// Rules on the logits of a step, and the greedy choice under them: the penalties for tokens that a slot already has, the
// biases listed for it, its grammar mask, and the first index of the largest logit left.
//
//   x' = x / r or x * r (x > 0 or not) for a token among the slot's tokens so far, r the repetition penalty;
//   x' -= frequency * (times generated);  x' -= presence (where generated at all);  x' += the listed biases, added up in
//   the list's order;  x' = -inf where the mask's bit is 0. In fp32, each operation rounded once.
//
// A pass over the logits is all the memory sees; what a token has to its name must be at hand when its logit passes. A cluster
// of up to eight CTAs takes a row, each a contiguous range of the vocabulary, and first counts in shared memory the slot's
// tokens that fall into its range: one 32-bit word per token, its low bits the times generated, one bit for "seen" and one for
// "has a bias". The counts are integers, so the order of the atomics changes nothing. A token with a bias looks its entries
// up in the list, in order, so a token listed twice gets both. No table per slot and token is kept between the steps: the
// tokens themselves are 100 times smaller.
#include <cooperative_groups.h>

#include "common.cuh"

using namespace b200dec_detail;
namespace cg = cooperative_groups;

namespace {

constexpr uint32_t SEEN = 1u << 31, BIASED = 1u << 30, TIMES = BIASED - 1;
constexpr int MAX_BIAS = 1024, MAX_CLUSTER = 8, TILE_MAX = 32768, NONE = 0x7fffffff;

struct RulesArgs {
  const void* logits;
  void* out;
  int64_t ldl, ldo;
  const int* active;
  b200dec_rules r;
  float* best;
  int* token;
  int* status;
  int vocab, slots, range, tile;  // range: tokens of a CTA, a multiple of 32; tile: of them counted at a time
};

template <int KIND>
struct Elem;
template <>
struct Elem<B200DEC_T_F32> {
  using type = float;
  static DEVI float load(float x) { return x; }
  static DEVI float store(float x) { return x; }
};
template <>
struct Elem<B200DEC_T_F16> {
  using type = __half;
  static DEVI float load(__half x) { return __half2float(x); }
  static DEVI __half store(float x) { return __float2half_rn(x); }
};
template <>
struct Elem<B200DEC_T_BF16> {
  using type = __nv_bfloat16;
  static DEVI float load(__nv_bfloat16 x) { return __bfloat162float(x); }
  static DEVI __nv_bfloat16 store(float x) { return __float2bfloat16_rn(x); }
};

struct Best {
  float v;
  int i;
  DEVI void take(float ov, int oi) {
    if (ov > v || (ov == v && oi < i)) v = ov, i = oi;
  }
};

template <int KIND, bool VECTOR, int NT>
__global__ void __launch_bounds__(NT) logit_rules_kernel(const RulesArgs p) {
  using E = Elem<KIND>;
  using T = typename E::type;
  constexpr int VEC = VECTOR ? 16 / (int)sizeof(T) : 1, UNROLL = VECTOR ? 4 : 8;
  extern __shared__ __align__(16) uint32_t words[];  // tile counts, then the slot's biases
  __shared__ float s_best[MAX_CLUSTER];
  __shared__ int s_arg[MAX_CLUSTER];
  __shared__ float w_best[NT / 32];
  __shared__ int w_arg[NT / 32];
  cluster_arrive_entry();
  cg::cluster_group cluster = cg::this_cluster();
  const int row = blockIdx.y, tid = threadIdx.x, rank = blockIdx.x, ranks = gridDim.x;
  pdl_wait();

  int s = p.active[row];
  if (s < 0 || s > p.slots) {
    if (tid == 0 && rank == 0) atomicOr(p.status, B200DEC_ST_SLOT_RANGE);
    s = p.slots;
  }
  const float4 par = *reinterpret_cast<const float4*>(p.r.params + 4 * (size_t)s);
  const float rep = par.x, presence = par.y, frequency = par.z;
  const bool penal = rep != 1.f || presence != 0.f || frequency != 0.f;
  const int have = penal ? min(p.r.last[s], p.r.hist_cols - 1) + 1 : 0;  // tokens that count
  const int plen = p.r.plen[s];
  const int64_t* hist = p.r.history + (size_t)s * p.r.hist_cols;
  const int nb = p.r.bias_ids ? max(0, min(p.r.bias_n[s], p.r.max_bias)) : 0;
  const uint32_t* mask = p.r.mask && (!p.r.mask_on || p.r.mask_on[s]) ? p.r.mask + (size_t)s * ((p.vocab + 31) / 32) : nullptr;
  const bool touched = have > 0 || nb > 0;
  int* b_id = reinterpret_cast<int*>(words + p.tile);
  float* b_val = reinterpret_cast<float*>(b_id + nb);
  for (int i = tid; i < nb; i += NT) {
    b_id[i] = p.r.bias_ids[(size_t)s * p.r.max_bias + i];
    b_val[i] = p.r.bias[(size_t)s * p.r.max_bias + i];
  }

  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.ldl;
  T* out = p.out ? reinterpret_cast<T*>(p.out) + row * p.ldo : nullptr;
  Best best{-INFINITY, NONE};
  const int last = min(p.vocab, (rank + 1) * p.range);
  for (int v0 = rank * p.range; v0 < last; v0 += p.tile) {
    const int v1 = min(last, v0 + p.tile);
    if (touched) {
      __syncthreads();  // the counts may still be read for the tile before; and the biases are in place
      for (int i = tid; i < (v1 - v0 + 3) / 4; i += NT) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      for (int i = tid; i < have; i += NT) {
        const int64_t tok = __ldg(hist + i);
        if (tok >= v0 && tok < v1) {
          if (i >= plen) atomicAdd(&words[tok - v0], 1u);
          else atomicOr(&words[tok - v0], SEEN);
        }
      }
      for (int i = tid; i < nb; i += NT)
        if (b_id[i] >= v0 && b_id[i] < v1) atomicOr(&words[b_id[i] - v0], BIASED);
      __syncthreads();
    }
    // one token's logit under the rules
    const auto apply = [&](float f, int v, uint32_t w) {
      if (w & ~BIASED) {
        f = f > 0.f ? __fdiv_rn(f, rep) : __fmul_rn(f, rep);
        const uint32_t n = w & TIMES;
        if (n) f = __fsub_rn(__fsub_rn(f, __fmul_rn(frequency, (float)n)), presence);
      }
      if (w & BIASED) {
        float b = 0.f;
        for (int i = 0; i < nb; ++i)
          if (b_id[i] == v) b += b_val[i];
        f = __fadd_rn(f, b);
      }
      return f;
    };
    for (int at = v0 + tid * VEC; at < v1; at += NT * VEC * UNROLL) {
      T raw[UNROLL][VEC];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int v = at + u * NT * VEC;
        if constexpr (VECTOR) {
          // v1 is a multiple of the vector or the end of the row; a vector across the end is taken one by one
          if (v + VEC <= v1) {
            const uint4 w = __ldcg(reinterpret_cast<const uint4*>(x + v));
            memcpy(raw[u], &w, 16);
          } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) raw[u][i] = v + i < v1 ? __ldcg(x + v + i) : T(0.f);
          }
        } else {
          raw[u][0] = v < v1 ? __ldcg(x + v) : T(0.f);
        }
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int v = at + u * NT * VEC;
        if (v >= v1) continue;
        const uint32_t bits = mask ? __ldg(mask + (v >> 5)) >> (v & 31) : 0xffffffffu;
        float f[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = E::load(raw[u][i]);
        if (touched) {
          uint32_t w[VEC], any = 0;
#pragma unroll
          for (int i = 0; i < VEC; ++i) w[i] = words[v - v0 + i], any |= w[i];
          if (any) {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
              if (w[i] && v + i < v1) f[i] = apply(f[i], v + i, w[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          if (!(bits >> i & 1)) f[i] = -INFINITY;
          if (f[i] > best.v && v + i < v1) best.v = f[i], best.i = v + i;  // ascending: the first of equals stays
        }
        if (out) {
          T o[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) o[i] = E::store(f[i]);
          if (VECTOR && v + VEC <= v1) {
            uint4 w;
            memcpy(&w, o, 16);
            *reinterpret_cast<uint4*>(out + v) = w;
          } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
              if (v + i < v1) out[v + i] = o[i];
          }
        }
      }
    }
  }
  // the row's first largest: over the warp, the CTA, the cluster
#pragma unroll
  for (int o = 16; o; o >>= 1)
    best.take(__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o));
  if ((tid & 31) == 0) w_best[tid >> 5] = best.v, w_arg[tid >> 5] = best.i;
  pdl_trigger();
  __syncthreads();
  cluster_wait_entry();
  if (tid == 0) {
    for (int i = 1; i < NT / 32; ++i) best.take(w_best[i], w_arg[i]);
    *cluster.map_shared_rank(&s_best[rank], 0) = best.v;
    *cluster.map_shared_rank(&s_arg[rank], 0) = best.i;
  }
  cluster.sync();
  if (rank == 0 && tid == 0) {
    Best all{-INFINITY, NONE};
    for (int i = 0; i < ranks; ++i) all.take(s_best[i], s_arg[i]);
    if (all.i == NONE) {  // nothing above -inf: the first token, and said so
      all.i = 0;
      if (s < p.slots) atomicOr(p.status, B200DEC_ST_NO_TOKEN);
    }
    p.token[row] = all.i;
    if (p.best) p.best[row] = all.v;
  }
}

template <int KIND, bool VECTOR>
cudaError_t launch_rules(const RulesArgs& p, int rows, int cluster, int nb, cudaStream_t st, int pdl) {
  const size_t smem = (size_t)p.tile * 4 + (size_t)nb * 8;
  const dim3 grid(cluster, rows);
  const auto go = [&](auto kern, int threads) {
    if (smem > 48 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TILE_MAX * 4 + MAX_BIAS * 8);
      if (e != cudaSuccess) return e;
    }
    return launch_kernel(kern, grid, dim3(threads), smem, st, cluster, pdl, p);
  };
  return p.tile > 8192 ? go(logit_rules_kernel<KIND, VECTOR, 512>, 512) : go(logit_rules_kernel<KIND, VECTOR, 256>, 256);
}

}  // namespace

namespace b200dec_detail {

int logit_rules_impl(const void* logits, int kind, int64_t ldl, int rows, int vocab, const int32_t* active, int slots,
                     const b200dec_rules* rules, void* out, int64_t ldo, float* best, int32_t* token, int32_t* status, int pdl,
                     void* stream) {
  B200_REQUIRE(logits && active && rules && token && status, "logit_rules: null pointer");
  B200_REQUIRE(kind == B200DEC_T_F32 || kind == B200DEC_T_F16 || kind == B200DEC_T_BF16, "logit_rules: kind %d", kind);
  B200_REQUIRE(rows >= 1 && rows <= 65535 && vocab >= 1 && vocab <= 1 << 24 && slots >= 0 && ldl >= vocab && (!out || ldo >= vocab),
               "logit_rules: rows %d vocab %d slots %d rows of %lld / %lld", rows, vocab, slots, (long long)ldl, (long long)ldo);
  B200_REQUIRE(rules->params && ((uintptr_t)rules->params & 15) == 0 && rules->history && rules->last && rules->plen &&
                   rules->hist_cols >= 1, "logit_rules: the penalties (16-byte aligned) and the slots' tokens are needed");
  B200_REQUIRE((rules->bias_ids == nullptr) == (rules->bias == nullptr) && (rules->bias_ids == nullptr) == (rules->bias_n == nullptr),
               "logit_rules: a bias list is ids, values and counts");
  B200_REQUIRE(!rules->bias_ids || (rules->max_bias >= 1 && rules->max_bias <= MAX_BIAS), "logit_rules: max_bias %d (1..%d)",
               rules->max_bias, MAX_BIAS);
  const int size = kind == B200DEC_T_F32 ? 4 : 2, vec = 16 / size;
  B200_REQUIRE(((uintptr_t)logits % size) == 0 && ((uintptr_t)out % size) == 0, "logit_rules: alignment");
  const bool vector = ((uintptr_t)logits & 15) == 0 && (rows == 1 || ldl % vec == 0) &&
                      (!out || (((uintptr_t)out & 15) == 0 && (rows == 1 || ldo % vec == 0)));
  // CTAs of a row: about four per SM in all, each with 2048 tokens or more
  int cluster = 1;
  while (cluster < MAX_CLUSTER && (int64_t)rows * cluster < 4 * 148 && vocab / (cluster * 2) >= 2048) cluster *= 2;
  RulesArgs p{logits, out, ldl, ldo, active, *rules, best, token, status, vocab, slots, 0, 0};
  p.range = ((vocab + cluster - 1) / cluster + 31) / 32 * 32;
  p.tile = p.range < TILE_MAX ? p.range : TILE_MAX;
  const int nb = rules->bias_ids ? rules->max_bias : 0;
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (kind == B200DEC_T_F32) e = vector ? launch_rules<B200DEC_T_F32, true>(p, rows, cluster, nb, st, pdl)
                                        : launch_rules<B200DEC_T_F32, false>(p, rows, cluster, nb, st, pdl);
  else if (kind == B200DEC_T_F16) e = vector ? launch_rules<B200DEC_T_F16, true>(p, rows, cluster, nb, st, pdl)
                                             : launch_rules<B200DEC_T_F16, false>(p, rows, cluster, nb, st, pdl);
  else e = vector ? launch_rules<B200DEC_T_BF16, true>(p, rows, cluster, nb, st, pdl)
                  : launch_rules<B200DEC_T_BF16, false>(p, rows, cluster, nb, st, pdl);
  if (e != cudaSuccess) return fail(B200DEC_ECUDA, "logit_rules launch: %s", cudaGetErrorString(e));
  return 0;
}

}  // namespace b200dec_detail

extern "C" int b200dec_logit_rules(const void* logits, int kind, int64_t ldl, int rows, int vocab, const int32_t* active, int slots,
                                   const b200dec_rules* rules, void* out, int64_t ldo, float* best, int32_t* token,
                                   int32_t* status, int pdl, void* stream) {
  return logit_rules_impl(logits, kind, ldl, rows, vocab, active, slots, rules, out, ldo, best, token, status, pdl, stream);
}
