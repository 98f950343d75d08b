// Rules on the logits of a step, and the greedy choice under them: the penalties for tokens that a slot already has, the
// biases listed for it, its grammar mask, and the first index of the largest logit left.
//
//   x' = x / r or x * r (x > 0 or not) for a token among the slot's tokens so far, r the repetition penalty;
//   x' -= frequency * (times generated);  x' -= presence (where generated at all);  x' += the listed biases, added up in
//   the list's order;  x' = -inf where the mask's bit is 0. In fp32, each operation rounded once.
//
// A pass over the logits is all the memory sees; what a token has to its name must be at hand when its logit passes. A cluster
// of up to eight CTAs takes a row, each a contiguous range of the vocabulary. A CTA first marks in a bitmap in shared memory
// the tokens of its range that the slot has or that have a bias; a running count of the marks gives each of them a word in a
// dense table (as many as the slot has tokens, not as many as the vocabulary), where it is counted: low bits the times
// generated, bits for "seen" and "has a bias". All of it is integers, so the order of the atomics changes nothing. Then each
// marked token is settled by one thread: inside the stream they would sit in a few threads, since a text's tokens have ids
// near one another, and the rules' code would be there once per unrolled element. A token with a bias is settled from its
// entry of the list, one listed twice by adding its entries up in order. The stream passes over the marked tokens.
//
// What bounds it is the chain in front of the stream (row -> slot -> its parameters and tokens -> marks -> counts -> their
// logits), about 4 us, which every wave of CTAs pays again: so there are no more CTAs of a row than fit at once.
#include <cooperative_groups.h>

#include "common.cuh"

using namespace b200dec_detail;
namespace cg = cooperative_groups;

namespace {

constexpr uint32_t SEEN = 1u << 31, BIASED = 1u << 30, TWICE = 1u << 29, DONE = 1u << 28, TIMES = DONE - 1;
constexpr int MAX_BIAS = 1024, MAX_CLUSTER = 8, NONE = 0x7fffffff, NT = 512, CTAS_PER_SM = 2;
// vectors of a thread on their way: a power of two, so that j % RING is an AND (128 rows of 16384 logits 9.7 us, with six 10.0);
// two and eight were as fast there, eight slower on 96 rows of 151 931 (39.0 us instead of 37.8)
constexpr int RING = 4;
constexpr int SMEM_BUDGET = 100 * 1024;  // of a CTA: two per SM
constexpr int SMEM_RING = RING * NT * 16;
constexpr int SMEM_STATIC = (2 * MAX_CLUSTER + 3 * (NT / 32)) * 4;  // the kernel's own arrays: the row's and its warps' best, the warps' sums

static_assert(MAX_BIAS <= 2 * NT, "a thread stages two biases");

struct RulesArgs {
  const void* logits;
  void* out;
  int64_t ldl, ldo;
  const int* active;
  b200dec_rules r;
  float* best;
  int* token;
  int* status;
  const uint8_t* finished;  // null: every row's choice is taken; else (slots + 1): not that of a row that has ended or is fed its prompt
  int vocab, slots, range;  // range: positions of a CTA, a multiple of 32
  int tile, dense;          // positions marked at a time, a multiple of 32, and the words of their table
};

// Elements of a kind, and what the stream does to 32-bit words of them: it only takes the largest and writes -inf where a
// token is left out, so 16-bit elements stay in pairs.
template <int KIND>
struct Elem;
template <>
struct Elem<B200DEC_T_F32> {
  using type = float;
  static constexpr uint32_t NEG = 0xff800000u;
  static DEVI float load(float x) { return x; }
  static DEVI float store(float x) { return x; }
  static DEVI uint32_t max2(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
  static DEVI float top(uint32_t w) { return __uint_as_float(w); }
};
template <>
struct Elem<B200DEC_T_F16> {
  using type = __half;
  static constexpr uint32_t NEG = 0xfc00fc00u;
  static DEVI float load(__half x) { return __half2float(x); }
  static DEVI __half store(float x) { return __float2half_rn(x); }
  static DEVI uint32_t max2(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2(reinterpret_cast<const __half2&>(a), reinterpret_cast<const __half2&>(b));
    return reinterpret_cast<const uint32_t&>(m);
  }
  static DEVI float top(uint32_t w) {
    const float2 f = __half22float2(reinterpret_cast<const __half2&>(w));
    return fmaxf(f.x, f.y);
  }
};
template <>
struct Elem<B200DEC_T_BF16> {
  using type = __nv_bfloat16;
  static constexpr uint32_t NEG = 0xff80ff80u;
  static DEVI float load(__nv_bfloat16 x) { return __bfloat162float(x); }
  static DEVI __nv_bfloat16 store(float x) { return __float2bfloat16_rn(x); }
  static DEVI uint32_t max2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmax2(reinterpret_cast<const __nv_bfloat162&>(a), reinterpret_cast<const __nv_bfloat162&>(b));
    return reinterpret_cast<const uint32_t&>(m);
  }
  static DEVI float top(uint32_t w) { return fmaxf(bf16_lo(w), bf16_hi(w)); }
};

struct Best {
  float v;
  int i;
  DEVI void take(float ov, int oi) {
    if (ov > v || (ov == v && oi < i)) v = ov, i = oi;
  }
};

// Positions: u = v + pad, pad the distance in elements of the row's start from the 16-byte boundary before it, so that a vector of
// VEC positions is an aligned 16-byte load whatever the rows' distance (a vocabulary of odd size gives every row another pad).
// Positions below pad and from vocab + pad on hold other rows' logits or none at all: the vectors that reach them are read one
// element at a time.
template <int KIND>
__global__ void __launch_bounds__(NT, CTAS_PER_SM) logit_rules_kernel(const RulesArgs p) {
  using E = Elem<KIND>;
  using T = typename E::type;
  constexpr int VEC = 16 / (int)sizeof(T), STEP = NT * VEC;
  extern __shared__ __align__(16) uint32_t dyn_smem[];
  uint4* ring = reinterpret_cast<uint4*>(dyn_smem) + threadIdx.x;  // RING vectors of this thread's, NT apart
  uint32_t* smem = dyn_smem + SMEM_RING / 4;
  const int tile_words = p.tile / 32;
  uint32_t* marks = smem;                    // a bit per position of the tile
  uint32_t* words = marks + tile_words;      // the marked positions' words, in order
  uint32_t* before = words + p.dense;        // per word of marks: how many marks are before it
  int* b_id = reinterpret_cast<int*>(before + tile_words);
  __shared__ float s_best[MAX_CLUSTER];
  __shared__ int s_arg[MAX_CLUSTER];
  __shared__ float w_best[NT / 32];
  __shared__ int w_arg[NT / 32], w_sum[NT / 32];
  cluster_arrive_entry();
  cg::cluster_group cluster = cg::this_cluster();
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = blockIdx.x, ranks = gridDim.x;
  const T* row_at = reinterpret_cast<const T*>(p.logits) + row * p.ldl;
  const int pad = (int)(((uintptr_t)row_at & 15) / sizeof(T));
  const T* x = row_at - pad;  // only aligned from here on; its first pad elements are not this row's
  const int end = p.vocab + pad, u_first = rank * p.range, u_last = min(end, u_first + p.range);
  T* out = p.out ? reinterpret_cast<T*>(p.out) + row * p.ldo - pad : nullptr;
  const bool out_vec = ((uintptr_t)out & 15) == 0;  // the logits' rows and the results' lie alike
  const auto clear = [&] {
    for (int i = tid; i < tile_words + p.dense; i += NT) smem[i] = 0;
  };
  clear();
  pdl_wait();

  // vector j of this thread in a tile: on its way into the ring, if it is all this row's (the others are read when it is
  // their turn). Only its own thread reads it, so nothing but that thread's wait orders the ring.
  const auto fetch = [&](int j, int u0, int u1) {
    const int u = u0 + tid * VEC + j * STEP;
    if (u >= pad && u + VEC <= u1) cp_async16(ring + j % RING * NT, x + u);
    cp_async_commit();
  };
  int s = p.active[row];
  if (s < 0 || s > p.slots) {
    if (tid == 0 && rank == 0) atomicOr(p.status, B200DEC_ST_SLOT_RANGE);
    s = p.slots;
  }
  const int64_t* hist = p.r.history + (size_t)s * p.r.hist_cols;
  // read together with the row's parameters: most rows have tokens, and whether this one counts is known a round trip later
  const auto token = [&](int i) {  // -1: outside the vocabulary
    const int64_t tok = __ldg(hist + i);
    return tok >= 0 && tok < p.vocab ? (int)tok : -1;
  };
  const int early = tid < p.r.hist_cols ? token(tid) : -1;
  const int early_id = p.r.bias_ids && tid < p.r.max_bias ? __ldg(p.r.bias_ids + (size_t)s * p.r.max_bias + tid) : -1;
  const float early_val = p.r.bias_ids && tid < p.r.max_bias ? __ldg(p.r.bias + (size_t)s * p.r.max_bias + tid) : 0.f;
  const float4 par = *reinterpret_cast<const float4*>(p.r.params + 4 * (size_t)s);
  const int newest = p.r.last[s], plen = p.r.plen[s];
  const int nb = p.r.bias_ids ? max(0, min(p.r.bias_n[s], p.r.max_bias)) : 0;
  const uint32_t* mask = p.r.mask && (!p.r.mask_on || p.r.mask_on[s]) ? p.r.mask + (size_t)s * ((p.vocab + 31) / 32) : nullptr;
  const float rep = par.x, presence = par.y, frequency = par.z;
  const bool penal = rep != 1.f || presence != 0.f || frequency != 0.f;
  const int have = penal ? min(max(newest, -1), p.r.hist_cols - 1) + 1 : 0;  // tokens that count
  const bool touched = have > 0 || nb > 0;
  float* b_val = reinterpret_cast<float*>(b_id + nb);
  // The first logits come in while the slot's tokens are counted: two vectors behind the loads of its tables, the others when
  // those are there, so that a full memory queue does not stand in front of them.
#pragma unroll
  for (int j = 0; j < 2; ++j) fetch(j, u_first, min(u_last, u_first + p.tile));
  if (tid < nb) b_id[tid] = early_id, b_val[tid] = early_val;
  if (tid + NT < nb) {  // MAX_BIAS is 2 NT
    b_id[tid + NT] = p.r.bias_ids[(size_t)s * p.r.max_bias + tid + NT];
    b_val[tid + NT] = p.r.bias[(size_t)s * p.r.max_bias + tid + NT];
  }

  Best best{-INFINITY, NONE};
  for (int u0 = u_first; u0 < u_last; u0 += p.tile) {
    const int u1 = min(u_last, u0 + p.tile);
    if (touched) {
      const auto place = [&](int tok) {  // a token's position in this tile, or -1
        const int at = tok + pad - u0;
        return tok >= 0 && tok < p.vocab && at >= 0 && at < u1 - u0 ? at : -1;
      };
      const auto mark = [&](int at) { atomicOr(&marks[at >> 5], 1u << (at & 31)); };
      const auto word_of = [&](int at) {
        return words + before[at >> 5] + __popc(marks[at >> 5] & ((1u << (at & 31)) - 1));
      };
      const int early_at = tid < have ? place(early) : -1;
      if (u0 == u_first) {
#pragma unroll
        for (int j = 2; j < RING; ++j) fetch(j, u0, u1);
      }
      __syncthreads();  // all is zero (or the tile before is done with), the biases are in place
      if (u0 != u_first) {
        clear();
        __syncthreads();
      }
      if (early_at >= 0) mark(early_at);
      for (int i = tid + NT; i < have; i += NT)
        if (const int at = place(token(i)); at >= 0) mark(at);
      for (int i = tid; i < nb; i += NT)
        if (const int at = place(b_id[i]); at >= 0) mark(at);
      __syncthreads();
      {  // the running count of the marks: a run of words per thread
        const int per = (tile_words + NT - 1) / NT, w0 = min(tid * per, tile_words), w1 = min(w0 + per, tile_words);
        int sum = 0;
        for (int w = w0; w < w1; ++w) sum += __popc(marks[w]);
        int upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        if (lane == 31) w_sum[warp] = upto;
        __syncthreads();
        int run = upto - sum;
        run += (int)__reduce_add_sync(0xffffffffu, lane < warp ? (unsigned)w_sum[lane] : 0u);
        for (int w = w0; w < w1; ++w) before[w] = run, run += __popc(marks[w]);
      }
      __syncthreads();
      const auto count = [&](int i, int at) {
        if (i >= plen) atomicAdd(word_of(at), 1u);
        else atomicOr(word_of(at), SEEN);
      };
      if (early_at >= 0) count(tid, early_at);
      for (int i = tid + NT; i < have; i += NT)
        if (const int at = place(token(i)); at >= 0) count(i, at);
      for (int i = tid; i < nb; i += NT)
        if (const int at = place(b_id[i]); at >= 0)
          if (uint32_t* w = word_of(at); atomicOr(w, BIASED) & BIASED) atomicOr(w, TWICE);
      __syncthreads();
      // Every marked token, once: one with a bias by a thread that has an entry of it, the others by whoever says so first. Its
      // logit and mask word are asked for only then, one token after the other: a text says the same things, so most of a
      // history's tokens are settled by another thread. Asking for all of a thread's at once, before they are counted, took
      // 7.3 us for a row of 217 tokens and 12.2 us for 128 of 457 (16384 logits) instead of 6.2 and 10.0: more requests and code.
      const auto claim = [&](int at, bool biased) -> uint32_t {  // the token's word if it is this thread's to settle, else 0
        uint32_t* word = word_of(at);
        const uint32_t w = *word;
        if ((w & DONE) || (!biased && (w & BIASED))) return 0;
        return atomicOr(word, DONE) & DONE ? 0 : w;
      };
      const auto settle = [&](int at, uint32_t w, T raw_x, uint32_t word, int entry) {
        const int u = u0 + at, v = u - pad;
        float f = E::load(raw_x);
        if (w & (SEEN | TIMES)) {
          f = f > 0.f ? __fdiv_rn(f, rep) : __fmul_rn(f, rep);
          const uint32_t n = w & TIMES;
          if (n) f = __fsub_rn(__fsub_rn(f, __fmul_rn(frequency, (float)n)), presence);
        }
        if (entry >= 0) {
          float sum = b_val[entry];
          if (w & TWICE) {  // added up in the list's order, whichever entry's thread this is
            sum = 0.f;
            for (int i = 0; i < nb; ++i)
              if (b_id[i] == v) sum += b_val[i];
          }
          f = __fadd_rn(f, sum);
        }
        if (!(word >> (v & 31) & 1)) f = -INFINITY;
        if (f > -INFINITY) best.take(f, v);
        if (out) out[u] = E::store(f);
      };
      const auto logit = [&](int at) { return __ldcg(x + u0 + at); };
      const auto mask_word = [&](int at) { return mask ? __ldg(mask + ((u0 + at - pad) >> 5)) : 0xffffffffu; };
#pragma unroll 1
      for (int i = tid; i < have + nb; i += NT) {  // the tokens that count, then the biases
        const int entry = i < have ? -1 : i - have;
        const int at = entry >= 0 ? place(b_id[entry]) : i < NT ? early_at : place(token(i));
        if (at < 0) continue;
        if (const uint32_t w = claim(at, entry >= 0); w) settle(at, w, logit(at), mask_word(at), entry);
      }
    }
    if (u0 != u_first || !touched) {
#pragma unroll
      for (int j = 0; j < RING; ++j)
        if (u0 != u_first || j >= 2) fetch(j, u0, u1);
    }
    // bit i of mine: position u + i is this row's and not settled; of the result: and the mask allows it
    const auto allowed = [&](int u, uint32_t& mine) {
      mine = (1u << VEC) - 1;
      if (u < pad) mine &= mine << (pad - u);
      if (u + VEC > u1) mine &= (1u << (u1 - u)) - 1;
      if (touched) mine &= ~(marks[(u - u0) >> 5] >> (u & 31));  // u0 is a multiple of 32
      if (!mask) return mine;
      // VEC bits from token v on: of one word, or two
      const int v = u - pad, w = max(v, 0) >> 5, z = (p.vocab - 1) >> 5;
      const uint32_t lo = __ldg(mask + min(w, z)), hi = pad ? __ldg(mask + min(w + 1, z)) : 0;
      return mine & (v < 0 ? lo << -v : __funnelshift_r(lo, hi, v & 31));
    };
    float stream = -INFINITY;  // the largest that streams by in this tile, and the vector that had it first
    int stream_u = -1;
    uint32_t mine, left = 0;
    if (u0 + tid * VEC < u1) left = allowed(u0 + tid * VEC, mine);
#pragma unroll 1
    for (int j = 0, u = u0 + tid * VEC; u < u1; ++j, u += STEP) {
      const bool whole = u >= pad && u + VEC <= u1;
      union {
        uint4 q;
        uint32_t w[4];
        T e[VEC];
      } raw;
      cp_async_wait_group<RING - 1>();
      if (whole) raw.q = ring[j % RING * NT];
      else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) raw.e[i] = u + i >= pad && u + i < u1 ? __ldcg(x + u + i) : T(0.f);
      }
      fetch(j + RING, u0, u1);
      const uint32_t now = left, stored = mine;
      if (u + STEP < u1) left = allowed(u + STEP, mine);  // the next one's, so that its mask is there in time
      if (now != (1u << VEC) - 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t keep;
          if constexpr (VEC == 4) keep = (uint32_t)((int)(now << (31 - i)) >> 31);
          else keep = __byte_perm((uint32_t)((int)(now << (31 - 2 * i)) >> 31), (uint32_t)((int)(now << (30 - 2 * i)) >> 31), 0x5410);
          raw.w[i] = (raw.w[i] & keep) | (E::NEG & ~keep);
        }
      }
      const float top = E::top(E::max2(E::max2(raw.w[0], raw.w[1]), E::max2(raw.w[2], raw.w[3])));
      if (top > stream) stream = top, stream_u = u;
      if (out) {
        if (out_vec && stored == (1u << VEC) - 1) {
          *reinterpret_cast<uint4*>(out + u) = raw.q;
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (stored >> i & 1) out[u + i] = raw.e[i];
        }
      }
    }
    if (stream_u >= 0) {  // which of the vector's tokens: the first
      left = allowed(stream_u, mine);
      T e[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = (left >> i & 1) ? __ldcg(x + stream_u + i) : T(0.f);
      int first = 0;
#pragma unroll
      for (int i = VEC - 1; i >= 0; --i)
        if ((left >> i & 1) && E::load(e[i]) == stream) first = i;
      best.take(stream, stream_u + first - pad);
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
      if (s < p.slots && (!p.finished || (!p.finished[s] && p.r.last[s] + 1 >= p.r.plen[s]))) atomicOr(p.status, B200DEC_ST_NO_TOKEN);
    }
    p.token[row] = all.i;
    if (p.best) p.best[row] = all.v;
  }
}

template <int KIND>
cudaError_t launch_rules(const RulesArgs& p, int rows, int cluster, int nb, cudaStream_t st, int pdl) {
  const size_t smem = SMEM_RING + (size_t)p.tile / 4 + (size_t)p.dense * 4 + (size_t)nb * 8;
  if (smem + SMEM_STATIC > 48 * 1024) {  // what a CTA has unasked holds the static arrays too
    const cudaError_t e = cudaFuncSetAttribute(logit_rules_kernel<KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BUDGET);
    if (e != cudaSuccess) return e;
  }
  return launch_kernel(logit_rules_kernel<KIND>, dim3(cluster, rows), dim3(NT), smem, st, cluster, pdl, p);
}

}  // namespace

namespace b200dec_detail {

int logit_rules_impl(const void* logits, int kind, int64_t ldl, int rows, int vocab, const int32_t* active, int slots,
                     const b200dec_rules* rules, void* out, int64_t ldo, float* best, int32_t* token, int32_t* status,
                     const uint8_t* finished, int pdl, void* stream) {
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
  const int size = kind == B200DEC_T_F32 ? 4 : 2;
  B200_REQUIRE(((uintptr_t)logits % size) == 0 && ((uintptr_t)out % size) == 0, "logit_rules: alignment");
  // CTAs of a row: a power of two, as long as all rows' fit at once (clusters have to lie in one part of the chip, so not every
  // place can be taken) and each has 2048 tokens or more. 96 rows of 151 931 bf16 logits, 2100 tokens: 51 us with one CTA a
  // row, 38 with two (this rule), 41 with three, 43 with four
  int cluster = 1;
  while (cluster < MAX_CLUSTER && rows * cluster * 2 <= CTAS_PER_SM * 148 * 9 / 10 && vocab / (cluster * 2) >= 2048) cluster *= 2;
  RulesArgs p{logits, out, ldl, ldo, active, *rules, best, token, status, finished, vocab, slots, 0, 0, 0};
  p.range = ((vocab + 7 + cluster - 1) / cluster + 31) / 32 * 32;  // of vocab + pad positions
  // a position takes 8 / 32 bytes of marks and counts, a marked one a word: no more of those than tokens and biases, or positions
  const int nb = rules->bias_ids ? rules->max_bias : 0;
  const int64_t entries = (int64_t)rules->hist_cols + nb, room = SMEM_BUDGET - SMEM_RING - nb * 8;
  const int64_t fit = entries * 4 <= room / 2 ? (room - entries * 4) * 4 : room * 4 / 17;
  p.tile = (int)(fit < p.range ? fit / 32 * 32 : p.range);
  p.dense = (int)(entries < p.tile ? entries : p.tile);
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (kind == B200DEC_T_F32) e = launch_rules<B200DEC_T_F32>(p, rows, cluster, nb, st, pdl);
  else if (kind == B200DEC_T_F16) e = launch_rules<B200DEC_T_F16>(p, rows, cluster, nb, st, pdl);
  else e = launch_rules<B200DEC_T_BF16>(p, rows, cluster, nb, st, pdl);
  if (e != cudaSuccess) return fail(B200DEC_ECUDA, "logit_rules launch: %s", cudaGetErrorString(e));
  return 0;
}

}  // namespace b200dec_detail

extern "C" int b200dec_logit_rules(const void* logits, int kind, int64_t ldl, int rows, int vocab, const int32_t* active, int slots,
                                   const b200dec_rules* rules, void* out, int64_t ldo, float* best, int32_t* token,
                                   int32_t* status, int pdl, void* stream) {
  return logit_rules_impl(logits, kind, ldl, rows, vocab, active, slots, rules, out, ldo, best, token, status, nullptr, pdl, stream);
}
