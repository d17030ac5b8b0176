// The router of a MoE layer on gfx950: which experts a token goes to and with what weight, how the
// tokens spread over the experts (counts and balance loss), and the gradient of both by the logits.
//
// Scores of a row's logits l: s = softmax(l), sigmoid(l) or sqrt(softplus(l)). A NaN logit counts as
// -inf and +inf as the largest float, so every score is a finite number; a row of -inf alone scores 0.
//
// Selection: the choice value c is the logit itself without a correction bias (every score grows
// with its logit) and s + bias in 64 bits with one: which of two experts wins a close race then is
// a matter of the formula and not of a 32-bit exponential's last bit. Equal values go to the lower index.
// With a bias the choice is first made in fp32 and its margins are compared with twice the fp32
// error's bound; only rows with a margin inside it (a few in a thousand; rows with equal values) are
// settled in 64 bits.
//
// Balance loss of a sequence with T rows: L_s = E / (k T) sum_e cnt_e P_e, P_e = 1/T sum_t s'_te,
// s' = s / sum_e s; L = alpha times the mean of L_s over the sequences that have rows.
//   dL/dl_te = s'_te r(l_te) (c_e - sum_j c_j s'_tj),  c_e = gloss coef cnt_e,
//   coef = alpha E / (S' k T^2),  r = 1, 1 - sigmoid(l), sigmoid(l) / (2 softplus(l)),
// with c counted from the row's largest share's, as whole numbers (16384 x 256 with the weights' gradient 15.5 us without
// that step, 16.2 with it, in turn).
//
// Layout: W lanes hold one row, lane i experts [V i, V i + V), so the lanes' order is the experts'
// and a lane's V logits are wide loads: 16 lanes (4 rows a wavefront) up to 64 experts, 32 up to 128,
// else 64 lanes with V = 4, 8 or 16; a choice of many rows takes 16 or 32 lanes up to 512 experts. A
// lane sorts its values once; a pick is then a max butterfly (DPP and permlane swaps) over the lanes' heads.
// What is counted of its time is instructions, not bytes: 16384 x 256 with a bias and 4 of 8 groups takes 17 to 20 us (830
// VALU instructions for two rows, 11 us of issue, the rest not accounted for; its 18 MB 3.7 us), by the logits alone 9.7;
// few rows a launch and its latency (8 x 256 4.4, where a launch that does nothing takes 1.4 to 1.6).
//
// Sums over rows: a workgroup takes R consecutive rows, cut where sequences begin and end; each piece
// writes its sums and counts to a slot of its own (slot = workgroup + sequence: from one piece to the
// next one of the two grows), and a second launch adds a sequence's slots in their order. No sum
// depends on which workgroup ends first. With the choice 16384 x 256 takes 22.4 us and 9.6 for the second launch (of
// which 1.5 are any launch's, the rest dependent reads: slots, ticket, parts), the gradient, again one pass, 16.2 (34
// MB); given ids, 8192 x 64 6.7, 9.0 and 7.7 (traced medians; in a graph, forward and gradient, 47.1 and 24.6 in all).
#include "afd_common.h"
#include "afd_internal.h"

namespace afd {
namespace router {

constexpr int kThreads = 256;
// threads of a workgroup that fills a slot: many where a row takes a wavefront (16384 x 256: the second
// launch 9.0 us with 1024 threads and 256 slots, 12.5 with 512 and 512), fewer where it takes less (8192 x
// 64: the first launch 6.6 us with 512, 9.0 with 1024) or where lanes hold many experts (registers, LDS)
__host__ __device__ constexpr int balance_threads(int W, int V) { return W == 64 && V == 4 ? 1024 : 512; }
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopk = 32;
constexpr int kMaxGroups = 64;
constexpr int kMaxSeqs = 1 << 20;
constexpr int kMaxRows = 1 << 26;
// rows a workgroup's slot sums at most: the sums are fp32, their error grows with the terms
constexpr int kMaxBlockRows = 1024;

struct Args {
  const void* logits;
  int64_t ld;
  const float* bias;
  const uint8_t* valid;
  int32_t n;
  int32_t experts, topk, scoring, groups, keep, renorm;
  int32_t group_lanes;  // lanes that make a group's value, a power of two
  bool whole_lanes;     // ... and hold its experts
  bool wide;            // rows take 4-element loads and stores
  float scale;
  int32_t* ids;  // selection: written; balance and gradient: read
  float* w;
  // balance
  const int32_t* cu;  // [seqs + 1], or nullptr: one sequence of all rows
  int32_t seqs;
  int32_t block_rows, blocks;
  float alpha;
  float* slots;  // [blocks + seqs] of slot_words(experts)
  int32_t* counts;
  float* coef;
  double* part;      // [seqs][chunks of experts] unscaled losses
  int32_t* rows;     // [seqs] rows
  uint32_t* ticket;  // workgroups of the second launch that are done
  float* loss;
  // gradient
  const float* gw;
  const float* gloss;
  void* dlogits;
};

// sums f32 [E], counts i32 [E], rows i32 (and 3 words of padding)
__host__ __device__ inline int64_t slot_words(int experts) { return 2 * int64_t(experts) + 4; }

// ---------------------------------------------------------------- reductions over W lanes
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true));
}
constexpr int kBcast15 = 0x142, kBcast31 = 0x143;
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;

// f(own, partner) over the lanes of a row; every lane gets the same bits (f commutes). After the
// quads agree, a mirrored half row is the exchange with the other quad, and so on. Over a whole
// wavefront the last two steps only gather towards lane 63, whose value is read into a scalar: every
// step is then one instruction with its DPP operand.
template <int W, typename F>
__device__ __forceinline__ uint32_t reduce32(uint32_t v, F f) {
  v = f(v, dpp<kXor1>(v));
  v = f(v, dpp<kXor2>(v));
  v = f(v, dpp<kHalfMirror>(v));
  v = f(v, dpp<kMirror>(v));
  if constexpr (W == 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f(r[0], r[1]);
  }
  if constexpr (W == 64) {
    // row 0's lane 15 into row 1 (and row 2's into row 3), then lane 31 into rows 2 and 3: lane 63 has all
    v = f(v, dpp<kBcast15>(v));
    v = f(v, dpp<kBcast31>(v));
    v = __builtin_amdgcn_readlane(v, 63);
  }
  return v;
}
template <int W>
__device__ __forceinline__ uint32_t max_u32(uint32_t v) {
  return reduce32<W>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int W>
__device__ __forceinline__ float max_f32(float v) {
  return __uint_as_float(reduce32<W>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
template <int W>
__device__ __forceinline__ float sum_f32(float v) {
  return __uint_as_float(reduce32<W>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = dpp<CTRL>(static_cast<uint32_t>(u)), hi = dpp<CTRL>(static_cast<uint32_t>(u >> 32));
  return __builtin_bit_cast(double, lo | hi << 32);
}
template <int W>
__device__ __forceinline__ double sum_f64(double v) {
  v += dpp_f64<kXor1>(v);
  v += dpp_f64<kXor2>(v);
  v += dpp_f64<kHalfMirror>(v);
  v += dpp_f64<kMirror>(v);
  auto halves = [](uint64_t u, auto swap) {
    const auto l = swap(static_cast<uint32_t>(u)), h = swap(static_cast<uint32_t>(u >> 32));
    return __builtin_bit_cast(double, uint64_t(l[0]) | uint64_t(h[0]) << 32) +
           __builtin_bit_cast(double, uint64_t(l[1]) | uint64_t(h[1]) << 32);
  };
  if constexpr (W >= 32)
    v = halves(__builtin_bit_cast(uint64_t, v),
               [](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
  if constexpr (W >= 64)
    v = halves(__builtin_bit_cast(uint64_t, v),
               [](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
  return v;
}

// ---------------------------------------------------------------- keys: unsigned order = value order
// key 0 is below every number's: an expert that is not there, already taken, or in a dropped group
__device__ __forceinline__ uint32_t key32(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);  // -0 and +0 are equal
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key ^ (~static_cast<uint32_t>(static_cast<int32_t>(key) >> 31) | 0x80000000u));
}
__device__ __forceinline__ double value_of(uint64_t key) {
  return __builtin_bit_cast(double, key ^ (~static_cast<uint64_t>(static_cast<int64_t>(key) >> 63) | 0x8000000000000000ull));
}
__device__ __forceinline__ uint64_t key64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
  return u ^ (static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | 0x8000000000000000ull);
}

// ---------------------------------------------------------------- scores
constexpr float kLowest = -__builtin_huge_valf();
constexpr float kLeast = 0x1p-126f;  // sums below it count as 0: their reciprocal may leave the floats
__device__ __forceinline__ float logit_f32(const float* p) { return *p; }
__device__ __forceinline__ float logit_f32(const uint16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float canon(float v) {
  return v != v ? kLowest : fminf(v, 3.402823466e38f);
}
// e^x from the hardware's 2^x: the product x log2(e) in two parts, the small one to first order, which
// keeps the relative error at two ulps for |x| <= 87.3; past that, where it is left out, 20 (0 below 2^-126)
__device__ __forceinline__ float exp_f32(float x) {
  constexpr float kLog2e = 1.44269502f, kLog2eLo = 1.92596299e-8f, kLn2 = 0.693147182f;
  const float t = x * kLog2e;
  float rest = __builtin_fmaf(x, kLog2e, -t);
  rest = __builtin_fmaf(x, kLog2eLo, rest);
  const float y = __builtin_amdgcn_exp2f(t);
  // no correction where t has left the floats
  return fabsf(t) < 126.0f ? __builtin_fmaf(y, rest * kLn2, y) : y;
}
// e^x to (|x| + 2) 2^-24 relative, an instruction instead of four: for terms of a row's sum and shares, of which the large
// ones have a small x. A gradient's entry carries the error of its own share and of its slope: 2^-18 where |x| is 40.
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.44269502f); }
// log(1 + e) for e in [0, 1]: 2 atanh(z), z = e / (2 + e) <= 1/3, by its series up to z^15 (the
// first term left out is (1/9)^8 / 17 of the sum, below 2^-29)
__device__ __forceinline__ float log1p_f32(float e) {
  const float z = e * __builtin_amdgcn_rcpf(2.0f + e), q = z * z;
  float p = 1.0f / 15.0f;
  p = __builtin_fmaf(p, q, 1.0f / 13.0f);
  p = __builtin_fmaf(p, q, 1.0f / 11.0f);
  p = __builtin_fmaf(p, q, 1.0f / 9.0f);
  p = __builtin_fmaf(p, q, 1.0f / 7.0f);
  p = __builtin_fmaf(p, q, 1.0f / 5.0f);
  p = __builtin_fmaf(p, q, 1.0f / 3.0f);
  const float h = z + z;
  return __builtin_fmaf(h * q, p, h);
}
// sigmoid or sqrt(softplus); the latter is e^(v/2) (1 - e^v / 4 + ..) of a small v, whose e^v may have left the floats
constexpr float kSmall = -17.0f;
template <bool EXACT>
__device__ __forceinline__ float score_f32(float v, int scoring) {
  auto e_to = [](float x) { return EXACT ? exp_f32(x) : exp_fast(x); };
  if (scoring == AFD_SCORE_SIGMOID) return __builtin_amdgcn_rcpf(1.0f + e_to(-v));
  const float e = e_to(v < kSmall ? 0.5f * v : -fabsf(v));
  return v < kSmall ? e : __builtin_amdgcn_sqrtf(log1p_f32(e) + fmaxf(v, 0.0f));
}
// e^v (softmax, v relative to the row's largest), sigmoid or sqrt(softplus) in 64 bits: called, not inlined, so
// its registers are not the callers'
__device__ __attribute__((noinline)) double score_f64(double v, int scoring) {
  const double e = exp(scoring == AFD_SCORE_SOFTMAX ? v : scoring == AFD_SCORE_SIGMOID ? -v : -fabs(v));
  if (scoring == AFD_SCORE_SOFTMAX) return e;
  return scoring == AFD_SCORE_SIGMOID ? 1.0 / (1.0 + e) : sqrt(log1p(e) + fmax(v, 0.0));
}
// d score / dl over the score: 1 - sigmoid, or sigmoid / (2 softplus), which tends to 1/2 where
// softplus(l) -> e^l leaves the floats
// (taken from the score where it is at hand)
__device__ __forceinline__ float slope_f32(float v, float score, int scoring) {
  if (scoring == AFD_SCORE_SOFTMAX) return 1.0f;
  if (scoring == AFD_SCORE_SIGMOID) return __builtin_amdgcn_rcpf(1.0f + exp_fast(v));
  if (v < kSmall) return 0.5f;
  return 0.5f * __builtin_amdgcn_rcpf((1.0f + exp_fast(-v)) * (score * score));
}

template <typename T, int W, int V>
struct Row {
  float l[V];  // canonical logits of the lane's experts, -inf past the last one
  int e0;      // the lane's first expert

  // A row's logits as they lie in memory, so that a row can be on its way while another is worked on
  struct Raw {
    static constexpr int kWords = V * sizeof(T) / 4;
    uint32_t u[kWords];
  };
  // WIDE: E, the stride and the address are multiples of 4 elements. No branches: lanes past the last
  // expert read it again (set() drops them), and a load that is not branched around is waited for only
  // where its row is used.
  template <bool WIDE>
  static __device__ __forceinline__ Raw fetch(const Args& a, int64_t t, int li) {
    Raw r;
    const T* p = static_cast<const T*>(a.logits) + t * a.ld;
    if constexpr (WIDE) {
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const T* q = p + min(li * V + j, a.experts - 4);
        if constexpr (sizeof(T) == 4) {
          const v4i x = *reinterpret_cast<const v4i*>(q);
#pragma unroll
          for (int i = 0; i < 4; ++i) r.u[j + i] = x[i];
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(q);
          r.u[j / 2] = x.x;
          r.u[j / 2 + 1] = x.y;
        }
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < V; ++j) r.u[j] = __float_as_uint(p[min(li * V + j, a.experts - 1)]);
    } else {
#pragma unroll
      for (int j = 0; j < V; j += 2)
        r.u[j / 2] = p[min(li * V + j, a.experts - 1)] | uint32_t(p[min(li * V + j + 1, a.experts - 1)]) << 16;
    }
    return r;
  }
  __device__ __forceinline__ void set(const Args& a, const Raw& r, int li) {
    e0 = li * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float v;
      if constexpr (sizeof(T) == 4)
        v = __uint_as_float(r.u[j]);
      else
        v = __uint_as_float(j & 1 ? r.u[j / 2] & 0xffff0000u : r.u[j / 2] << 16);
      l[j] = e0 + j < a.experts ? canon(v) : kLowest;
    }
  }
  // The row's scores in fp32: s[j] (0 past the last expert), and their sum. EXACT: to a few ulps, for choosing.
  template <bool EXACT>
  __device__ __forceinline__ float scores(const Args& a, float (&s)[V]) const {
    float sum = 0.0f;
    if (a.scoring == AFD_SCORE_SOFTMAX) {
      float m = l[0];
#pragma unroll
      for (int j = 1; j < V; ++j) m = fmaxf(m, l[j]);
      m = max_f32<W>(m);
      const float at = m == kLowest ? 0.0f : m;  // a row of -inf: all scores 0
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[j] = EXACT ? exp_f32(l[j] - at) : exp_fast(l[j] - at);
        sum += s[j];
      }
      return sum_f32<W>(sum);
    }
    if (a.scoring == AFD_SCORE_SIGMOID) {
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] = score_f32<EXACT>(l[j], AFD_SCORE_SIGMOID);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] = score_f32<EXACT>(l[j], AFD_SCORE_SQRTSOFTPLUS);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) sum += s[j];  // 0 of -inf, past the last expert
    return sum_f32<W>(sum);
  }
};

// The lane of this row that holds the first of the set bits
template <int W>
__device__ __forceinline__ int first_lane(bool bit, int lane) {
  const uint64_t all = __ballot(bit);
  if constexpr (W == 64) return __builtin_ctzll(all);
  const uint32_t half = lane & 32 ? static_cast<uint32_t>(all >> 32) : static_cast<uint32_t>(all);
  if constexpr (W == 32) return __builtin_ctz(half);
  return __builtin_ctz(half >> (lane & 16));  // the other row's bits lie above this one's, of which one is set
}

// A lane's value in all lanes of its row
template <int W>
__device__ __forceinline__ int from_lane(int v, int lane) {
  if constexpr (W == 64) return __builtin_amdgcn_readlane(v, lane);
  return __shfl(v, lane, W);
}

// The row's keys, taken largest first (lowest index of equals). A lane sorts its own keys once and only
// its head takes part in a round. Low bits of a key say which expert it is:
// kIndexed (bf16 logits, 16 spare bits): kMaxExperts - 1 - e, so that no two are equal, the winning key
//   names the winner and equal logits are already in index order;
// kPlaced: V - 1 - the place in the lane, over the value's lowest bits; values that this could bring out of
//   order are looked at again;
// kBare (4 fp32 logits a lane, no bias): the places are sorted along, by adjacent exchanges (equals keep
//   their order).
enum KeyKind { kBare, kPlaced, kIndexed };

// A bf16 logit's key with its low half free: the low half is 0 of a positive number and all ones of a
// negative one or of the largest float (+inf), which rounds to the next key, unused by any other.
__device__ __forceinline__ uint32_t index_key(uint32_t key) { return (key + 0x8000u) & 0xffff0000u; }
__device__ __forceinline__ float index_value(uint32_t key) {
  key &= 0xffff0000u;
  return canon(value_of(key >> 31 ? key : key - 1));
}

template <int W, int V, KeyKind KIND>
struct Keys {
  uint32_t key[V];
  uint32_t order;  // bare keys: byte i is the place of the i-th largest

  __device__ __forceinline__ void start(int e0) {
    if constexpr (KIND == kBare) {
      static_assert(V == 4, "places are bytes of a word");
      uint32_t at[4] = {0, 1, 2, 3};
#pragma unroll
      for (int end = 3; end > 0; --end)
#pragma unroll
        for (int i = 0; i < end; ++i) {
          const bool swap = key[i + 1] > key[i];
          const uint32_t x = at[i], lo = min(key[i], key[i + 1]);
          key[i] = max(key[i], key[i + 1]);
          key[i + 1] = lo;
          at[i] = swap ? at[i + 1] : x;
          at[i + 1] = swap ? x : at[i + 1];
        }
      order = at[0] | at[1] << 8 | at[2] << 16 | at[3] << 24;
      return;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (KIND == kIndexed)
        key[j] = key[j] ? index_key(key[j]) | (kMaxExperts - 1 - e0 - j) : 0u;
      else
        key[j] = key[j] ? (key[j] & ~uint32_t(V - 1)) | (V - 1 - j) : 0u;
    }
    // odd-even merge sort, largest first: 5, 19 or 63 exchanges of a maximum and a minimum
#pragma unroll
    for (int p = 1; p < V; p *= 2)
#pragma unroll
      for (int k = p; k >= 1; k /= 2)
#pragma unroll
        for (int j = k % p; j + k < V; j += 2 * k)
#pragma unroll
          for (int i = 0; i < k; ++i)
            if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
              const uint32_t x = key[i + j], y = key[i + j + k];
              key[i + j] = max(x, y);
              key[i + j + k] = min(x, y);
            }
  }
  __device__ __forceinline__ uint32_t head() const { return key[0]; }
  // Takes the largest key m and returns its expert, the same in every lane of the row.
  __device__ __forceinline__ int next(int lane, int e0, uint32_t& m) {
    m = max_u32<W>(key[0]);
    bool mine;
    int e = 0, win = 0;
    if constexpr (KIND == kIndexed) {
      mine = key[0] == m;
      e = kMaxExperts - 1 - static_cast<int>(m & (kMaxExperts - 1));
    } else {
      win = first_lane<W>(key[0] == m, lane);
      mine = (lane & (W - 1)) == win;
      if constexpr (KIND == kPlaced) {
        e = win * V + V - 1 - static_cast<int>(m & (V - 1));
      } else {
        e = e0 + static_cast<int>(order & 0xff);
        order = mine ? order >> 8 : order;
      }
    }
#pragma unroll
    for (int j = 0; j + 1 < V; ++j) key[j] = mine ? key[j + 1] : key[j];
    key[V - 1] = mine ? 0u : key[V - 1];
    if constexpr (KIND == kBare) {
      return from_lane<W>(e, win);  // the winner's e
    }
    return e;
  }
};

// A placed key's value for comparisons (-inf, whose place bits make it a NaN, is -inf)
__device__ __forceinline__ float placed_value(uint32_t key) {
  const float v = value_of(key);
  return v != v ? kLowest : v;
}

// LDS of a row: the keys of the 64-bit choice
__host__ __device__ constexpr int row_words(int W, int V) { return W * V; }

__device__ __forceinline__ void lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The lane with the row's largest 64-bit key (the first of equals)
template <int W>
__device__ __forceinline__ int best_lane(uint64_t key, int lane) {
  const uint32_t hi = static_cast<uint32_t>(key >> 32), m_hi = max_u32<W>(hi);
  const uint32_t lo = hi == m_hi ? static_cast<uint32_t>(key) : 0u, m_lo = max_u32<W>(lo);
  return first_lane<W>(hi == m_hi && static_cast<uint32_t>(key) == m_lo, lane);
}

// A softmax's largest logit and sum in 64 bits
template <typename T, int W, int V>
__device__ __forceinline__ void softmax_f64(const Args& a, const T* p, int e0, double& at, double& sum) {
  float m = kLowest;
#pragma unroll 1
  for (int j = 0; j < V; ++j) m = fmaxf(m, e0 + j < a.experts ? canon(logit_f32(p + e0 + j)) : kLowest);
  m = max_f32<W>(m);
  at = m == kLowest ? 0.0 : static_cast<double>(m);
  sum = 0.0;
#pragma unroll 1
  for (int j = 0; j < V; ++j)
    if (e0 + j < a.experts) sum += score_f64(canon(logit_f32(p + e0 + j)) - at, AFD_SCORE_SOFTMAX);
  sum = sum_f64<W>(sum);
  if (sum == 0.0) sum = 1.0;
}

// The choice in 64 bits, groups of any size: lane kk < topk gets the kk-th expert. Rare, so
// its values live in LDS and its loops stay loops: it must not cost the usual case its registers.
template <typename T, int W, int V, bool BIAS>
__device__ __forceinline__ int choose_f64(const Args& a, int64_t t, int lane, uint64_t* keys) {
  const int li = lane & (W - 1), e0 = li * V;
  const T* p = static_cast<const T*>(a.logits) + t * a.ld;
  double at = 0.0, sum = 1.0;
  if (BIAS && a.scoring == AFD_SCORE_SOFTMAX) softmax_f64<T, W, V>(a, p, e0, at, sum);
#pragma unroll 1
  for (int j = 0; j < V; ++j) {
    uint64_t key = 0;
    if (e0 + j < a.experts) {
      double c = canon(logit_f32(p + e0 + j));
      if constexpr (BIAS) {
        c = score_f64(c - at, a.scoring);  // at is 0 but for softmax
        if (a.scoring == AFD_SCORE_SOFTMAX) c /= sum;
        c += a.bias[e0 + j];
        if (c != c) c = -__builtin_huge_val();
      }
      key = key64(c);
    }
    keys[e0 + j] = key;
  }
  lds_fence();
  if (a.groups > 1) {
    // lane g < groups (groups <= W) makes group g's value: its largest choice value (no bias) or the
    // sum of its two largest
    const int size = a.experts / a.groups;
    uint64_t gkey = 0;
    if (li < a.groups) {
      uint64_t first = 0, second = 0;
#pragma unroll 1
      for (int i = 0; i < size; ++i) {
        const uint64_t k = keys[li * size + i];
        second = k > first ? first : k > second ? k : second;
        first = k > first ? k : first;
      }
      double value = value_of(first);
      if (BIAS && size > 1) value += value_of(second);
      if (value != value) value = -__builtin_huge_val();
      gkey = key64(value);
    }
    uint64_t kept = 0;
    for (int i = 0; i < a.keep; ++i) {
      const int g = best_lane<W>(gkey, lane);
      if (li == g) gkey = 0;
      kept |= uint64_t(1) << g;
    }
    lds_fence();
#pragma unroll 1
    for (int j = 0; j < V; ++j)
      if (e0 + j < a.experts && !(kept >> ((e0 + j) / size) & 1)) keys[e0 + j] = 0;
    lds_fence();
  }
  int id = 0;
#pragma unroll 1
  for (int kk = 0; kk < a.topk; ++kk) {
    uint64_t best = 0;
    int e = e0;
#pragma unroll 1
    for (int j = 0; j < V; ++j) {
      const uint64_t k = keys[e0 + j];
      e = k > best ? e0 + j : e;
      best = k > best ? k : best;
    }
    const int win = best_lane<W>(best, lane);
    if (li == win) keys[e] = 0;
    const int got = __shfl(e, win, W);
    id = li == kk ? got : id;
    lds_fence();
  }
  return id;
}

// A butterfly step of lane distance D (1, 2, .. 32) inside a row, for values that agree within D lanes
template <int D>
__device__ __forceinline__ float step_f32(float v, int lane) {
  const uint32_t u = __float_as_uint(v);
  if constexpr (D == 1) return __uint_as_float(dpp<kXor1>(u));
  if constexpr (D == 2) return __uint_as_float(dpp<kXor2>(u));
  if constexpr (D == 4) return __uint_as_float(dpp<kHalfMirror>(u));
  if constexpr (D == 8) return __uint_as_float(dpp<kMirror>(u));
  if constexpr (D == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __uint_as_float(lane & 16 ? r[0] : r[1]);
  }
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(lane & 32 ? r[0] : r[1]);
}

// A bit for each lane of a row
template <int W>
using Lanes = std::conditional_t<W == 64, uint64_t, uint32_t>;

// Which groups stay, by choice values in fp32, as the bits of their first lanes (lane gl g of the row stands for
// group g, gl = a.group_lanes). sure: false if the worst kept and the best dropped are within `margin`.
// Groups of 1, 2, 4, .. whole lanes are made from the lanes' own values; others go through LDS, where the
// gl = 1, 2, 4, .. lanes that a group can have read its values in turn (16384 rows, 160 experts in 8
// groups: 11.7 us, as the 64-bit choice below 47.6).
template <int W, int V, bool BIAS>
__device__ __forceinline__ Lanes<W> keep_groups(const Args& a, const float (&c)[V], int lane, float* lds_row,
                                                float margin, bool& sure) {
  const int li = lane & (W - 1), gl = a.group_lanes;
  float first = kLowest, second = kLowest;
  auto add = [&](float f) {
    second = fmaxf(second, fminf(first, f));
    first = fmaxf(first, f);
  };
  auto merge = [&](float f, float s) {
    second = fmaxf(fmaxf(second, s), fminf(first, f));
    first = fmaxf(first, f);
  };
  const int size = a.experts / a.groups;
  if (a.whole_lanes) {
#pragma unroll
    for (int j = 0; j < V; ++j) add(c[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) lds_row[li * V + j] = c[j];
    lds_fence();
    // (lanes past the last group read the last one's values)
    const int log_gl = __builtin_ctz(gl), g = min(li >> log_gl, a.groups - 1);
    for (int i = li & (gl - 1); i < size; i += gl) add(lds_row[g * size + i]);
    lds_fence();
  }
  if (gl > 1) merge(step_f32<1>(first, lane), step_f32<1>(second, lane));
  if (gl > 2) merge(step_f32<2>(first, lane), step_f32<2>(second, lane));
  if (gl > 4) merge(step_f32<4>(first, lane), step_f32<4>(second, lane));
  if (gl > 8) merge(step_f32<8>(first, lane), step_f32<8>(second, lane));
  if constexpr (W > 16)
    if (gl > 16) merge(step_f32<16>(first, lane), step_f32<16>(second, lane));
  if constexpr (W > 32)
    if (gl > 32) merge(step_f32<32>(first, lane), step_f32<32>(second, lane));
  float value = BIAS && size > 1 ? first + second : first;
  if constexpr (BIAS) value = value != value ? kLowest : value;  // +inf and -inf
  uint32_t key = (li & (gl - 1)) == 0 && li < a.groups * gl ? key32(value) : 0u;
  Lanes<W> kept = 0;
  float worst = 0.0f;
  for (int i = 0; i < a.keep; ++i) {
    const uint32_t m = max_u32<W>(key);
    const int win = first_lane<W>(key == m, lane);
    if (li == win) key = 0;
    kept |= Lanes<W>(1) << win;
    worst = value_of(m);
  }
  if constexpr (BIAS) {
    const uint32_t m = max_u32<W>(key);
    sure = sure && (m == 0 || worst - value_of(m) > margin);
  }
  return kept;
}

// keep_groups in 64 bits, for groups of whole lanes whose fp32 values are close. Rare: its loops stay loops.
template <typename T, int W, int V>
__device__ __forceinline__ Lanes<W> keep_groups_f64(const Args& a, int64_t t, int lane) {
  const int li = lane & (W - 1), e0 = li * V, gl = a.group_lanes;
  const T* p = static_cast<const T*>(a.logits) + t * a.ld;
  double at = 0.0, sum = 1.0;
  if (a.scoring == AFD_SCORE_SOFTMAX) softmax_f64<T, W, V>(a, p, e0, at, sum);
  double first = -__builtin_huge_val(), second = first;
#pragma unroll 1
  for (int j = 0; j < V; ++j) {
    if (e0 + j >= a.experts) break;
    double c = score_f64(canon(logit_f32(p + e0 + j)) - at, a.scoring);
    if (a.scoring == AFD_SCORE_SOFTMAX) c /= sum;
    c += a.bias[e0 + j];
    if (c != c) c = -__builtin_huge_val();
    second = fmax(second, fmin(first, c));
    first = fmax(first, c);
  }
#pragma unroll 1
  for (int d = 1; d < gl; d *= 2) {
    const double f = __shfl_xor(first, d, W), s = __shfl_xor(second, d, W);
    second = fmax(fmax(second, s), fmin(first, f));
    first = fmax(first, f);
  }
  double value = first + second;
  if (value != value) value = -__builtin_huge_val();
  uint64_t key = (li & (gl - 1)) == 0 && li < a.groups * gl ? key64(value) : 0u;
  Lanes<W> kept = 0;
  for (int i = 0; i < a.keep; ++i) {
    const int win = best_lane<W>(key, lane);
    if (li == win) key = 0;
    kept |= Lanes<W>(1) << win;
  }
  return kept;
}

// A placed key is off by at most 15 ulps of 2^-23 of its value or, near zero, of 2^-149; two of them by twice that.
__device__ __forceinline__ float place_error(float v) { return __builtin_fmaf(fabsf(v), 0x1p-18f, 0x1p-144f); }

// Close choice values in 64 bits (no bias: the logits themselves). The fp32 choice is right but for experts within
// `margin` of each other, so the chosen ones and every other within it of the last (taken on from `keys`) are
// ranked by their 64-bit values, one a lane. False if they are more than the row's lanes.
template <typename T, int W, int V, bool BIAS>
__device__ __forceinline__ bool settle(const Args& a, int64_t t, int lane, uint64_t* lds_row,
                                       Keys<W, V, kPlaced>& keys, float margin, uint32_t taken, int& id) {
  const int li = lane & (W - 1), e0 = li * V;
  const float worst = placed_value(__shfl(taken, a.topk - 1, W));
  const float bar = worst - (BIAS ? margin : 2.0f * place_error(worst));
  int count = a.topk;
  while (true) {
    const uint32_t top = max_u32<W>(keys.head());
    const bool more = top != 0 && !(placed_value(top) < bar);
    if (__ballot(more && count == W)) return false;
    if (!__ballot(more)) break;
    const Keys<W, V, kPlaced> before = keys;
    uint32_t m;
    const int e = keys.next(lane, e0, m);
    if (!more) keys = before;  // another row of the wavefront goes on
    if (more && li == count) id = e;
    count += more ? 1 : 0;
  }
  const T* p = static_cast<const T*>(a.logits) + t * a.ld;
  double c = canon(logit_f32(p + (li < count ? id : 0)));
  if constexpr (BIAS) {
    double at = 0.0, sum = 1.0;
    if (a.scoring == AFD_SCORE_SOFTMAX) softmax_f64<T, W, V>(a, p, e0, at, sum);
    c = score_f64(c - at, a.scoring);
    if (a.scoring == AFD_SCORE_SOFTMAX) c /= sum;
    c += a.bias[li < count ? id : 0];
    if (c != c) c = -__builtin_huge_val();
  }
  const uint64_t key = key64(c);
  const uint32_t lo = static_cast<uint32_t>(key), hi = static_cast<uint32_t>(key >> 32);
  int rank = 0;
  const int most = W == 64 ? count : static_cast<int>(max_u32<64>(count));
  for (int i = 0; i < most; ++i) {
    const uint64_t other = uint64_t(__shfl(hi, i, W)) << 32 | __shfl(lo, i, W);
    const int e = __shfl(id, i, W);
    rank += i < count && (other > key || (other == key && e < id)) ? 1 : 0;
  }
  int* picks = reinterpret_cast<int*>(lds_row);
  if (li < count && rank < a.topk) picks[rank] = id;
  lds_fence();
  id = li < a.topk ? picks[li] : 0;
  lds_fence();
  return true;
}

// Selection of one row: lane kk < topk gets the kk-th expert and `chosen`, its logit, or with a bias and
// scores of their own its score (-inf in other lanes).
// bias: the lane's experts', bias_most: the largest (BIAS); s, sum: the row's scores (BIAS).
template <typename T, int W, int V, bool BIAS>
__device__ __forceinline__ int choose(const Args& a, const Row<T, W, V>& row, int64_t t, int lane, uint64_t* lds_row,
                                      const float (&bias)[V], float bias_most, const float (&s)[V], float sum,
                                      float& chosen) {
  const int li = lane & (W - 1), e0 = row.e0;
  float c[V], margin = 0.0f;
  bool sure = true;
  if constexpr (BIAS) {
    // An fp32 choice value is off by less than 2^-20 (s + |bias|): the hardware's exponential, reciprocal and root
    // are within one ulp of 2^-23, every other step within 2^-24, at most 9 of these together, and two bits
    // that hold the place take 6. Three such bits take 14 (2^-19 then), four 30, a softmax's sum over 16 values a
    // lane and 6 butterflies 24: 2^-18 there. A score below 2^-126 may count as 0. Two values stand apart if
    // they differ by twice the row's largest such bound.
    const float inv = a.scoring == AFD_SCORE_SOFTMAX ? (sum >= kLeast ? __builtin_amdgcn_rcpf(sum) : 0.0f) : 1.0f;
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float score = s[j] * inv;
      c[j] = e0 + j < a.experts ? score + bias[j] : kLowest;
      most = fmaxf(most, score);
    }
    const float part = a.scoring == AFD_SCORE_SOFTMAX || V > 8 ? 0x1p-17f : V > 4 ? 0x1p-18f : 0x1p-19f;
    margin = __builtin_fmaf(max_f32<W>(most) + bias_most, part, 0x1p-124f);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) c[j] = row.l[j];
  }
  constexpr KeyKind kKind = BIAS ? kPlaced : sizeof(T) == 2 ? kIndexed : V == 4 ? kBare : kPlaced;
  Keys<W, V, kKind> keys;
#pragma unroll
  for (int j = 0; j < V; ++j) keys.key[j] = e0 + j < a.experts ? key32(c[j]) : 0;
  if (a.groups > 1) {
    // a group's value is the sum of two choice values: twice the margin
    Lanes<W> kept = keep_groups<W, V, BIAS>(a, c, lane, reinterpret_cast<float*>(lds_row), 2.0f * margin, sure);
    if constexpr (BIAS) {
      sure = !__ballot(!sure);
      if (!sure && a.whole_lanes) {
        kept = keep_groups_f64<T, W, V>(a, t, lane);
        sure = true;
      }
    }
    if (a.whole_lanes) {
      const bool mine = kept >> (li & ~(a.group_lanes - 1)) & 1;
#pragma unroll
      for (int j = 0; j < V; ++j) keys.key[j] = mine ? keys.key[j] : 0;
    } else {
      // e / size for e < 1024: the quotient of e + 1/2 is at least 1 / (2 size) from a whole number
      const float per = 1.0f / (a.experts / a.groups);
      const int gl = a.group_lanes;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int g = static_cast<int>((e0 + j + 0.5f) * per);
        keys.key[j] = kept >> ((g * gl) & (W - 1)) & 1 ? keys.key[j] : 0;
      }
    }
  }
  keys.start(e0);
  int id = 0;
  uint32_t taken = 0;  // lane kk: the kk-th key
  for (int kk = 0; kk < a.topk; ++kk) {
    uint32_t m;
    const int e = keys.next(lane, e0, m);
    id = li == kk ? e : id;
    taken = li == kk ? m : taken;
  }
  const bool live = li < a.topk;
  bool all = !sure;  // close groups that are not whole lanes: the whole choice in 64 bits
  if constexpr (kKind == kPlaced) {
    if (!all) {
      // lane kk compares the kk-th with the next one, the last with the best that is left
      const uint32_t left = max_u32<W>(keys.head());
      const uint32_t after = __shfl_down(taken, 1, W);
      const uint32_t below = li == a.topk - 1 ? left : after;
      const float x = placed_value(taken), y = placed_value(below);
      const float apart = BIAS ? margin : place_error(fmaxf(fabsf(x), fabsf(y)));
      // (-inf behind a number is far)
      const bool close = live && below != 0 && !(x - y > apart || (y == kLowest && x != kLowest && !BIAS));
      if (__ballot(close)) all = !settle<T, W, V, BIAS>(a, t, lane, lds_row, keys, margin, taken, id);
    }
  }
  if constexpr (kKind == kPlaced) {
    if (all) id = choose_f64<T, W, V, BIAS>(a, t, lane, lds_row);
    // the row's logits (scores) by way of LDS
    float* mine = reinterpret_cast<float*>(lds_row);
    if (BIAS && a.scoring != AFD_SCORE_SOFTMAX) {
#pragma unroll
      for (int j = 0; j < V; ++j) mine[e0 + j] = s[j];
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) mine[e0 + j] = row.l[j];
    }
    lds_fence();
    chosen = live ? mine[id] : kLowest;
    lds_fence();
  } else {
    chosen = live ? sizeof(T) == 2 ? index_value(taken) : value_of(taken) : kLowest;  // the key is the logit
  }
  return id;
}

// The weight of lane kk's expert from what choose() gave, the chosen ones' alone where nothing else is needed.
template <typename T, int W, int V, bool BIAS>
__device__ __forceinline__ float weigh(const Args& a, const Row<T, W, V>& row, float l) {
  float s;
  if (a.scoring == AFD_SCORE_SOFTMAX) {
    // renormalized, the largest chosen logit is the reference: the others' ratios to it survive
    // however small the scores are
    float m = l;
    if (!a.renorm) {
#pragma unroll
      for (int j = 0; j < V; ++j) m = fmaxf(m, row.l[j]);
    }
    m = max_f32<W>(m);
    const float at = m == kLowest ? 0.0f : m;
    s = exp_f32(l - at);  // 0 in lanes without a pick
    float sum = s;
    if (!a.renorm) {
      sum = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) sum += exp_fast(row.l[j] - at);
    }
    sum = sum_f32<W>(sum);
    return sum >= kLeast ? s * __builtin_amdgcn_rcpf(sum) * a.scale : 0.0f;
  }
  s = BIAS ? fmaxf(l, 0.0f) : score_f32<true>(l, a.scoring);
  if (a.renorm) {
    const float sum = sum_f32<W>(s);
    s = sum >= kLeast ? s * __builtin_amdgcn_rcpf(sum) : 0.0f;
  }
  return s * a.scale;
}

// Returns the largest |bias| of all experts (-inf, which bars an expert, aside)
template <int W, int V>
__device__ __forceinline__ float load_bias(const Args& a, int e0, float (&bias)[V]) {
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < V; ++j) {  // no branches: the loads travel together
    const float b = a.bias != nullptr ? a.bias[min(e0 + j, a.experts - 1)] : 0.0f;
    bias[j] = b != b ? kLowest : b;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) most = fmaxf(most, bias[j] == kLowest ? 0.0f : fabsf(bias[j]));
  return max_f32<W>(most);
}

// ---------------------------------------------------------------- selection
template <typename T, int W, int V, bool BIAS, bool WIDE>
__device__ __forceinline__ void topk_rows(const Args& a, uint64_t* lds) {
  constexpr int kRows = kThreads / W;  // rows in flight of a workgroup
  const int t = threadIdx.x, lane = t & 63, li = lane & (W - 1), sub = t / W;
  float bias[V];
  const float bias_most = load_bias<W, V>(a, li * V, bias);
  using R = Row<T, W, V>;
  const int64_t step = int64_t(gridDim.x) * kRows;
  // the lanes of a wavefront stay together: rows past the end are the last one again
  auto clamp_row = [&](int64_t r) { return r < a.n ? r : int64_t(a.n) - 1; };
  int64_t r0 = int64_t(blockIdx.x) * kRows;
  typename R::Raw next = R::template fetch<WIDE>(a, clamp_row(r0 + sub), li);
  for (; r0 < a.n; r0 += step) {
    const int64_t r = r0 + sub, rr = clamp_row(r);
    const typename R::Raw raw = next;
    next = R::template fetch<WIDE>(a, clamp_row(r + step), li);
    const bool valid = a.valid == nullptr || a.valid[rr] != 0;
    R row;
    row.set(a, raw, li);
    float s[V] = {}, sum = 0.0f, l;
    if constexpr (BIAS) sum = row.template scores<true>(a, s);
    int id = choose<T, W, V, BIAS>(a, row, rr, lane, lds + sub * row_words(W, V), bias, bias_most, s, sum, l);
    float w = weigh<T, W, V, BIAS>(a, row, l);
    if (!valid) id = -1, w = 0.0f;
    if (r < a.n && li < a.topk) {
      a.ids[r * a.topk + li] = id;
      a.w[r * a.topk + li] = w;
    }
  }
}

template <typename T, int W, int V, bool BIAS>
__global__ __launch_bounds__(kThreads) void topk_kernel(Args a) {
  __shared__ uint64_t lds[kThreads / W * row_words(W, V)];
  if (a.wide)
    topk_rows<T, W, V, BIAS, true>(a, lds);
  else
    topk_rows<T, W, V, BIAS, false>(a, lds);
}

// ---------------------------------------------------------------- pieces of a block of rows
// The piece of rows that starts at r: up to `end` within one sequence (`seq`), or between sequences (-1).
// Whatever cu holds, end > r and seq < seqs.
struct Piece {
  int32_t end, seq;
};
__device__ __forceinline__ Piece next_piece(const Args& a, int32_t r, int32_t r1) {
  if (a.cu == nullptr) return {r1, 0};
  int lo = 0, hi = a.seqs;  // first sequence that ends behind r
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.cu[mid + 1] > r)
      hi = mid;
    else
      lo = mid + 1;
  }
  if (lo == a.seqs) return {r1, -1};
  const int32_t from = a.cu[lo];
  if (from > r) return {min(from, r1), -1};
  return {min(a.cu[lo + 1], r1), lo};
}

// ---------------------------------------------------------------- a sequence's slots together
// A workgroup takes CH experts of a sequence, its threads 1024 / CH slots side by side, so that a long
// sequence's slots are in flight together; their sums are added in one order. 16 experts (one 64-byte line of a
// slot) where a sequence has many slots, 64 where it has few.
constexpr int kFinishWaves = 16;
constexpr int kFinishThreads = 64 * kFinishWaves;
constexpr int kNarrow = 16, kBroad = 64;

__host__ __device__ inline int chunks_of(int experts, int ch) { return (experts + ch - 1) / ch; }

// counts of experts [CH c, + CH) of sequence s, their part of the unscaled loss, and (c = 0) the rows
template <int CH>
__device__ __forceinline__ void finish_chunk(const Args& a, int s, int c) {
  __shared__ double p_red[kFinishWaves][CH];
  __shared__ int32_t c_red[kFinishWaves][CH];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  int32_t lo = 0, hi = a.n;
  if (a.cu != nullptr) {
    lo = min(max(a.cu[s], 0), a.n);
    hi = min(max(a.cu[s + 1], 0), a.n);
  }
  const int b0 = lo / a.block_rows, slots = hi > lo ? (hi - 1) / a.block_rows + 1 - b0 : 0;
  const int64_t words = slot_words(a.experts);
  const float* first = a.slots + (int64_t(b0) + s) * words;
  const int e = c * CH + (lane & (CH - 1));
  double p = 0.0;
  int cnt = 0;
  if (e < a.experts) {
#pragma unroll 8
    for (int b = t / CH; b < slots; b += kFinishThreads / CH) {
      const float* slot = first + b * words;
      p += slot[e];
      cnt += reinterpret_cast<const int32_t*>(slot)[a.experts + e];
    }
  }
  // the wavefront's slots, then the wavefronts
#pragma unroll
  for (int d = CH; d < 64; d *= 2) {
    p += __shfl_xor(p, d);
    cnt += __shfl_xor(cnt, d);
  }
  if (lane < CH) {
    p_red[w][lane] = p;
    c_red[w][lane] = cnt;
  }
  if (w == 1 && c == 0 && a.loss != nullptr) {
    double rows = 0.0;
    for (int b = lane; b < slots; b += 64) rows += reinterpret_cast<const int32_t*>(first + b * words)[2 * a.experts];
    rows = sum_f64<64>(rows);
    if (lane == 0) a.rows[s] = static_cast<int32_t>(rows);
  }
  __syncthreads();
  if (w == 0) {
    p = 0.0;
    cnt = 0;
    if (lane < CH) {
#pragma unroll
      for (int i = 0; i < kFinishWaves; ++i) {
        p += p_red[i][lane];
        cnt += c_red[i][lane];
      }
      if (e < a.experts) a.counts[int64_t(s) * a.experts + e] = cnt;
    }
    if (a.loss != nullptr) {
      const double loss = sum_f64<64>(p * cnt);
      if (lane == 0) a.part[int64_t(s) * chunks_of(a.experts, CH) + c] = loss;
    }
  }
  __syncthreads();
}

// The sum over the workgroup, in one order, the same in every thread
__device__ __forceinline__ double block_sum(double v, double* red) {
  const int t = threadIdx.x;
  v = sum_f64<64>(v);
  if ((t & 63) == 0) red[t >> 6] = v;
  __syncthreads();
  v = 0.0;
  for (int i = 0; i < kFinishWaves; ++i) v += red[i];
  __syncthreads();
  return v;
}

// One workgroup, after every sequence: the loss and the sequences' coefficients.
__device__ __forceinline__ void finish_loss(const Args& a, int chunks) {
  __shared__ double red[kFinishWaves];
  const int t = threadIdx.x;
  double sum = 0.0, used = 0.0;
  // 16 threads a sequence, its chunks dealt to them
  for (int64_t s = t >> 4; s < a.seqs; s += kFinishThreads / 16) {
    const double rows = a.rows[s];
    double loss = 0.0;
    for (int c = t & 15; c < chunks; c += 16) loss += a.part[s * chunks + c];
    if (rows > 0.0) {
      sum += loss * a.experts / (a.topk * rows * rows);
      used += (t & 15) == 0 ? 1.0 : 0.0;
    }
  }
  sum = block_sum(sum, red);
  used = block_sum(used, red);
  if (t == 0) *a.loss = used > 0.0 ? static_cast<float>(a.alpha * sum / used) : 0.0f;
  for (int s = t; s < a.seqs; s += kFinishThreads) {
    const double rows = a.rows[s];
    a.coef[s] = rows > 0 ? static_cast<float>(double(a.alpha) * a.experts / (used * a.topk * rows * rows)) : 0.0f;
  }
}

template <int CH>
__global__ __launch_bounds__(kFinishThreads) void finish_kernel(Args a) {
  __shared__ uint32_t done;
  const int chunks = chunks_of(a.experts, CH);
  for (int64_t i = blockIdx.x; i < int64_t(a.seqs) * chunks; i += gridDim.x)
    finish_chunk<CH>(a, static_cast<int>(i / chunks), static_cast<int>(i % chunks));
  if (a.loss == nullptr) return;
  // the last workgroup adds the sequences up: what it reads (part and rows) was written by the first two
  // wavefronts, which order their writes device-wide before the first one's count
  if (threadIdx.x < 128) __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) done = atomicAdd(a.ticket, 1u);
  __syncthreads();
  if (done != gridDim.x - 1) return;
  __threadfence();
  finish_loss(a, chunks);
}

// ---------------------------------------------------------------- selection, counts and balance sums
// The rows of one piece: p, the lane's sums of s' over its rows; mine, their number; cnt, the counts (LDS).
template <typename T, int W, int V, bool SELECT, bool BIAS, bool WIDE>
__device__ __forceinline__ void balance_rows(const Args& a, int32_t at, const Piece& piece, const float (&bias)[V],
                                             float bias_most, float (&p)[V], int& mine, int32_t* cnt, uint64_t* lds) {
  constexpr int kRows = balance_threads(W, V) / W;
  const int t = threadIdx.x, lane = t & 63, li = lane & (W - 1), sub = t / W;
  const bool counted = piece.seq >= 0;
  using R = Row<T, W, V>;
  auto clamp_row = [&](int32_t r) { return min(r, piece.end - 1); };
  typename R::Raw next = R::template fetch<WIDE>(a, clamp_row(at + sub), li);
  for (int32_t base = at; base < piece.end; base += kRows) {
    const int32_t r = base + sub;
    const bool in = r < piece.end;
    const int32_t rr = in ? r : piece.end - 1;
    const bool live = in && (a.valid == nullptr || a.valid[rr]);
    R row;
    float s[V];
    const typename R::Raw raw = next;
    next = R::template fetch<WIDE>(a, clamp_row(r + kRows), li);
    row.set(a, raw, li);
    const float sum = row.template scores<BIAS>(a, s);
    if constexpr (SELECT) {
      float l;
      const int id = choose<T, W, V, BIAS>(a, row, rr, lane, lds + sub * row_words(W, V), bias, bias_most, s, sum, l);
      const float w = weigh<T, W, V, BIAS>(a, row, l);
      if (in && li < a.topk) {
        a.ids[int64_t(r) * a.topk + li] = live ? id : -1;
        a.w[int64_t(r) * a.topk + li] = live ? w : 0.0f;
        if (live && counted) atomicAdd(&cnt[id], 1);
      }
    } else if (live && counted) {
      for (int kk = li; kk < a.topk; kk += W) {
        const int id = a.ids[int64_t(r) * a.topk + kk];
        if (id >= 0 && id < a.experts) atomicAdd(&cnt[id], 1);
      }
    }
    const float inv = live && sum >= kLeast ? __builtin_amdgcn_rcpf(sum) : 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) p[j] += s[j] * inv;
    mine += live ? 1 : 0;
  }
}

// SELECT: choose the experts (else read a.ids). SCORES: sums of s' (else counts alone).
template <typename T, int W, int V, bool SELECT, bool BIAS, bool SCORES>
__global__ __launch_bounds__(balance_threads(W, V)) void balance_kernel(Args a) {
  constexpr int kRows = balance_threads(W, V) / W;
  __shared__ uint64_t lds[SELECT ? kRows * row_words(W, V) : 1];
  __shared__ float sums[SCORES ? kRows * W * V : 1];
  __shared__ int32_t cnt[kMaxExperts];
  __shared__ int32_t live_rows;
  const int t = threadIdx.x, lane = t & 63, li = lane & (W - 1), sub = t / W;
  if (blockIdx.x == 0 && t == 0 && a.ticket != nullptr) *a.ticket = 0;  // for the second launch
  float bias[V];
  float bias_most = 0.0f;
  if constexpr (SELECT) bias_most = load_bias<W, V>(a, li * V, bias);
  const int32_t r0 = blockIdx.x * a.block_rows;
  const int32_t r1 = a.n - r0 < a.block_rows ? a.n : r0 + a.block_rows;
  for (int32_t at = r0; at < r1;) {
    const Piece piece = next_piece(a, at, r1);
    const bool counted = piece.seq >= 0;
    for (int e = t; e < a.experts; e += balance_threads(W, V)) cnt[e] = 0;
    if (t == 0) live_rows = 0;
    __syncthreads();
    float p[V] = {};
    int mine = 0;
    if constexpr (!SCORES) {
      // the rows' ids are one run of memory
      const int64_t last = counted ? int64_t(piece.end) * a.topk : 0;
      for (int64_t i = int64_t(at) * a.topk + t; i < last; i += balance_threads(W, V)) {
        const int id = a.ids[i];
        const bool live = a.valid == nullptr || a.valid[i / a.topk] != 0;
        if (live && static_cast<uint32_t>(id) < static_cast<uint32_t>(a.experts)) atomicAdd(&cnt[id], 1);
      }
      __syncthreads();
    } else if (a.wide) {
      balance_rows<T, W, V, SELECT, BIAS, true>(a, at, piece, bias, bias_most, p, mine, cnt, lds);
    } else {
      balance_rows<T, W, V, SELECT, BIAS, false>(a, at, piece, bias, bias_most, p, mine, cnt, lds);
    }
    if (counted) {
      if (li == 0) atomicAdd(&live_rows, mine);
      if constexpr (SCORES) {
#pragma unroll
        for (int j = 0; j < V; ++j) sums[sub * (W * V) + li * V + j] = p[j];
      }
      __syncthreads();
      float* slot = a.slots + (int64_t(blockIdx.x) + piece.seq) * slot_words(a.experts);
      int32_t* slot_i = reinterpret_cast<int32_t*>(slot);
      for (int e = t; e < a.experts; e += balance_threads(W, V)) {
        if constexpr (SCORES) {
          float s = 0.0f;
          for (int i = 0; i < kRows; ++i) s += sums[i * (W * V) + e];
          slot[e] = s;
        } else {
          slot[e] = 0.0f;
        }
        slot_i[a.experts + e] = cnt[e];
      }
      if (t == 0) slot_i[2 * a.experts] = live_rows;
    }
    __syncthreads();
    at = piece.end;
  }
}

// ---------------------------------------------------------------- counts alone, few ids
// One launch: a workgroup counts a sequence's ids in LDS, a histogram for every two of its 16 wavefronts (popular
// experts meet in fewer atomics).
constexpr int kCountThreads = 1024, kHists = 8;
constexpr int64_t kDirectIds = 16384;

__global__ __launch_bounds__(kCountThreads) void count_kernel(Args a) {
  __shared__ int32_t hist[kHists][kMaxExperts];
  const int t = threadIdx.x;
  for (int i = t; i < kHists * kMaxExperts; i += kCountThreads) (&hist[0][0])[i] = 0;
  int32_t lo = 0, hi = a.n;
  if (a.cu != nullptr) {
    lo = min(max(a.cu[blockIdx.x], 0), a.n);
    hi = min(max(a.cu[blockIdx.x + 1], 0), a.n);
  }
  __syncthreads();
  int32_t* mine = hist[t >> 7];
  // the rows' ids are one run of memory
  const int64_t first = int64_t(lo) * a.topk, last = int64_t(hi) * a.topk;
#pragma unroll 4
  for (int64_t i = first + t; i < last; i += kCountThreads) {
    const int id = a.ids[i];
    const bool live = a.valid == nullptr || a.valid[i / a.topk] != 0;
    if (live && static_cast<uint32_t>(id) < static_cast<uint32_t>(a.experts)) atomicAdd(&mine[id], 1);
  }
  __syncthreads();
  for (int e = t; e < a.experts; e += kCountThreads) {
    int sum = 0;
#pragma unroll
    for (int h = 0; h < kHists; ++h) sum += hist[h][e];
    a.counts[int64_t(blockIdx.x) * a.experts + e] = sum;
  }
}

// ---------------------------------------------------------------- gradient by the logits
template <typename T>
__device__ __forceinline__ void store_logit(T* p, float v);
template <>
__device__ __forceinline__ void store_logit<float>(float* p, float v) { *p = v; }
template <>
__device__ __forceinline__ void store_logit<uint16_t>(uint16_t* p, float v) { *p = f32_to_bf16(v); }

template <typename T, int W, int V, bool WIDE>
__device__ __forceinline__ void grad_rows(const Args& a, float* spread) {
  constexpr int kRows = kThreads / W;
  const int t = threadIdx.x, lane = t & 63, li = lane & (W - 1), sub = t / W;
  const float gloss = a.coef != nullptr ? *a.gloss : 0.0f;
  const int32_t r0 = blockIdx.x * a.block_rows;
  const int32_t r1 = a.n - r0 < a.block_rows ? a.n : r0 + a.block_rows;
  for (int32_t at = r0; at < r1;) {
    Piece piece = {r1, -1};
    if (a.coef != nullptr) piece = next_piece(a, at, r1);
    const bool balanced = piece.seq >= 0;
    float f = 0.0f;
    int32_t cnt[V] = {};
    if (balanced) {
      f = gloss * a.coef[piece.seq];
#pragma unroll
      for (int j = 0; j < V; ++j)
        cnt[j] = a.counts[int64_t(piece.seq) * a.experts + min(li * V + j, a.experts - 1)];
    }
    using R = Row<T, W, V>;
    auto clamp_row = [&](int32_t r) { return min(r, piece.end - 1); };
    // what a row needs is fetched a row ahead
    struct Ahead {
      typename R::Raw raw;
      int id;
      float gw;
      bool live;
    };
    const int pick = min(li, a.topk - 1);
    auto fetch = [&](int32_t r) {
      Ahead x;
      x.raw = R::template fetch<WIDE>(a, r, li);
      x.id = a.gw != nullptr ? a.ids[int64_t(r) * a.topk + pick] : -1;
      x.gw = a.gw != nullptr ? a.gw[int64_t(r) * a.topk + pick] : 0.0f;
      x.live = a.valid == nullptr || a.valid[r] != 0;
      return x;
    };
    Ahead next = fetch(clamp_row(at + sub));
    for (int32_t base = at; base < piece.end; base += kRows) {
      const int32_t r = base + sub;
      const bool in = r < piece.end;
      const Ahead now = next;
      next = fetch(clamp_row(r + kRows));
      const bool live = now.live;
      R row;
      row.set(a, now.raw, li);
      float s[V], d[V];
      const float total = row.template scores<false>(a, s);
      const float inv = total >= kLeast ? __builtin_amdgcn_rcpf(total) : 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = 0.0f;
      // Both sums are of the form p_e (v_e - sum_j p_j v_j) with shares p that add up to one. v counts from the largest
      // share's value: a share close to one then leaves no difference of two close numbers, and equal v leave 0.
      const bool all_shares = a.gw != nullptr && !a.renorm && a.scoring == AFD_SCORE_SOFTMAX;
      int top = 0;
      int32_t top_cnt = 0;
      if (balanced || all_shares) {
        float most = row.l[0];
        top = row.e0;
        top_cnt = cnt[0];
#pragma unroll
        for (int j = 1; j < V; ++j) {
          const bool up = row.l[j] > most;
          most = fmaxf(most, row.l[j]);
          top = up ? row.e0 + j : top;
          top_cnt = up ? cnt[j] : top_cnt;
        }
        const int win = first_lane<W>(most == max_f32<W>(most), lane);
        top = from_lane<W>(top, win);
        top_cnt = from_lane<W>(top_cnt, win);
      }
      if (balanced) {
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) dot += static_cast<float>(cnt[j] - top_cnt) * (s[j] * inv);
        dot = sum_f32<W>(dot);
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = s[j] * inv * (f * (static_cast<float>(cnt[j] - top_cnt) - dot));
      }
      float* mine = spread + sub * (W * V);
      if (all_shares) {
        // every expert's share has a value: its weight's gradient, 0 where it was not chosen (an id that comes twice is
        // added up)
        const int id = li < a.topk && static_cast<uint32_t>(now.id) < static_cast<uint32_t>(a.experts) ? now.id : -1;
#pragma unroll
        for (int j = 0; j < V; ++j) mine[row.e0 + j] = 0.0f;
        lds_fence();
        if (id >= 0) atomicAdd(mine + id, now.gw);
        lds_fence();
        const float top_g = mine[top];
        float g[V], mean = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          g[j] = mine[row.e0 + j] - top_g;
          mean += g[j] * (s[j] * inv);
        }
        lds_fence();
        mean = sum_f32<W>(mean);
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] += s[j] * inv * (a.scale * (g[j] - mean));
      } else if (a.gw != nullptr) {
        // lane kk < topk: the kk-th chosen expert's share of the chosen scores (renormalized) or its score, and its gradient
        const int id = li < a.topk && static_cast<uint32_t>(now.id) < static_cast<uint32_t>(a.experts) ? now.id : -1;
        float g = id >= 0 ? now.gw : 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) mine[row.e0 + j] = row.l[j];
        lds_fence();
        const float l = id >= 0 ? mine[id] : kLowest;
        lds_fence();
        float share;
        if (a.scoring == AFD_SCORE_SOFTMAX) {
          const float m = max_f32<W>(l);
          share = id >= 0 ? exp_f32(l - (m == kLowest ? 0.0f : m)) : 0.0f;
        } else {
          share = id >= 0 ? score_f32<true>(l, a.scoring) : 0.0f;
        }
        float mean = 0.0f;
        if (a.renorm) {
          const float chosen = sum_f32<W>(share);
          share = chosen >= kLeast ? share * __builtin_amdgcn_rcpf(chosen) : 0.0f;
          g -= __shfl(g, first_lane<W>(share == max_f32<W>(share), lane), W);
        }
        g *= a.scale;
        if (a.renorm) mean = sum_f32<W>(g * share);
        const float u = share * (g - mean);
        // to the lanes that hold the experts, through LDS (an id that comes twice is added up)
#pragma unroll
        for (int j = 0; j < V; ++j) mine[row.e0 + j] = 0.0f;
        lds_fence();
        if (id >= 0) atomicAdd(mine + id, u);
        lds_fence();
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] += mine[row.e0 + j];
        lds_fence();
      }
      if (in) {
        T* out = static_cast<T*>(a.dlogits) + int64_t(r) * a.experts + row.e0;
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = live ? d[j] * slope_f32(row.l[j], s[j], a.scoring) : 0.0f;
        if constexpr (WIDE) {
#pragma unroll
          for (int j = 0; j < V; j += 4) {
            if (row.e0 + j >= a.experts) continue;
            if constexpr (sizeof(T) == 4)
              *reinterpret_cast<v4f*>(out + j) = v4f{d[j], d[j + 1], d[j + 2], d[j + 3]};
            else
              *reinterpret_cast<uint2*>(out + j) = uint2{pk_bf16(d[j], d[j + 1]), pk_bf16(d[j + 2], d[j + 3])};
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (row.e0 + j < a.experts) store_logit<T>(out + j, d[j]);
        }
      }
    }
    at = piece.end;
  }
}

template <typename T, int W, int V>
__global__ __launch_bounds__(kThreads) void grad_kernel(Args a) {
  __shared__ __attribute__((aligned(16))) float spread[kThreads * V];
  if (a.wide)
    grad_rows<T, W, V, true>(a, spread);
  else
    grad_rows<T, W, V, false>(a, spread);
}

// ---------------------------------------------------------------- host
// f(W, V) for a row of `experts` whose first `lanes` lanes hold picks or groups
template <typename F>
int with_shape(int experts, int lanes, F&& f) {
  using std::integral_constant;
  if (experts <= 64 && lanes <= 16) return f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
  if (experts <= 128 && lanes <= 32) return f(integral_constant<int, 32>{}, integral_constant<int, 4>{});
  if (experts <= 256) return f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  if (experts <= 512) return f(integral_constant<int, 64>{}, integral_constant<int, 8>{});
  return f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}
// Choosing among many rows: fewer lanes a row, so that what a row costs beside its experts (rounds, sums, weights)
// is shared by the rows of a wavefront. By the logits alone 16 lanes (256 experts: 4096 rows 5.4 us
// against 5.0 in the shapes above, 8192 6.4 against 7.5, 65536 26.7 against 43.7), with a bias, whose scores
// cost more than the rounds and whose close rows take longer the more experts a lane has, 32 (8192 rows 11.9
// against 10.4, 16384 14.5 against 16.4, 65536 41.2 against 50.8; 16 lanes: 16384 rows 19.3). Up to 512 experts 32
// lanes by the logits (8192 rows 9.5 against 11.4, 65536 46.6 against 55.9); with a bias as good as 64 up to 16384 rows.
constexpr int kManyRows = 6144, kManyBiasedRows = 12288;
template <typename F>
int with_choice_shape(int experts, int lanes, bool bias, int n, F&& f) {
  using std::integral_constant;
  if (!bias && n >= kManyRows && experts > 64) {
    if (experts <= 128 && lanes <= 16) return f(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    if (experts <= 256 && lanes <= 16) return f(integral_constant<int, 16>{}, integral_constant<int, 16>{});
    if (experts > 256 && experts <= 512 && lanes <= 32) return f(integral_constant<int, 32>{}, integral_constant<int, 16>{});
  }
  if (bias && n >= kManyBiasedRows && lanes <= 32 && experts > 128 && experts <= 256)
    return f(integral_constant<int, 32>{}, integral_constant<int, 8>{});
  return with_shape(experts, lanes, f);
}
template <typename F>
int with_logits(int fmt, F&& f) {
  return fmt == AFD_LOGITS_F32 ? f(float{}) : f(uint16_t{});
}

static int check_cfg(const afd_router_cfg* c) {
  if (!c) return AFD_ERR_ARG;
  if (c->num_experts < 1 || c->num_experts > kMaxExperts) return AFD_ERR_SHAPE;
  if (c->topk < 1 || c->topk > kMaxTopk || c->topk > c->num_experts) return AFD_ERR_SHAPE;
  if (c->scoring < AFD_SCORE_SOFTMAX || c->scoring > AFD_SCORE_SQRTSOFTPLUS) return AFD_ERR_UNSUPPORTED;
  if (c->logits_fmt != AFD_LOGITS_F32 && c->logits_fmt != AFD_LOGITS_BF16) return AFD_ERR_UNSUPPORTED;
  if (c->num_groups < 0 || c->num_groups > kMaxGroups) return AFD_ERR_SHAPE;
  if (c->num_groups > 1) {
    if (c->num_experts % c->num_groups) return AFD_ERR_SHAPE;
    if (c->topk_groups < 1 || c->topk_groups > c->num_groups) return AFD_ERR_SHAPE;
    if (c->topk > c->topk_groups * (c->num_experts / c->num_groups)) return AFD_ERR_SHAPE;
  }
  return AFD_OK;
}
static int check_rows(int32_t n, int32_t topk) {
  if (n < 0 || n > kMaxRows || int64_t(n) * topk > 0x7fffffffll) return AFD_ERR_ARG;
  return AFD_OK;
}
static int check_logits(const afd_router_cfg& c, const void* logits, int64_t ld, int32_t n) {
  if (n > 0 && !logits) return AFD_ERR_ARG;
  if (ld < c.num_experts) return AFD_ERR_SHAPE;
  return AFD_OK;
}
static int check_seqs(const int32_t* cu, int32_t seqs) {
  if (seqs < 1 || seqs > kMaxSeqs || (!cu && seqs != 1)) return AFD_ERR_ARG;
  return AFD_OK;
}

static Args base_args(const afd_router_cfg& c, const void* logits, int64_t ld, int32_t n) {
  Args a = {};
  a.logits = logits;
  a.ld = ld;
  a.n = n;
  a.experts = c.num_experts;
  a.topk = c.topk;
  a.scoring = c.scoring;
  a.groups = c.num_groups > 1 ? c.num_groups : 1;
  a.keep = c.topk_groups;
  a.renorm = c.renormalize != 0;
  a.scale = c.scale;
  return a;
}
// what depends on the lanes' share V of a row
static void set_shape(Args& a, int W, int V, size_t logit_bytes) {
  a.wide = a.experts % 4 == 0 && a.ld % 4 == 0 && reinterpret_cast<uintptr_t>(a.logits) % (4 * logit_bytes) == 0 &&
           reinterpret_cast<uintptr_t>(a.dlogits) % (4 * logit_bytes) == 0;
  const int size = a.experts / a.groups, lanes = size / V;
  a.whole_lanes = size % V == 0 && (lanes & (lanes - 1)) == 0;
  a.group_lanes = lanes;
  if (!a.whole_lanes)
    for (a.group_lanes = 1; 2 * a.group_lanes * a.groups <= W;) a.group_lanes *= 2;
}
static int lanes_needed(const Args& a, bool select) {
  return select && a.groups > a.topk ? a.groups : a.topk;
}

// rows of a workgroup: `groups` workgroups of `threads`, whole passes of their wavefronts, at most kMaxBlockRows
static int block_rows_for(int32_t n, int lanes_per_row, int threads, int groups) {
  const int pass = threads / lanes_per_row;
  int64_t rows = (int64_t(n) + groups - 1) / groups;
  rows = (rows + pass - 1) / pass * pass;
  return static_cast<int>(rows < pass ? pass : rows > kMaxBlockRows ? kMaxBlockRows : rows);
}
static int blocks_for(int32_t n, int block_rows) { return static_cast<int>((int64_t(n) + block_rows - 1) / block_rows); }

// The workspace: slots, part f64, rows i32, ticket. Slots are counted for the smallest block of rows.
struct WsPlan {
  uint64_t slots, part, rows, ticket, total;
};
static WsPlan plan(int32_t n, int32_t experts, int32_t seqs) {
  WsPlan p = {};
  const int rows = block_rows_for(n, 64, balance_threads(64, 16), 256);
  const uint64_t count = uint64_t(blocks_for(n, rows)) + seqs;
  auto round = [](uint64_t v) { return (v + 255) / 256 * 256; };
  p.slots = 0;
  p.part = round(count * slot_words(experts) * 4);
  p.rows = p.part + round(uint64_t(seqs) * chunks_of(experts, kNarrow) * 8);
  p.ticket = p.rows + round(uint64_t(seqs) * 4);
  p.total = p.ticket + 256;
  return p;
}
static void place(Args& a, void* ws, const WsPlan& p) {
  uint8_t* b = static_cast<uint8_t*>(ws);
  a.slots = reinterpret_cast<float*>(b + p.slots);
  a.part = reinterpret_cast<double*>(b + p.part);
  a.rows = reinterpret_cast<int32_t*>(b + p.rows);
  a.ticket = reinterpret_cast<uint32_t*>(b + p.ticket);
}

__global__ __launch_bounds__(kThreads) void no_rows_kernel(Args a) {
  for (int64_t i = blockIdx.x * int64_t(kThreads) + threadIdx.x; i < int64_t(a.seqs) * a.experts;
       i += int64_t(gridDim.x) * kThreads)
    a.counts[i] = 0;
  if (a.loss == nullptr) return;
  for (int64_t s = blockIdx.x * int64_t(kThreads) + threadIdx.x; s < a.seqs; s += int64_t(gridDim.x) * kThreads)
    a.coef[s] = 0.0f;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.loss = 0.0f;
}

// As many workgroups as the CUs hold at once share the rows: those that came after would run behind them (with
// 145 registers 3 a CU: 65536 x 256 with a bias 50.8 us in 4 a CU, 41.2 in 3).
template <void (*KERNEL)(Args)>
static int launch_topk(const Args& a, int rows, hipStream_t s) {
  static const int per_cu = [] {
    int v = 0;
    return hipOccupancyMaxActiveBlocksPerMultiprocessor(&v, KERNEL, kThreads, 0) == hipSuccess && v > 0 ? v : 1;
  }();
  const int64_t need = (int64_t(a.n) + rows - 1) / rows, most = int64_t(per_cu) * device_cu_count();
  hipLaunchKernelGGL(KERNEL, dim3(static_cast<unsigned>(need < most ? need : most)), dim3(kThreads), 0, s, a);
  AFD_CHECK_LAUNCH();
  return AFD_OK;
}

// select: a.ids / a.w are written; scores: with the balance sums
static int launch_balance(Args a, int fmt, bool select, bool scores, hipStream_t s) {
  if (a.n == 0) {
    hipLaunchKernelGGL(no_rows_kernel, dim3(64), dim3(kThreads), 0, s, a);
    AFD_CHECK_LAUNCH();
    return AFD_OK;
  }
  const int st = with_logits(fmt, [&](auto tag) {
    using T = decltype(tag);
    return with_shape(a.experts, lanes_needed(a, select), [&](auto wc, auto vc) {
      constexpr int W = decltype(wc)::value, V = decltype(vc)::value;
      // counts alone are soon summed: fewer slots for the second launch to read
      a.block_rows = block_rows_for(a.n, W, balance_threads(W, V), scores ? 256 : 64);
      a.blocks = blocks_for(a.n, a.block_rows);
      set_shape(a, W, V, sizeof(T));
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(a.blocks), dim3(scores ? balance_threads(W, V) : balance_threads(64, 4)), 0, s, a);
        AFD_CHECK_LAUNCH();
        return int(AFD_OK);
      };
      if (!scores) return go(balance_kernel<float, 64, 4, false, false, false>);
      if (!select) return go(balance_kernel<T, W, V, false, false, true>);
      return a.bias ? go(balance_kernel<T, W, V, true, true, true>) : go(balance_kernel<T, W, V, true, false, true>);
    });
  });
  if (st != AFD_OK) return st;
  // (8192 x 64 in 32 sequences, 8 slots each: 9.9 us with workgroups of 64 experts, 12.0 with 16)
  const bool broad = a.blocks / a.seqs <= kFinishThreads / kBroad;
  const int64_t items = int64_t(a.seqs) * chunks_of(a.experts, broad ? kBroad : kNarrow);
  const dim3 grid(static_cast<unsigned>(items < 2048 ? items : 2048));
  if (broad)
    hipLaunchKernelGGL(finish_kernel<kBroad>, grid, dim3(kFinishThreads), 0, s, a);
  else
    hipLaunchKernelGGL(finish_kernel<kNarrow>, grid, dim3(kFinishThreads), 0, s, a);
  AFD_CHECK_LAUNCH();
  return AFD_OK;
}

}  // namespace router
}  // namespace afd

using namespace afd;

extern "C" int afd_topk(const afd_router_cfg* cfg, const void* logits, int64_t ld, const float* bias,
                        const uint8_t* valid, int32_t n, int32_t* ids, float* w, afd_stream_t stream) {
  int st = router::check_cfg(cfg);
  if (st == AFD_OK) st = router::check_rows(n, cfg->topk);
  if (st == AFD_OK) st = router::check_logits(*cfg, logits, ld, n);
  if (st != AFD_OK) return st;
  if (n == 0) return AFD_OK;
  if (!ids || !w) return AFD_ERR_ARG;
  router::Args a = router::base_args(*cfg, logits, ld, n);
  a.bias = bias;
  a.valid = valid;
  a.ids = ids;
  a.w = w;
  return router::with_logits(cfg->logits_fmt, [&](auto tag) {
    using T = decltype(tag);
    return router::with_choice_shape(a.experts, router::lanes_needed(a, true), bias != nullptr, n, [&](auto wc, auto vc) {
      constexpr int W = decltype(wc)::value, V = decltype(vc)::value, kRows = router::kThreads / W;
      router::set_shape(a, W, V, sizeof(T));
      hipStream_t s = static_cast<hipStream_t>(stream);
      if constexpr ((W == 16 && V > 4) || (W == 32 && V == 16))
        return router::launch_topk<router::topk_kernel<T, W, V, false>>(a, kRows, s);
      else if constexpr (W == 32 && V == 8)
        return router::launch_topk<router::topk_kernel<T, W, V, true>>(a, kRows, s);
      else
        return bias ? router::launch_topk<router::topk_kernel<T, W, V, true>>(a, kRows, s)
                    : router::launch_topk<router::topk_kernel<T, W, V, false>>(a, kRows, s);
    });
  });
}

extern "C" int afd_balance_workspace(int32_t n, int32_t num_experts, int32_t num_seqs, uint64_t* bytes) {
  if (!bytes || n < 0 || n > router::kMaxRows || num_seqs < 1 || num_seqs > router::kMaxSeqs) return AFD_ERR_ARG;
  if (num_experts < 1 || num_experts > router::kMaxExperts) return AFD_ERR_SHAPE;
  *bytes = router::plan(n, num_experts, num_seqs).total;
  return AFD_OK;
}

extern "C" int afd_topk_balance(const afd_router_cfg* cfg, const void* logits, int64_t ld, const float* bias,
                                const uint8_t* valid, const int32_t* cu_seqlens, int32_t num_seqs, int32_t n,
                                float alpha, int32_t* ids, float* w, int32_t* counts, float* coef, float* loss,
                                void* ws, uint64_t ws_bytes, afd_stream_t stream) {
  int st = router::check_cfg(cfg);
  if (st == AFD_OK) st = router::check_rows(n, cfg->topk);
  if (st == AFD_OK) st = router::check_logits(*cfg, logits, ld, n);
  if (st == AFD_OK) st = router::check_seqs(cu_seqlens, num_seqs);
  if (st != AFD_OK) return st;
  if (!counts || !coef || !loss || !ws || (n > 0 && (!ids || !w))) return AFD_ERR_ARG;
  const router::WsPlan p = router::plan(n, cfg->num_experts, num_seqs);
  if (ws_bytes < p.total || reinterpret_cast<uintptr_t>(ws) % 16) return AFD_ERR_WORKSPACE;
  router::Args a = router::base_args(*cfg, logits, ld, n);
  a.bias = bias;
  a.valid = valid;
  a.ids = ids;
  a.w = w;
  a.cu = cu_seqlens;
  a.seqs = num_seqs;
  a.alpha = alpha;
  a.counts = counts;
  a.coef = coef;
  a.loss = loss;
  router::place(a, ws, p);
  return router::launch_balance(a, cfg->logits_fmt, true, true, static_cast<hipStream_t>(stream));
}

extern "C" int afd_balance(const afd_router_cfg* cfg, const void* logits, int64_t ld, const int32_t* ids,
                           const uint8_t* valid, const int32_t* cu_seqlens, int32_t num_seqs, int32_t n, float alpha,
                           int32_t* counts, float* coef, float* loss, void* ws, uint64_t ws_bytes,
                           afd_stream_t stream) {
  int st = router::check_cfg(cfg);
  if (st == AFD_OK) st = router::check_rows(n, cfg->topk);
  if (st == AFD_OK) st = router::check_logits(*cfg, logits, ld, n);
  if (st == AFD_OK) st = router::check_seqs(cu_seqlens, num_seqs);
  if (st != AFD_OK) return st;
  if (!counts || !coef || !loss || !ws || (n > 0 && !ids)) return AFD_ERR_ARG;
  const router::WsPlan p = router::plan(n, cfg->num_experts, num_seqs);
  if (ws_bytes < p.total || reinterpret_cast<uintptr_t>(ws) % 16) return AFD_ERR_WORKSPACE;
  router::Args a = router::base_args(*cfg, logits, ld, n);
  a.groups = 1;  // the choice is made
  a.valid = valid;
  a.ids = const_cast<int32_t*>(ids);
  a.cu = cu_seqlens;
  a.seqs = num_seqs;
  a.alpha = alpha;
  a.counts = counts;
  a.coef = coef;
  a.loss = loss;
  router::place(a, ws, p);
  return router::launch_balance(a, cfg->logits_fmt, false, true, static_cast<hipStream_t>(stream));
}

extern "C" int afd_expert_counts(const int32_t* ids, int32_t n, int32_t topk, int32_t num_experts,
                                 const uint8_t* valid, const int32_t* cu_seqlens, int32_t num_seqs, int32_t* counts,
                                 void* ws, uint64_t ws_bytes, afd_stream_t stream) {
  if (num_experts < 1 || num_experts > router::kMaxExperts || topk < 1 || topk > router::kMaxTopk)
    return AFD_ERR_SHAPE;
  int st = router::check_rows(n, topk);
  if (st == AFD_OK) st = router::check_seqs(cu_seqlens, num_seqs);
  if (st != AFD_OK) return st;
  if (!counts || !ws || (n > 0 && !ids)) return AFD_ERR_ARG;
  const router::WsPlan p = router::plan(n, num_experts, num_seqs);
  if (ws_bytes < p.total || reinterpret_cast<uintptr_t>(ws) % 16) return AFD_ERR_WORKSPACE;
  router::Args a = {};
  a.ids = const_cast<int32_t*>(ids);
  a.n = n;
  a.topk = topk;
  a.experts = num_experts;
  a.groups = 1;
  a.valid = valid;
  a.cu = cu_seqlens;
  a.seqs = num_seqs;
  a.counts = counts;
  router::place(a, ws, p);
  // one workgroup a sequence up to 16384 ids, which may all be one sequence's (4096 ids 2.8 us against 5.6 in two
  // launches, 32768 ids 6.3, popular experts 10.5, against 5.7)
  if (n > 0 && int64_t(n) * topk <= router::kDirectIds) {
    hipLaunchKernelGGL(router::count_kernel, dim3(num_seqs), dim3(router::kCountThreads), 0,
                       static_cast<hipStream_t>(stream), a);
    AFD_CHECK_LAUNCH();
    return AFD_OK;
  }
  return router::launch_balance(a, AFD_LOGITS_F32, false, false, static_cast<hipStream_t>(stream));
}

extern "C" int afd_router_grad(const afd_router_cfg* cfg, const void* logits, int64_t ld, const int32_t* ids,
                               const uint8_t* valid, int32_t n, const float* gw, const int32_t* cu_seqlens,
                               int32_t num_seqs, const int32_t* counts, const float* coef, const float* gloss,
                               void* dlogits, afd_stream_t stream) {
  int st = router::check_cfg(cfg);
  if (st == AFD_OK) st = router::check_rows(n, cfg->topk);
  if (st == AFD_OK) st = router::check_logits(*cfg, logits, ld, n);
  if (st == AFD_OK && coef) st = router::check_seqs(cu_seqlens, num_seqs);
  if (st != AFD_OK) return st;
  if (coef && (!counts || !gloss)) return AFD_ERR_ARG;
  if (n == 0) return AFD_OK;
  if (!dlogits || (gw && !ids)) return AFD_ERR_ARG;
  router::Args a = router::base_args(*cfg, logits, ld, n);
  a.groups = 1;
  a.valid = valid;
  a.ids = const_cast<int32_t*>(ids);
  a.gw = gw;
  a.cu = cu_seqlens;
  a.seqs = num_seqs;
  a.counts = const_cast<int32_t*>(counts);
  a.coef = const_cast<float*>(coef);
  a.gloss = gloss;
  a.dlogits = dlogits;
  return router::with_logits(cfg->logits_fmt, [&](auto tag) {
    using T = decltype(tag);
    return router::with_shape(a.experts, router::lanes_needed(a, false), [&](auto wc, auto vc) {
      constexpr int W = decltype(wc)::value, V = decltype(vc)::value;
      a.block_rows = router::block_rows_for(n, W, router::kThreads, 2048);
      a.blocks = router::blocks_for(n, a.block_rows);
      router::set_shape(a, W, V, sizeof(T));
      hipLaunchKernelGGL((router::grad_kernel<T, W, V>), dim3(a.blocks), dim3(router::kThreads), 0,
                         static_cast<hipStream_t>(stream), a);
      AFD_CHECK_LAUNCH();
      return int(AFD_OK);
    });
  });
}
