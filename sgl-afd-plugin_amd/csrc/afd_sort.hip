// Tokens sorted by expert and back, on gfx950. Pair p = t topk + j sends token t to expert ids[p]; with e = ids[p] -
// expert_lo a pair with 0 <= e < num_experts is here, the others are nowhere (position -1):
//
//   position[p] = #{pairs here with (e', p') < (e, p)}          rows[position[p]] = x[t]
//   out[t] = sum_j w[t, j] rows[position[t, j]]                  (j ascending, in fp32, rounded once)
//   d rows[position[p]] = w[p] d out[t],  d w[p] = < d out[t], rows[position[p]] >,  d x[t] = sum_j d rows[position[t, j]]
//
// All of it moves rows: bound by HBM where there are many, by launches and latency where there are few.
#include "afd_common.h"
#include "afd_internal.h"
#include "afd_rows_dev.h"

namespace afd {
namespace sorting {

using namespace rows;

constexpr int kMaxExperts = 1024;
constexpr int kMaxTokens = 1 << 26;
constexpr int kMaxColumns = 65536;

// ---------------------------------------------------------------- positions
struct Pairs {
  const int32_t* ids;
  int32_t pairs, expert_lo, experts;
  int32_t *positions, *counts, *offsets;
};
__device__ __forceinline__ int expert_of(const Pairs& p, int i) {
  const int32_t id = p.ids[i];
  return id >= p.expert_lo && id - p.expert_lo < p.experts ? id - p.expert_lo : -1;  // (expert_lo >= 0: no difference wraps)
}

// Exclusive sums of v over the THREADS threads of a workgroup, and the total. waves: LDS, one a wavefront
template <int THREADS>
__device__ __forceinline__ int scan(int v, int* waves, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(s, d);
    if (lane >= d) s += o;
  }
  if (lane == 63) waves[w] = s;
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < THREADS / 64; ++i) {
    before += i < w ? waves[i] : 0;
    all += waves[i];
  }
  *total = all;
  return before + s - v;
}

// ---------------------------------------------------------------- moving
// x's row t to each of its positions, 16 bytes at a time. VEC: rows are aligned and made of whole ones; else at the
// alignment they have, with up to seven pieces of 2 bytes behind the last. A token is L lanes' work.
struct Move {
  const char* x;
  char* rows;
  int64_t ldx, ld;  // in bytes
  int32_t bytes, n, topk;
  int32_t behind;  // whether rows past the last pair's, up to n topk, are zeroed
};
template <bool VEC, bool NT, int L>
__device__ __forceinline__ void move_token(const Move& m, int64_t t, const int* at, int lane) {
  const char* from = m.x + t * m.ldx;
  const int words = m.bytes / 16;
  for (int u = lane; u < words; u += L) {
    const v4i v = load_words<VEC>(from + 16 * u);
    for (int j = 0; j < m.topk; ++j)
      if (at[j] >= 0) store_words<VEC, NT>(m.rows + at[j] * m.ld + 16 * u, v);
  }
  if constexpr (!VEC) {
    const int left = words * 8 + lane;  // (pieces of 2 bytes)
    if (left < m.bytes / 2) {
      const uint16_t v = reinterpret_cast<const uint16_t*>(from)[left];
      for (int j = 0; j < m.topk; ++j)
        if (at[j] >= 0) reinterpret_cast<uint16_t*>(m.rows + at[j] * m.ld)[left] = v;
    }
  }
}
template <bool VEC, int L>
__device__ __forceinline__ void zero_behind(const Move& m, int64_t t, int total, int lane) {
  if (!m.behind) return;
  for (int64_t r = int64_t(total) + t; r < int64_t(m.n) * m.topk; r += m.n) {
    char* row = m.rows + r * m.ld;
    for (int u = lane; u < m.bytes / 16; u += L) store_words<VEC>(row + 16 * u, v4i{0, 0, 0, 0});
    if constexpr (!VEC) {
      const int left = m.bytes / 16 * 8 + lane;
      if (left < m.bytes / 2) reinterpret_cast<uint16_t*>(row)[left] = 0;
    }
  }
}

// Few pairs: one launch. A workgroup for each token and one more: each reads all pairs' ids (at most 16 a lane) and
// counts the pairs before its own: a pair's key is (expert, pair), and its position the number of smaller keys. The one more writes
// the tables. 8 tokens of 4096 to 8 of 256 experts: 6.2 us in a trace, where a launch that does nothing takes 1.4; three
// launches take 13.7 for 6124 pairs. The limit is what 16 keys a lane hold; beside it the two forms have not been compared.
constexpr int kFewThreads = 256, kFewEach = 16, kFewPairs = kFewThreads * kFewEach;
template <bool VEC>
__global__ __launch_bounds__(kFewThreads) void few_kernel(Pairs p, Move m) {
  constexpr int kWaves = kFewThreads / 64;
  __shared__ int part[kWaves][kMaxTopk + 1];
  __shared__ int at[kMaxTopk];
  __shared__ int hist[kMaxExperts];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  uint32_t key[kFewEach];
#pragma unroll
  for (int i = 0; i < kFewEach; ++i) {
    const int at = i * kFewThreads + t;
    const int e = at < p.pairs ? expert_of(p, at) : -1;
    key[i] = e < 0 ? 0xffffffffu : static_cast<uint32_t>(e * p.pairs + at);
  }
  if (static_cast<int>(blockIdx.x) == m.n) {
    for (int e = t; e < p.experts; e += kFewThreads) hist[e] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kFewEach; ++i)
      if (key[i] != 0xffffffffu) atomicAdd(&hist[key[i] / static_cast<uint32_t>(p.pairs)], 1);
    __syncthreads();
    constexpr int kEach = kMaxExperts / kFewThreads;
    int c[kEach], sum = 0, total;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      c[i] = t * kEach + i < p.experts ? hist[t * kEach + i] : 0;
      sum += c[i];
    }
    int before = scan<kFewThreads>(sum, &part[0][0], &total);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int e = t * kEach + i;
      if (e < p.experts) {
        p.counts[e] = c[i];
        p.offsets[e] = before;
      }
      before += c[i];
    }
    if (t == 0) p.offsets[p.experts] = total;
    return;
  }
  const int64_t token = blockIdx.x;
  for (int j = 0; j <= m.topk; ++j) {
    // (the last: the number of pairs that are here)
    const int i0 = static_cast<int>(token) * m.topk + j;
    const int e = j < m.topk ? expert_of(p, i0) : 0;
    const uint32_t own = j < m.topk ? static_cast<uint32_t>(e * p.pairs + i0) : 0xffffffffu;
    int before = 0;
#pragma unroll
    for (int i = 0; i < kFewEach; ++i)
      if (i * kFewThreads < p.pairs) before += __popcll(__ballot(key[i] < own));
    if (lane == 0) part[w][j] = before;
  }
  __syncthreads();
  if (t < m.topk) {
    int pos = -1;
    if (expert_of(p, static_cast<int>(token) * m.topk + t) >= 0) {
      pos = 0;
      for (int i = 0; i < kWaves; ++i) pos += part[i][t];
    }
    at[t] = pos;
    p.positions[token * m.topk + t] = pos;
  }
  int total = 0;
  for (int i = 0; i < kWaves; ++i) total += part[i][m.topk];
  __syncthreads();
  move_token<VEC, false, kFewThreads>(m, token, at, t);
  zero_behind<VEC, kFewThreads>(m, token, total, t);
}

// Many pairs: chunks of a multiple of 1024, at most kMaxChunks. Each chunk's counts by expert, then each chunk's
// positions from the counts of all chunks (which every workgroup adds up), then the rows (131072 pairs of 256 experts: 4.7 and
// 5.4 us before the rows' 83).
constexpr int kChunk = 1024, kMaxChunks = 256, kChunkWaves = kChunk / 64;

inline int chunk_of(int64_t pairs) {
  const int64_t c = (pairs + kMaxChunks - 1) / kMaxChunks;
  return static_cast<int>((c + kChunk - 1) / kChunk * kChunk);
}

// hist [chunks][experts]
__global__ __launch_bounds__(kChunk) void count_kernel(Pairs p, int chunk, int32_t* __restrict__ hist) {
  __shared__ int cnt[kMaxExperts];
  const int t = threadIdx.x;
  if (t < p.experts) cnt[t] = 0;
  __syncthreads();
  const int64_t lo = int64_t(blockIdx.x) * chunk, hi = min(lo + chunk, int64_t(p.pairs));
  for (int64_t i = lo + t; i < hi; i += kChunk) {
    const int e = expert_of(p, static_cast<int>(i));
    if (e >= 0) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  if (t < p.experts) hist[int64_t(blockIdx.x) * p.experts + t] = cnt[t];
}

__global__ __launch_bounds__(kChunk) void place_kernel(Pairs p, int chunk, const int32_t* __restrict__ hist) {
  __shared__ int all_part[kChunk], before_part[kChunk];
  __shared__ int run[kMaxExperts];
  __shared__ int waves[kChunkWaves];
  __shared__ int wcnt[kChunkWaves][kMaxExperts];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int chunks = gridDim.x, c = blockIdx.x;
  // experts' counts in all chunks and in those before this one: the chunks are dealt to kChunk / experts threads
  // an expert
  const int groups = kChunk / p.experts, e = t % p.experts, g = t / p.experts;
  int all = 0, before = 0;
  if (g < groups)
#pragma unroll 8
    for (int i = g; i < chunks; i += groups) {
      const int v = hist[int64_t(i) * p.experts + e];
      all += v;
      before += i < c ? v : 0;
    }
  all_part[t] = all;
  before_part[t] = before;
  for (int i = t; i < kChunkWaves * kMaxExperts; i += kChunk) (&wcnt[0][0])[i] = 0;
  __syncthreads();
  all = before = 0;
  if (t < p.experts)
    for (int i = 0; i < groups; ++i) {
      all += all_part[i * p.experts + t];
      before += before_part[i * p.experts + t];
    }
  int total;
  const int first = scan<kChunk>(all, waves, &total);
  if (t < p.experts) {
    run[t] = first + before;
    if (c == 0) {
      p.counts[t] = all;
      p.offsets[t] = first;
    }
  }
  if (c == 0 && t == 0) p.offsets[p.experts] = total;
  __syncthreads();
  const uint64_t below = (uint64_t(1) << lane) - 1;
  const int64_t lo = int64_t(c) * chunk, hi = min(lo + chunk, int64_t(p.pairs));
  for (int64_t i0 = lo; i0 < hi; i0 += kChunk) {
    const int64_t i = i0 + t;
    const int key = i < hi ? expert_of(p, static_cast<int>(i)) : -1;
    // the wavefront's lanes with the same expert (-1 has all bits set)
    uint64_t peers = ~uint64_t(0);
#pragma unroll
    for (int b = 0; b <= 10; ++b) {
      const uint64_t with = __ballot((key >> b) & 1);
      peers &= (key >> b) & 1 ? with : ~with;
    }
    const int rank = __popcll(peers & below);
    if (key >= 0 && rank == 0) wcnt[w][key] = __popcll(peers);
    __syncthreads();
    if (i < hi) {
      int pos = -1;
      if (key >= 0) {
        pos = run[key] + rank;
        for (int o = 0; o < w; ++o) pos += wcnt[o][key];
      }
      p.positions[i] = pos;
    }
    __syncthreads();
    if (i0 + kChunk < hi) {
      if (t < p.experts) {
        int add = 0;
        for (int o = 0; o < kChunkWaves; ++o) {
          add += wcnt[o][t];
          wcnt[o][t] = 0;
        }
        run[t] += add;
      }
      __syncthreads();
    }
  }
}

// A wavefront a token. NT: past the caches, where all pairs' rows would be more than kPastBytes, whichever of them are here. It is
// even over a pass and not best everywhere: 16384 x 4096 with a quarter of the 8 experts here 83 us for 88 through the caches,
// and the way back behind it 69 for 72; 8192 x 2048 with all here 78 for 60, the way back 58 for 61 (twice) and its gradient 116
// for 127, the pass 310 for 309; 2048 x 2048 (67 MB of rows, which the memory-side cache holds) 18.7 for 15.0
template <bool VEC, bool NT>
__global__ __launch_bounds__(256) void move_kernel(Move m, const int32_t* __restrict__ positions,
                                                   const int32_t* __restrict__ total) {
  const int64_t t = block_of_many() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= m.n) return;
  const int lane = threadIdx.x & 63;
  move_token<VEC, NT, 64>(m, t, positions + t * m.topk, lane);
  if (m.behind) zero_behind<VEC, 64>(m, t, *total, lane);
}

// ---------------------------------------------------------------- back
struct Back {
  const void* rows;
  int64_t ld;
  const int32_t* positions;
  const float* w;  // null: ones
  int32_t n, topk, columns;
  int64_t num_rows;
  void* out;
  // the gradient's
  const void* g;  // [n][columns]
  void* d_rows;   // [num_rows][columns]
  float* d_w;
  const int32_t* total;
};
// the position of pair i, -1 if there is no such row
__device__ __forceinline__ int64_t position_of(const Back& p, int64_t i) {
  const int64_t at = p.positions[i];
  return at < p.num_rows ? at : -1;
}

// A wavefront a token's 512 columns, kBatch of its rows on their way at once; rows are read once: past the caches. No
// loop over the columns, so that many short wavefronts keep loads on their way whatever share of the pairs is here (8192 x 2048
// with 8 rows a token 58 us, 5.2 TB/s, where a wavefront for all of a token's columns took 77; 16384 x 4096 with 2 of 8 here 68
// for 119; 8 tokens 3.8 for 5.7).
constexpr int kBatch = 8;
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void back_kernel(Back p, uint32_t chunks) {
  using R = Row<T, 64, VEC>;
  using Held = typename T::Held;
  const uint64_t item = uint64_t(block_of_many()) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = static_cast<int64_t>(item / chunks);
  if (t >= p.n) return;
  const int c = static_cast<int>(item % chunks), lane = threadIdx.x & 63;
  const Held* rows = static_cast<const Held*>(p.rows);
  float acc[8] = {};
  for (int j0 = 0; j0 < p.topk; j0 += kBatch) {
    typename R::Raw raw[kBatch];
    float w[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int64_t i = t * p.topk + min(j0 + j, p.topk - 1), at = j0 + j < p.topk ? position_of(p, i) : -1;
      w[j] = at < 0 ? 0.0f : p.w ? p.w[i] : 1.0f;
      raw[j] = {};
      if (at >= 0) raw[j] = R::template fetch<true>(rows + at * p.ld, p.columns, lane, c);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      float v[8];
      raw[j].widen(v);
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] = __builtin_fmaf(w[j], v[q], acc[q]);
    }
  }
  R::store(static_cast<Held*>(p.out) + t * p.columns, p.columns, lane, c, acc);
}

// The gradient of the rows and the weights, a token at a time: its row of g is read for each batch of its pairs (once where
// there are no more), the pairs' rows once. 8192 x 2048 with 8 rows a token: 116 us, 4.9 TB/s
template <typename T, int L, bool VEC>
__global__ __launch_bounds__(256) void back_grad_kernel(Back p) {
  using R = Row<T, L, VEC>;
  using Held = typename T::Held;
  __shared__ float part[2][4 * kBatch];
  const int64_t t = block_of_many() * (256 / L) + (L == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
  if (t >= p.n) return;
  const int lane = threadIdx.x & (L - 1);
  const Held* rows = static_cast<const Held*>(p.rows);
  const Held* g = static_cast<const Held*>(p.g) + t * p.columns;
  Held* d_rows = static_cast<Held*>(p.d_rows);
  int turn = 0;  // of the LDS that the sums meet in
  for (int j0 = 0; j0 < p.topk; j0 += kBatch) {
    int64_t at[kBatch];
    float w[kBatch], dot[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int64_t i = t * p.topk + min(j0 + j, p.topk - 1);
      at[j] = j0 + j < p.topk ? position_of(p, i) : -1;
      w[j] = p.w ? p.w[i] : 1.0f;
      dot[j] = 0.0f;
    }
    for (int c = 0; c * L * 8 < p.columns; ++c) {
      float go[8];
      typename R::Raw raw[kBatch];
      const typename R::Raw g_raw = R::fetch(g, p.columns, lane, c);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        raw[j] = {};
        if (p.d_w && at[j] >= 0) raw[j] = R::template fetch<true>(rows + at[j] * p.ld, p.columns, lane, c);
      }
      g_raw.widen(go);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (at[j] < 0) continue;
        float v[8];
        if (p.d_w) {
          raw[j].widen(v);
#pragma unroll
          for (int q = 0; q < 8; ++q) dot[j] = __builtin_fmaf(go[q], v[q], dot[j]);
        }
        if (p.d_rows) {
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] = w[j] * go[q];
          R::store(d_rows + at[j] * p.columns, p.columns, lane, c, v);
        }
      }
    }
    if (p.d_w) {
      row_sum<L>(dot, part[turn ^= 1], lane);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (lane == 0 && j0 + j < p.topk) p.d_w[t * p.topk + j0 + j] = at[j] < 0 ? 0.0f : dot[j];
    }
  }
  // rows that no pair has
  if (p.d_rows) {
    const float zero[8] = {};
    for (int64_t r = max(*p.total, 0) + t; r < p.num_rows; r += p.n)
      for (int c = 0; c * L * 8 < p.columns; ++c) R::store(d_rows + r * p.columns, p.columns, lane, c, zero);
  }
}

// ---------------------------------------------------------------- host
static int check(int32_t n, int32_t topk, int32_t fmt, int32_t columns) {
  if (n < 0 || n > kMaxTokens) return AFD_ERR_ARG;
  if (topk < 1 || topk > kMaxTopk || int64_t(n) * topk > 0x7fffffff || columns < 1 || columns > kMaxColumns) return AFD_ERR_SHAPE;
  return known_fmt(fmt) ? AFD_OK : AFD_ERR_UNSUPPORTED;
}

template <bool VEC>
static int launch_sort(const Pairs& p, const Move& m, int32_t* hist, hipStream_t s) {
  if (p.pairs <= kFewPairs) {
    hipLaunchKernelGGL(few_kernel<VEC>, dim3(m.n + 1), dim3(kFewThreads), 0, s, p, m);
    AFD_CHECK_LAUNCH();
    return AFD_OK;
  }
  const int chunk = chunk_of(p.pairs);
  const dim3 chunks(static_cast<unsigned>((int64_t(p.pairs) + chunk - 1) / chunk));
  hipLaunchKernelGGL(count_kernel, chunks, dim3(kChunk), 0, s, p, chunk, hist);
  AFD_CHECK_LAUNCH();
  hipLaunchKernelGGL(place_kernel, chunks, dim3(kChunk), 0, s, p, chunk, hist);
  AFD_CHECK_LAUNCH();
  const dim3 grid = grid_of_many((int64_t(m.n) + 3) / 4);
  if (VEC && int64_t(p.pairs) * m.bytes > kPastBytes)
    hipLaunchKernelGGL((move_kernel<VEC, VEC>), grid, dim3(256), 0, s, m, p.positions, p.offsets + p.experts);
  else
    hipLaunchKernelGGL((move_kernel<VEC, false>), grid, dim3(256), 0, s, m, p.positions, p.offsets + p.experts);
  AFD_CHECK_LAUNCH();
  return AFD_OK;
}

// tokens of fewer are a workgroup's work each, of more a wavefront's
constexpr int kFewTokens = 1024;
template <typename F>
static int with_shape(const Back& p, int32_t fmt, bool vec, F f) {
  return with_fmt(fmt, [&](auto type) -> int {
    auto go = [&](auto lanes) {
      constexpr int L = decltype(lanes)::value;
      const dim3 grid = grid_of_many((int64_t(p.n) * L + 255) / 256);
      if (vec)
        f(type, lanes, std::true_type{}, grid);
      else
        f(type, lanes, std::false_type{}, grid);
    };
    if (p.n < kFewTokens)
      go(std::integral_constant<int, 256>{});
    else
      go(std::integral_constant<int, 64>{});
    AFD_CHECK_LAUNCH();
    return AFD_OK;
  });
}

}  // namespace sorting
}  // namespace afd

using namespace afd;

extern "C" int afd_sort_workspace(int32_t n, int32_t topk, int32_t num_experts, uint64_t* bytes) {
  if (!bytes) return AFD_ERR_ARG;
  const int st = sorting::check(n, topk, AFD_V_F32, 1);
  if (st != AFD_OK) return st;
  if (num_experts < 1 || num_experts > sorting::kMaxExperts) return AFD_ERR_SHAPE;
  const int64_t pairs = int64_t(n) * topk;
  const int64_t chunk = pairs > sorting::kFewPairs ? sorting::chunk_of(pairs) : pairs + 1;
  *bytes = static_cast<uint64_t>((pairs + chunk - 1) / chunk * num_experts * 4);
  if (pairs <= sorting::kFewPairs) *bytes = 0;
  return AFD_OK;
}

extern "C" int afd_sort_tokens(int32_t fmt, const int32_t* ids, int32_t n, int32_t topk, int32_t expert_lo,
                               int32_t num_experts, const void* x, int64_t ldx, int32_t columns, void* rows, int64_t ld,
                               int32_t zero_behind, int32_t* positions, int32_t* counts, int32_t* offsets, void* ws,
                               uint64_t ws_bytes, afd_stream_t stream) {
  const int st = sorting::check(n, topk, fmt, columns);
  if (st != AFD_OK) return st;
  uint64_t need;
  const int sized = afd_sort_workspace(n, topk, num_experts, &need);
  if (sized != AFD_OK) return sized;
  if (ldx < columns || ld < columns) return AFD_ERR_SHAPE;
  if (expert_lo < 0) return AFD_ERR_ARG;
  if (!counts || !offsets || (n > 0 && (!ids || !x || !rows || !positions))) return AFD_ERR_ARG;
  if (need > 0 && (!ws || ws_bytes < need || reinterpret_cast<uintptr_t>(ws) % 4)) return AFD_ERR_WORKSPACE;
  const sorting::Pairs p = {ids, n * topk, expert_lo, num_experts, positions, counts, offsets};
  const int size = rows::value_size(fmt);
  const sorting::Move m = {static_cast<const char*>(x), static_cast<char*>(rows), ldx * size, ld * size, columns * size,
                           n, topk, zero_behind};
  int32_t* hist = static_cast<int32_t*>(ws);
  const bool vec = rows::aligned_rows(x, ldx, fmt) && rows::aligned_rows(rows, ld, fmt) && m.bytes % 16 == 0;
  return vec ? sorting::launch_sort<true>(p, m, hist, static_cast<hipStream_t>(stream))
             : sorting::launch_sort<false>(p, m, hist, static_cast<hipStream_t>(stream));
}

extern "C" int afd_unsort_tokens(int32_t fmt, const void* rows, int64_t ld, int64_t num_rows, const int32_t* positions,
                                 const float* w, int32_t n, int32_t topk, int32_t columns, void* out, afd_stream_t stream) {
  const int st = sorting::check(n, topk, fmt, columns);
  if (st != AFD_OK) return st;
  if (ld < columns || num_rows < 0) return AFD_ERR_SHAPE;
  if (n == 0) return AFD_OK;
  if ((!rows && num_rows > 0) || !positions || !out) return AFD_ERR_ARG;
  sorting::Back p = {};
  p.rows = rows;
  p.ld = ld;
  p.positions = positions;
  p.w = w;
  p.n = n;
  p.topk = topk;
  p.columns = columns;
  p.num_rows = num_rows;
  p.out = out;
  const bool vec = rows::aligned_rows(rows, ld, fmt) && rows::aligned_rows(out, columns, fmt) && columns % 8 == 0;
  const uint32_t chunks = (columns + 511) / 512;
  return rows::with_fmt(fmt, [&](auto type) -> int {
    using T = decltype(type);
    const dim3 blocks = rows::grid_of_many((int64_t(n) * chunks + 3) / 4);
    if (vec)
      hipLaunchKernelGGL((sorting::back_kernel<T, true>), blocks, dim3(256), 0, static_cast<hipStream_t>(stream), p, chunks);
    else
      hipLaunchKernelGGL((sorting::back_kernel<T, false>), blocks, dim3(256), 0, static_cast<hipStream_t>(stream), p, chunks);
    AFD_CHECK_LAUNCH();
    return AFD_OK;
  });
}

extern "C" int afd_unsort_grad(int32_t fmt, const void* g, const void* rows, int64_t ld, int64_t num_rows,
                               const int32_t* positions, const int32_t* total, const float* w, int32_t n, int32_t topk,
                               int32_t columns, void* d_rows, float* d_w, afd_stream_t stream) {
  const int st = sorting::check(n, topk, fmt, columns);
  if (st != AFD_OK) return st;
  if (num_rows < 0 || (d_w && ld < columns)) return AFD_ERR_SHAPE;
  if (n == 0 || (!d_rows && !d_w)) return AFD_OK;
  if (!g || !positions || (d_w && num_rows > 0 && !rows) || (d_rows && !total)) return AFD_ERR_ARG;
  sorting::Back p = {};
  p.rows = rows;
  p.ld = ld;
  p.positions = positions;
  p.w = w;
  p.n = n;
  p.topk = topk;
  p.columns = columns;
  p.num_rows = num_rows;
  p.g = g;
  p.d_rows = d_rows;
  p.d_w = d_w;
  p.total = total;
  const bool vec = rows::aligned_rows(d_w ? rows : nullptr, ld, fmt) && rows::aligned_rows(g, columns, fmt) &&
                   rows::aligned_rows(d_rows, columns, fmt) && columns % 8 == 0;
  return sorting::with_shape(p, fmt, vec, [&](auto type, auto lanes, auto v, dim3 grid) {
    hipLaunchKernelGGL((sorting::back_grad_kernel<decltype(type), decltype(lanes)::value, decltype(v)::value>), grid, dim3(256),
                       0, static_cast<hipStream_t>(stream), p);
  });
}
