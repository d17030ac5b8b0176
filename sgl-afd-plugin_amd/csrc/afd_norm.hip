// The norms before and after a block, its gate and the residual's scale in one pass over a token's row, on gfx950:
//
//   rms(v) = v / sqrt(mean(v^2) + eps)
//   h = residual + scale gate (rms(y) w_post, or y)          normed = rms(h) w_next
//
// y: the block's output; gate: none, one value per channel, per token or per element. Without y, h is the residual itself and
// normed the norm before a block. A row's values stay in registers in fp32 from its one read to what is written, each
// result rounded once (normed is that of h before h is rounded).
//
// The gradient, from that of h (dh) and of normed (dn), with u = rms(h), v = rms(y):
//
//   d = dh + r_h (g - u mean(g u)),  g = dn w_next            d residual = d
//   d w_next = sum_t dn u
//   (h is made again from y and the residual: in fp32, as normed saw it)
//   d y = r_y (q - v mean(q v)),  q = scale gate w_post d     (without the norm: scale gate d)
//   d w_post = sum_t scale gate d v,  d gate = scale d v w_post, summed over what shares the gate's value
//
// Sums over tokens have one order: a workgroup adds up its own tokens in registers, and a second launch the workgroups'.
#include "afd_common.h"
#include "afd_internal.h"
#include "afd_rows_dev.h"

namespace afd {
namespace norm {

using namespace rows;

constexpr int kMaxTokens = 1 << 26;

struct Args {
  const void *y, *residual;
  int64_t ldy, ldr;
  const void *w_post, *gate, *w_next;
  bool wide_post, wide_gate, wide_next;  // held in fp32
  int32_t gate_kind;
  bool post;
  float scale, eps;
  int32_t n, columns;
  void *h, *normed;
  float* rstd;  // [2][n]: of y, of h
  // the gradient's
  const void *dh, *dn;
  void *d_res, *d_y, *d_gate;
  float* sums;  // [slots][2][columns]: of w_next, of w_post and the channels' gate
  bool sum_next, sum_block;
  bool block;  // anything that belongs to y is wanted
};

// a lane's chunk of a parameter's row, which is held in T or in fp32. VEC only where both are aligned
template <typename T, int L, bool VEC>
__device__ __forceinline__ void load_param(const void* p, bool wide, int64_t offset, int columns, int lane, int c, float (&v)[8]) {
  if (wide)
    Row<F32, L, VEC>::load(static_cast<const float*>(p) + offset, columns, lane, c, v);
  else
    Row<T, L, VEC>::load(static_cast<const typename T::Held*>(p) + offset, columns, lane, c, v);
}
template <typename T>
__device__ __forceinline__ float load_one(const void* p, bool wide, int64_t at) {
  return wide ? static_cast<const float*>(p)[at] : T::wide(static_cast<const typename T::Held*>(p)[at]);
}

// A row is L lanes' of NC chunks each. With L 64 a workgroup has four, a wavefront each, and no barrier.
template <int L>
constexpr int kThreads = L == 64 ? 256 : L;
template <int L>
constexpr int kRows = kThreads<L> / L;
template <int L>
__device__ __forceinline__ int64_t first_row() {
  return block_of_many() * kRows<L> + (L == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
}

// 1 / sqrt(mean of the squares of a row's values + eps). Where their sum leaves fp32 (ss is the row's, so all of its lanes agree)
// it is made again of values scaled by a power of two, so any row of numbers has its root; one that holds an infinity
// gets 0. part: LDS as row_sum's, two of them
template <int L, int NC>
__device__ __forceinline__ float inv_root(const float (&v)[NC][8], float inv, float eps, float* part, float* again, int lane) {
  float ss[1] = {0.0f};
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) ss[0] = __builtin_fmaf(v[c][j], v[c][j], ss[0]);
  row_sum<L>(ss, part, lane);
  if (ss[0] != __builtin_inff()) return 1.0f / sqrtf(__builtin_fmaf(ss[0], inv, eps));
  constexpr float kDown = 0x1p-72f;  // 16384 squares of the largest float are then 2^126
  float small[1] = {0.0f};
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) small[0] = __builtin_fmaf(kDown * v[c][j], kDown * v[c][j], small[0]);
  row_sum<L>(small, again, lane);
  return kDown / sqrtf(__builtin_fmaf(small[0], inv, kDown * (kDown * eps)));
}

// NT: results past the caches, where they are more than those hold (16384 x 4096 bf16 96.5 -> 95.2 us; 8192 rows in training 58 ->
// 61, and the gradient behind it 83 -> 72)
template <typename T, int L, int NC, bool VEC, bool NT>
__global__ __launch_bounds__(kThreads<L>) void forward_kernel(Args p) {
  using R = Row<T, L, VEC>;
  using Held = typename T::Held;
  __shared__ float part[3][L / 64];  // (the third one's two uses have the second's barrier between them)
  const int64_t t = first_row<L>();
  if (t >= p.n) return;  // (a whole wavefront, and with one row a workgroup none)
  const int lane = threadIdx.x & (L - 1), columns = p.columns;
  const float inv = 1.0f / static_cast<float>(columns);
  const bool vector = p.gate_kind == AFD_GATE_CHANNEL || p.gate_kind == AFD_GATE_ELEMENT;
  typename R::Raw h_raw[NC], y_raw[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) h_raw[c] = R::fetch(static_cast<const Held*>(p.residual) + t * p.ldr, columns, lane, c);
  float h[NC][8], w_next[NC][8];
  if (p.y) {
    float y[NC][8], w[NC][8], g[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      y_raw[c] = R::fetch(static_cast<const Held*>(p.y) + t * p.ldy, columns, lane, c);
      if (p.post) load_param<T, L, VEC>(p.w_post, p.wide_post, 0, columns, lane, c, w[c]);
      if (vector)
        load_param<T, L, VEC>(p.gate, p.wide_gate, p.gate_kind == AFD_GATE_ELEMENT ? t * columns : 0, columns, lane, c, g[c]);
      if (p.normed) load_param<T, L, VEC>(p.w_next, p.wide_next, 0, columns, lane, c, w_next[c]);
    }
    const float s = p.gate_kind == AFD_GATE_TOKEN ? p.scale * load_one<T>(p.gate, p.wide_gate, t) : p.scale;
#pragma unroll
    for (int c = 0; c < NC; ++c) y_raw[c].widen(y[c]);
    if (p.post) {
      const float r = inv_root<L, NC>(y, inv, p.eps, part[0], part[2], lane);
      if (p.rstd && lane == 0) p.rstd[t] = r;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) y[c][j] = y[c][j] * r * w[c][j];
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      h_raw[c].widen(h[c]);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[c][j] = __builtin_fmaf(vector ? g[c][j] * s : s, y[c][j], h[c][j]);
    }
    if (p.h)
#pragma unroll
      for (int c = 0; c < NC; ++c) R::template store<NT>(static_cast<Held*>(p.h) + t * columns, columns, lane, c, h[c]);
  } else {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (p.normed) load_param<T, L, VEC>(p.w_next, p.wide_next, 0, columns, lane, c, w_next[c]);
      h_raw[c].widen(h[c]);
    }
  }
  if (p.normed) {
    const float r = inv_root<L, NC>(h, inv, p.eps, part[1], part[2], lane);
    if (p.rstd && lane == 0) p.rstd[int64_t(p.n) + t] = r;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int j = 0; j < 8; ++j) h[c][j] = h[c][j] * r * w_next[c][j];
      R::template store<NT>(static_cast<Held*>(p.normed) + t * columns, columns, lane, c, h[c]);
    }
  }
}

// Slot s (of gridDim.x kRows) takes every slots-th row, the next one's values on their way while it works on one. The
// slot's sums over its rows stay in registers, and so do the parameters: w_next and k = scale w_post (the channels' gate).
// With g the row's or the element's gate (1 without) everything of the block goes through k and one sum,
//
//   h = residual + g k v,   q = g k d,   a = sum_t g d v
//   d w_post = scale (the channels' gate) a,   the channels' d gate = scale w_post a,   others': k d v, or its sum over the row
//
// 18 operations a value and 16 registers of sums for 8 columns, so that 16 wavefronts fit a CU: 8192 x 4096 bf16 with a gate per
// channel 72 us (5.6 TB/s), where sums of each parameter's own and parameters from LDS took 141, without a row ahead 160.
template <typename T, int L, int NC, bool VEC>
__global__ __launch_bounds__(kThreads<L>) __attribute__((amdgpu_waves_per_eu(sizeof(typename T::Held) == 2 && VEC ? 4 : 2))) void
backward_kernel(Args p) {
  using R = Row<T, L, VEC>;
  using Held = typename T::Held;
  __shared__ float part[2][L / 64];
  const int64_t slot = first_row<L>(), slots = int64_t(gridDim.x) * kRows<L>;
  const int lane = threadIdx.x & (L - 1), columns = p.columns;
  const float inv = 1.0f / static_cast<float>(columns);
  int turn = 0;  // of the LDS that a row's sums meet in
  const bool element = p.gate_kind == AFD_GATE_ELEMENT, token = p.gate_kind == AFD_GATE_TOKEN;
  float sum_next[NC][8] = {}, sum_block[NC][8] = {};
  float w_next[NC][8], k[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (p.dn) load_param<T, L, VEC>(p.w_next, p.wide_next, 0, columns, lane, c, w_next[c]);
#pragma unroll
    for (int j = 0; j < 8; ++j) k[c][j] = p.scale;
    float w[8];
    if (p.post) {
      load_param<T, L, VEC>(p.w_post, p.wide_post, 0, columns, lane, c, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) k[c][j] *= w[j];
    }
    if (p.gate_kind == AFD_GATE_CHANNEL) {
      load_param<T, L, VEC>(p.gate, p.wide_gate, 0, columns, lane, c, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) k[c][j] *= w[j];
    }
  }
  // what a row needs
  struct In {
    typename R::Raw dh[NC], dn[NC], res[NC], y[NC];
    float gate, r_y, r_h;
  };
  auto fetch = [&](int64_t t) {
    In in = {};
    if (t >= p.n) return in;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (p.dh) in.dh[c] = R::fetch(static_cast<const Held*>(p.dh) + t * columns, columns, lane, c);
      if (p.dn) in.dn[c] = R::fetch(static_cast<const Held*>(p.dn) + t * columns, columns, lane, c);
      if (p.dn) in.res[c] = R::fetch(static_cast<const Held*>(p.residual) + t * p.ldr, columns, lane, c);
      if (p.y) in.y[c] = R::fetch(static_cast<const Held*>(p.y) + t * p.ldy, columns, lane, c);
    }
    in.gate = token ? load_one<T>(p.gate, p.wide_gate, t) : 1.0f;
    in.r_y = p.post ? p.rstd[t] : 1.0f;
    in.r_h = p.dn ? p.rstd[int64_t(p.n) + t] : 0.0f;
    return in;
  };
  constexpr bool kAhead = NC == 1;  // (two chunks a lane leave no registers for another row)
  In next = {};
  if constexpr (kAhead) next = fetch(slot);
  for (int64_t t = slot; t < p.n; t += slots) {
    const In in = kAhead ? next : fetch(t);
    if constexpr (kAhead) next = fetch(t + slots);
    float g[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (element) {
        load_param<T, L, VEC>(p.gate, p.wide_gate, t * columns, columns, lane, c, g[c]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[c][j] = in.gate;
      }
    }
    // v: rms(y), or y (0 where it is not needed)
    float d[NC][8], v[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      in.dh[c].widen(d[c]);
      in.y[c].widen(v[c]);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] *= in.r_y;
    }
    if (p.dn) {
      float u[NC][8], e[NC][8], dot[1] = {0.0f};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        in.res[c].widen(u[c]);
        in.dn[c].widen(e[c]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (p.y) u[c][j] = __builtin_fmaf(g[c][j] * k[c][j], v[c][j], u[c][j]);
          u[c][j] *= in.r_h;
          sum_next[c][j] = __builtin_fmaf(e[c][j], u[c][j], sum_next[c][j]);
          e[c][j] *= w_next[c][j];
          dot[0] = __builtin_fmaf(e[c][j], u[c][j], dot[0]);
        }
      }
      row_sum<L>(dot, part[turn ^= 1], lane);
      const float mean = dot[0] * inv;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) d[c][j] = __builtin_fmaf(in.r_h, __builtin_fmaf(-mean, u[c][j], e[c][j]), d[c][j]);
    }
    if (p.d_res)
#pragma unroll
      for (int c = 0; c < NC; ++c) R::store(static_cast<Held*>(p.d_res) + t * columns, columns, lane, c, d[c]);
    if (!p.block) continue;
    // d becomes q; dot: of q and v (an element's gate), else of k d and v
    float dot[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sum_block[c][j] = __builtin_fmaf(element || token ? g[c][j] * d[c][j] : d[c][j], v[c][j], sum_block[c][j]);
      if (element) {
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          e[j] = k[c][j] * d[c][j] * v[c][j];
          d[c][j] *= k[c][j] * g[c][j];
          dot[0] = __builtin_fmaf(d[c][j], v[c][j], dot[0]);
        }
        if (p.d_gate) {
          if (p.wide_gate)
            Row<F32, L, VEC>::store(static_cast<float*>(p.d_gate) + t * columns, columns, lane, c, e);
          else
            R::store(static_cast<Held*>(p.d_gate) + t * columns, columns, lane, c, e);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          d[c][j] *= k[c][j];
          dot[0] = __builtin_fmaf(d[c][j], v[c][j], dot[0]);
          d[c][j] *= in.gate;
        }
      }
    }
    if (p.post || (token && p.d_gate)) row_sum<L>(dot, part[turn ^= 1], lane);
    if (token && p.d_gate && lane == 0) {
      if (p.wide_gate)
        static_cast<float*>(p.d_gate)[t] = dot[0];
      else
        static_cast<Held*>(p.d_gate)[t] = T::held(dot[0]);
    }
    if (p.d_y) {
      const float mean = dot[0] * inv * in.gate;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (p.post)  // (without, an infinite y leaves its gradient as it is)
#pragma unroll
          for (int j = 0; j < 8; ++j) d[c][j] = in.r_y * __builtin_fmaf(-mean, v[c][j], d[c][j]);
        R::store(static_cast<Held*>(p.d_y) + t * columns, columns, lane, c, d[c]);
      }
    }
  }
  float* sums = p.sums + slot * 2 * columns;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (p.sum_next) Row<F32, L, VEC>::store(sums, columns, lane, c, sum_next[c]);
    if (p.sum_block) Row<F32, L, VEC>::store(sums + columns, columns, lane, c, sum_block[c]);
  }
}

// The slots' sums, 64 columns a workgroup (5.2 us of 512 slots of 4096 columns): d w_next, and d w_post and the channels' d gate from one sum
struct Finish {
  const float* sums;
  int32_t slots, columns;
  float scale;
  const void *w_post, *gate;  // null: 1
  bool wide_next, wide_post, wide_gate;
  void *d_next, *d_post, *d_gate;
};
constexpr int kFinishWaves = 16;
template <typename T>
__global__ __launch_bounds__(64 * kFinishWaves) void finish_kernel(Finish p) {
  __shared__ float part[kFinishWaves][64];
  const bool block = blockIdx.y == 1;
  if (block ? !p.d_post && !p.d_gate : !p.d_next) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
  float sum = 0.0f;
  if (col < p.columns)
#pragma unroll 8
    for (int s = w; s < p.slots; s += kFinishWaves) sum += p.sums[(int64_t(s) * 2 + block) * p.columns + col];
  part[w][lane] = sum;
  __syncthreads();
  if (w != 0 || col >= p.columns) return;
  for (int i = 1; i < kFinishWaves; ++i) sum += part[i][lane];
  auto store = [&](void* to, bool wide, float v) {
    if (wide)
      static_cast<float*>(to)[col] = v;
    else
      static_cast<typename T::Held*>(to)[col] = T::held(v);
  };
  if (!block) return store(p.d_next, p.wide_next, sum);
  sum *= p.scale;
  if (p.d_post) store(p.d_post, p.wide_post, p.gate ? sum * load_one<T>(p.gate, p.wide_gate, col) : sum);
  if (p.d_gate) store(p.d_gate, p.wide_gate, p.w_post ? sum * load_one<T>(p.w_post, p.wide_post, col) : sum);
}

// ---------------------------------------------------------------- host
static int check(const afd_norm_cfg* cfg, int32_t n) {
  if (!cfg || n < 0 || n > kMaxTokens) return AFD_ERR_ARG;
  if (cfg->columns < 1 || cfg->columns > kMaxHidden) return AFD_ERR_SHAPE;
  if (!known_fmt(cfg->fmt) || cfg->gate_kind < AFD_GATE_NONE || cfg->gate_kind > AFD_GATE_ELEMENT) return AFD_ERR_UNSUPPORTED;
  if (!(cfg->eps > 0.0f)) return AFD_ERR_ARG;
  return AFD_OK;
}

// f(lanes, chunks): the lanes that share a row and the chunks of 8 values each of them holds
template <typename F>
static void with_lanes(int columns, F f) {
  using std::integral_constant;
  if (columns <= 512) return f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  if (columns <= 1024) return f(integral_constant<int, 128>{}, integral_constant<int, 1>{});
  if (columns <= 2048) return f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  if (columns <= 4096) return f(integral_constant<int, 512>{}, integral_constant<int, 1>{});
  if (columns <= 8192) return f(integral_constant<int, 1024>{}, integral_constant<int, 1>{});
  return f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
}
// Workgroups of the gradient's launch: two a CU, which are the 16 wavefronts that the registers let a CU hold at 2049 to 4096
// columns of 16-bit values, where the number was measured. Other widths take it as well: 8 wavefronts a CU at 1025 to 2048 columns and up
// to 512, 4 at 513 to 1024, and above 4096 two workgroups of 16, of which one at a time fits.
static int grid_of(int32_t n, int32_t columns) {
  const int rows = columns <= 512 ? 4 : 1;
  const int64_t need = (int64_t(n) + rows - 1) / rows, most = 2 * 256;
  return static_cast<int>(need < most ? need : most);
}
static int slots_of(int32_t n, int32_t columns) { return grid_of(n, columns) * (columns <= 512 ? 4 : 1); }

static bool aligned_params(const Args& p, int fmt) {
  auto fine = [&](const void* v) { return reinterpret_cast<uintptr_t>(v) % 16 == 0; };
  return p.columns % 8 == 0 && fine(p.w_post) && fine(p.w_next) && (p.gate_kind == AFD_GATE_TOKEN || fine(p.gate)) &&
         aligned_rows(p.y, p.ldy, fmt) && aligned_rows(p.residual, p.ldr, fmt);
}

}  // namespace norm
}  // namespace afd

using namespace afd;

extern "C" int afd_residual_norm(const afd_norm_cfg* cfg, const void* y, int64_t ldy, const void* residual, int64_t ldr,
                                 const void* w_post, const void* gate, const void* w_next, int32_t n, void* h, void* normed,
                                 float* rstd, afd_stream_t stream) {
  const int st = norm::check(cfg, n);
  if (st != AFD_OK) return st;
  if ((y && ldy < cfg->columns) || ldr < cfg->columns) return AFD_ERR_SHAPE;
  if (n == 0) return AFD_OK;
  if (!residual || (!h && !normed) || (!y && h) || (normed && !w_next) || (y && cfg->gate_kind != AFD_GATE_NONE && !gate))
    return AFD_ERR_ARG;
  norm::Args p = {};
  p.y = y;
  p.residual = residual;
  p.ldy = ldy;
  p.ldr = ldr;
  p.w_post = w_post;
  p.gate = gate;
  p.w_next = w_next;
  p.wide_post = cfg->post_f32;
  p.wide_gate = cfg->gate_f32;
  p.wide_next = cfg->next_f32;
  p.gate_kind = cfg->gate_kind;
  p.post = w_post != nullptr;
  p.scale = cfg->scale;
  p.eps = cfg->eps;
  p.n = n;
  p.columns = cfg->columns;
  p.h = h;
  p.normed = normed;
  p.rstd = rstd;
  const bool vec = norm::aligned_params(p, cfg->fmt) && rows::aligned_rows(h, p.columns, cfg->fmt) &&
                   rows::aligned_rows(normed, p.columns, cfg->fmt);
  const bool past = int64_t(n) * p.columns * rows::value_size(cfg->fmt) > rows::kPastBytes;
  return rows::with_fmt(cfg->fmt, [&](auto type) -> int {
    norm::with_lanes(p.columns, [&](auto l, auto nc) {
      using T = decltype(type);
      constexpr int L = decltype(l)::value, NC = decltype(nc)::value;
      const dim3 grid = rows::grid_of_many((int64_t(n) + norm::kRows<L> - 1) / norm::kRows<L>);
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(norm::kThreads<L>), 0, static_cast<hipStream_t>(stream), p);
      };
      if (vec && past)
        go(norm::forward_kernel<T, L, NC, true, true>);
      else if (vec)
        go(norm::forward_kernel<T, L, NC, true, false>);
      else
        go(norm::forward_kernel<T, L, NC, false, false>);
    });
    AFD_CHECK_LAUNCH();
    return AFD_OK;
  });
}

extern "C" int afd_residual_norm_workspace(const afd_norm_cfg* cfg, int32_t n, uint64_t* bytes) {
  const int st = norm::check(cfg, n);
  if (st != AFD_OK) return st;
  if (!bytes) return AFD_ERR_ARG;
  *bytes = uint64_t(norm::slots_of(n, cfg->columns)) * 2 * cfg->columns * 4;
  return AFD_OK;
}

extern "C" int afd_residual_norm_grad(const afd_norm_cfg* cfg, const void* y, int64_t ldy, const void* residual, int64_t ldr,
                                      const void* w_post, const void* gate, const void* w_next, const float* rstd, int32_t n,
                                      const void* dh, const void* dn, void* d_residual, void* d_y, void* d_gate, void* d_post,
                                      void* d_next, void* ws, uint64_t ws_bytes, afd_stream_t stream) {
  uint64_t need;
  const int st = afd_residual_norm_workspace(cfg, n, &need);
  if (st != AFD_OK) return st;
  if ((y && ldy < cfg->columns) || (dn && ldr < cfg->columns)) return AFD_ERR_SHAPE;
  const int kind = y || d_y ? cfg->gate_kind : AFD_GATE_NONE;
  const bool sums = d_next || d_post || (kind == AFD_GATE_CHANNEL && d_gate);
  if (n == 0) return AFD_OK;
  if ((!dh && !dn) || (dn && (!residual || !w_next || !rstd)) || (kind != AFD_GATE_NONE && !gate) || ((y || d_y) && w_post && !rstd) ||
      (d_next && !dn) || (d_post && !(y && w_post)) || (d_gate && (!y || kind == AFD_GATE_NONE)) || (d_y && !y && (w_post || dn)))
    return AFD_ERR_ARG;
  if (sums && (!ws || ws_bytes < need || reinterpret_cast<uintptr_t>(ws) % 16)) return AFD_ERR_WORKSPACE;
  norm::Args p = {};
  p.y = y;
  p.residual = residual;
  p.ldy = ldy;
  p.ldr = ldr;
  p.w_post = w_post;
  p.gate = gate;
  p.w_next = w_next;
  p.wide_post = cfg->post_f32;
  p.wide_gate = cfg->gate_f32;
  p.wide_next = cfg->next_f32;
  p.gate_kind = kind;
  p.post = y && w_post;
  p.scale = cfg->scale;
  p.eps = cfg->eps;
  p.n = n;
  p.columns = cfg->columns;
  p.rstd = const_cast<float*>(rstd);
  p.dh = dh;
  p.dn = dn;
  p.d_res = d_residual;
  p.d_y = d_y;
  p.d_gate = kind == AFD_GATE_CHANNEL ? nullptr : d_gate;
  p.sums = static_cast<float*>(ws);
  p.sum_next = d_next != nullptr;
  p.sum_block = d_post || (kind == AFD_GATE_CHANNEL && d_gate);
  p.block = d_y || d_post || d_gate;
  const int fmt = cfg->fmt;
  bool vec = norm::aligned_params(p, fmt);
  for (const void* v : {dh, dn, static_cast<const void*>(d_residual), static_cast<const void*>(d_y)})
    vec = vec && rows::aligned_rows(v, p.columns, fmt);
  if (kind == AFD_GATE_ELEMENT) vec = vec && reinterpret_cast<uintptr_t>(d_gate) % 16 == 0;
  return rows::with_fmt(fmt, [&](auto type) -> int {
    using T = decltype(type);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    norm::with_lanes(p.columns, [&](auto l, auto nc) {
      constexpr int L = decltype(l)::value, NC = decltype(nc)::value;
      const dim3 grid(static_cast<unsigned>(norm::grid_of(n, p.columns)));
      if (vec)
        hipLaunchKernelGGL((norm::backward_kernel<T, L, NC, true>), grid, dim3(norm::kThreads<L>), 0, s, p);
      else
        hipLaunchKernelGGL((norm::backward_kernel<T, L, NC, false>), grid, dim3(norm::kThreads<L>), 0, s, p);
    });
    AFD_CHECK_LAUNCH();
    if (sums) {
      norm::Finish f = {};
      f.sums = p.sums;
      f.slots = norm::slots_of(n, p.columns);
      f.columns = p.columns;
      f.scale = p.scale;
      f.w_post = w_post;
      f.gate = kind == AFD_GATE_CHANNEL ? gate : nullptr;
      f.wide_next = p.wide_next;
      f.wide_post = p.wide_post;
      f.wide_gate = p.wide_gate;
      f.d_next = d_next;
      f.d_post = d_post;
      f.d_gate = kind == AFD_GATE_CHANNEL ? d_gate : nullptr;
      hipLaunchKernelGGL(norm::finish_kernel<T>, dim3((p.columns + 63) / 64, 2), dim3(64 * norm::kFinishWaves), 0, s, f);
      AFD_CHECK_LAUNCH();
    }
    return AFD_OK;
  });
}
