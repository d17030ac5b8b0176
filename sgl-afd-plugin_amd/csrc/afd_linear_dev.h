// What the dense products with 8-bit weights share (afd_linear.hip: e4m3 with block scales, afd_linear_i8.hip: int8 with a
// scale per token and channel): the fragment images' pieces, the activations as they are read, and which tile
// a workgroup takes.
#pragma once

#include "afd_common.h"
#include "afd_internal.h"

namespace afd {
namespace linear {

constexpr int kPiece = 1024;  // 16 rows x 64 columns of a byte each
constexpr int kMaxDim = 65536;
constexpr int kMaxRows = 1 << 22;
// an x above this is read past the caches (the memory-side cache has 256 MB, shared with codes and weights)
constexpr int64_t kCachedBytes = int64_t(64) << 20;

inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// 16 bf16 values of a row from column k0 (a multiple of 16) on, two a word. VEC: rows are 16-byte aligned and k_in is a
// multiple of 16 (then the 16 are whole or missing). What lies past k_in reads as 0.
struct Half {
  uint32_t u[8];
};
template <bool VEC, bool NT = false>
__device__ __forceinline__ Half load_half(const uint16_t* p, int k_in, int k0) {
  Half r;
  if constexpr (VEC) {
    const uint16_t* src = p + min(k0, k_in - 16);
    const v4i lo = load_words<true, NT>(src), hi = load_words<true, NT>(src + 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.u[i] = k0 < k_in ? lo[i] : 0;
      r.u[4 + i] = k0 < k_in ? hi[i] : 0;
    }
  } else if (k0 + 16 <= k_in) {
    const v4i lo = load_words<false>(p + k0), hi = load_words<false>(p + k0 + 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.u[i] = lo[i];
      r.u[4 + i] = hi[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = k0 + 2 * i;
      const uint32_t lo = p[min(k, k_in - 1)], hi = p[min(k + 1, k_in - 1)];
      r.u[i] = (k < k_in ? lo : 0u) | (k + 1 < k_in ? hi << 16 : 0u);
    }
  }
  return r;
}
// A wavefront's share of an activation image: 16 rows x one K block, lane l chunks l / 16 of both
// 64-column pieces of row l % 16. p: the row; c: the lane's chunk.
struct Raw {
  Half h[2];
};
template <bool VEC, bool NT = false>
__device__ __forceinline__ Raw load_raw(const uint16_t* p, int k_in, int b, int c) {
  Raw r;
#pragma unroll
  for (int h = 0; h < 2; ++h) r.h[h] = load_half<VEC, NT>(p, k_in, b * 128 + h * 64 + c * 16);
  return r;
}
// bf16(silu(g) u) of a lane's gate and up values
__device__ __forceinline__ Half silu_mul(const Half& g, const Half& u) {
  Half r;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = g.u[i], b = u.u[i];
    r.u[i] = pk_bf16(act_swiglu(__uint_as_float(a << 16), __uint_as_float(b << 16)),
                     act_swiglu(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u)));
  }
  return r;
}
__device__ __forceinline__ Raw silu_mul(const Raw& g, const Raw& u) {
  return {{silu_mul(g.h[0], u.h[0]), silu_mul(g.h[1], u.h[1])}};
}

// ---------------------------------------------------------------- tiles
// Workgroup b runs on XCD b % 8, each with its own L2. Where there are many row tiles an XCD takes a
// contiguous eighth of them with all the columns, so that x is read by one L2 and the weights by all; else an eighth
// of the columns with all the rows. Inside, 8 tiles of the long side at a time, the other side
// running behind it: the 32 workgroups of an XCD work on about 8 x 4 tiles and share their operands 4 and 8 ways.
constexpr int kSplitRows = 16;
struct TileAt {
  int mt, nt;
};
__host__ __device__ inline TileAt tile_at(unsigned block, int mts, int nts) {
  const bool rows = mts >= kSplitRows;
  const int major = rows ? mts : nts, minor = rows ? nts : mts;
  const int xcd = block & 7, lo = static_cast<int>(int64_t(major) * xcd / 8);
  const int here = static_cast<int>(int64_t(major) * (xcd + 1) / 8) - lo;
  const int64_t i = block >> 3;
  if (i >= int64_t(here) * minor) return {-1, -1};
  const int full = here / 8;
  int rb = static_cast<int>(i / (8 * minor)), wide = 8;
  if (rb >= full) {
    rb = full;
    wide = here - 8 * full;
  }
  const int j = static_cast<int>(i - int64_t(rb) * 8 * minor);
  const int a = lo + rb * 8 + j % wide, b = j / wide;
  return rows ? TileAt{a, b} : TileAt{b, a};
}
// workgroups that cover every tile
inline int64_t tile_grid(int64_t mts, int64_t nts) {
  return mts >= kSplitRows ? round_up(mts, 8) * nts : round_up(nts, 8) * mts;
}

// Launches the layout of codes [n_out][ld] into an image (load time).
int launch_pack(const uint8_t* codes, int64_t ld, int32_t n_out, int32_t k_in, uint8_t* image, hipStream_t stream);
int check_dims(int32_t n_out, int32_t k_in);

}  // namespace linear
}  // namespace afd
