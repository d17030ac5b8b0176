// Rows of values in the three formats that training and serving hold them in (enum afd_value_fmt), read and written eight
// values a lane at a time, and sums over the lanes that share a row.
#pragma once

#include "afd_common.h"

namespace afd {
namespace rows {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));

struct F32 {
  using Held = float;
  static __device__ __forceinline__ float wide(float v) { return v; }
  static __device__ __forceinline__ float held(float v) { return v; }
};
struct Bf16 {
  using Held = uint16_t;
  static __device__ __forceinline__ float wide(uint16_t v) { return bf16_to_f32(v); }
  static __device__ __forceinline__ uint16_t held(float v) { return f32_to_bf16(v); }
};
struct F16 {
  using Held = _Float16;
  static __device__ __forceinline__ float wide(_Float16 v) { return static_cast<float>(v); }
  static __device__ __forceinline__ _Float16 held(float v) { return static_cast<_Float16>(v); }
};

// Eight values at p, 16-byte aligned
template <typename T>
__device__ __forceinline__ void load8(const typename T::Held* p, float (&v)[8]) {
  if constexpr (sizeof(typename T::Held) == 4) {
    const v4f lo = reinterpret_cast<const v4f*>(p)[0], hi = reinterpret_cast<const v4f*>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = lo[i];
      v[4 + i] = hi[i];
    }
  } else {
    const v4i raw = *reinterpret_cast<const v4i*>(p);
    if constexpr (std::is_same<T, Bf16>::value) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(static_cast<uint32_t>(raw[i]) << 16);
        v[2 * i + 1] = __uint_as_float(static_cast<uint32_t>(raw[i]) & 0xffff0000u);
      }
    } else {
      const v8h h = __builtin_bit_cast(v8h, raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(h[i]);
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(typename T::Held* p, const float (&v)[8]) {
  if constexpr (sizeof(typename T::Held) == 4) {
    reinterpret_cast<v4f*>(p)[0] = v4f{v[0], v[1], v[2], v[3]};
    reinterpret_cast<v4f*>(p)[1] = v4f{v[4], v[5], v[6], v[7]};
  } else if constexpr (std::is_same<T, Bf16>::value) {
    v4i raw;
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = static_cast<int>(pk_bf16(v[2 * i], v[2 * i + 1]));
    *reinterpret_cast<v4i*>(p) = raw;
  } else {
    v8h h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = static_cast<_Float16>(v[i]);
    *reinterpret_cast<v4i*>(p) = __builtin_bit_cast(v4i, h);
  }
}

// A row of `columns` values shared by LANES lanes, lane l's chunk c (of 8 values). VEC: neighbouring values in 16-byte
// loads (the row is 16-byte aligned, its length a multiple of 8); else values LANES apart, so that a wavefront's lanes still
// touch neighbouring values. What lies past the end reads as 0 and is not written.
template <typename T, int LANES, bool VEC>
struct Row {
  using Held = typename T::Held;
  static __device__ __forceinline__ int column(int lane, int c, int j) {
    return VEC ? (c * LANES + lane) * 8 + j : (c * 8 + j) * LANES + lane;
  }
  static __device__ __forceinline__ void load(const Held* p, int columns, int lane, int c, float (&v)[8]) {
    if constexpr (VEC) {
      const int at = column(lane, c, 0);
      if (at < columns) {
        load8<T>(p + at, v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = column(lane, c, j);
        v[j] = at < columns ? T::wide(p[at]) : 0.0f;
      }
    }
  }
  static __device__ __forceinline__ void store(Held* p, int columns, int lane, int c, const float (&v)[8]) {
    if constexpr (VEC) {
      const int at = column(lane, c, 0);
      if (at < columns) store8<T>(p + at, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = column(lane, c, j);
        if (at < columns) p[at] = T::held(v[j]);
      }
    }
  }
};

// The sums of v over the wavefront, in every lane; one order of additions
template <int N>
__device__ __forceinline__ void wave_sum(float (&v)[N]) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], d);
}
// The sums of v over LANES lanes that share a row. part: LDS of LANES / 64 x N floats, not used again before a barrier
// (callers alternate between two).
template <int LANES, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* part, int lane) {
  wave_sum(v);
  if constexpr (LANES > 64) {
    constexpr int kWaves = LANES / 64;
    const int w = lane >> 6;
    if ((lane & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) part[w * N + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = part[i];
#pragma unroll
      for (int o = 1; o < kWaves; ++o) v[i] += part[o * N + i];
    }
  }
}

inline int value_size(int fmt) { return fmt == AFD_V_F32 ? 4 : 2; }
inline bool known_fmt(int fmt) { return fmt == AFD_V_F32 || fmt == AFD_V_BF16 || fmt == AFD_V_F16; }
// Whether rows at p, `ld` values apart, take 16-byte loads
inline bool aligned_rows(const void* p, int64_t ld, int fmt) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * value_size(fmt) % 16 == 0);
}
// f(F32 / Bf16 / F16)
template <typename F>
int with_fmt(int fmt, F f) {
  if (fmt == AFD_V_F32) return f(F32{});
  if (fmt == AFD_V_BF16) return f(Bf16{});
  return f(F16{});
}

}  // namespace rows
}  // namespace afd
