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

// Eight values as they are held, and in fp32
template <typename T>
struct Raw8 {
  static constexpr int kWords = 8 * sizeof(typename T::Held) / 16;
  v4i w[kWords];
  __device__ __forceinline__ void widen(float (&v)[8]) const {
    if constexpr (sizeof(typename T::Held) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __int_as_float(w[i / 4][i % 4]);
    } else if constexpr (std::is_same<T, Bf16>::value) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(static_cast<uint32_t>(w[0][i]) << 16);
        v[2 * i + 1] = __uint_as_float(static_cast<uint32_t>(w[0][i]) & 0xffff0000u);
      }
    } else {
      const v8h h = __builtin_bit_cast(v8h, w[0]);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(h[i]);
    }
  }
  __device__ __forceinline__ void narrow(const float (&v)[8]) {
    if constexpr (sizeof(typename T::Held) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i / 4][i % 4] = __float_as_int(v[i]);
    } else if constexpr (std::is_same<T, Bf16>::value) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[0][i] = static_cast<int>(pk_bf16(v[2 * i], v[2 * i + 1]));
    } else {
      v8h h;
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = static_cast<_Float16>(v[i]);
      w[0] = __builtin_bit_cast(v4i, h);
    }
  }
};

// A row of `columns` values shared by LANES lanes, lane l's chunk c: eight neighbouring values from (c LANES + l) 8 on. VEC: the
// row is 16-byte aligned and its length a multiple of 8; else its whole chunks are read and written at the alignment they
// have, and the last one value by value. Either way a lane holds the same values, so results do not depend on
// it. What lies past the end reads as 0 and is not written. NT: past the caches (aligned rows).
template <typename T, int LANES, bool VEC>
struct Row {
  using Held = typename T::Held;
  using Raw = Raw8<T>;
  static __device__ __forceinline__ int column(int lane, int c) { return (c * LANES + lane) * 8; }
  template <bool NT = false>
  static __device__ __forceinline__ Raw fetch(const Held* p, int columns, int lane, int c) {
    Raw r = {};
    const int at = column(lane, c);
    if (VEC ? at < columns : at + 8 <= columns) {
#pragma unroll
      for (int i = 0; i < Raw::kWords; ++i) r.w[i] = load_words<VEC, NT>(reinterpret_cast<const char*>(p + at) + 16 * i);
    } else if (!VEC && at < columns) {
      typedef Held v8x __attribute__((ext_vector_type(8)));
      v8x h = {};
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (at + j < columns) h[j] = p[at + j];
      r = __builtin_bit_cast(Raw, h);
    }
    return r;
  }
  static __device__ __forceinline__ void load(const Held* p, int columns, int lane, int c, float (&v)[8]) {
    fetch(p, columns, lane, c).widen(v);
  }
  template <bool NT = false>
  static __device__ __forceinline__ void store(Held* p, int columns, int lane, int c, const float (&v)[8]) {
    const int at = column(lane, c);
    if (VEC ? at < columns : at + 8 <= columns) {
      Raw r;
      r.narrow(v);
#pragma unroll
      for (int i = 0; i < Raw::kWords; ++i) store_words<VEC, NT>(reinterpret_cast<char*>(p + at) + 16 * i, r.w[i]);
    } else if (!VEC && at < columns) {
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (at + j < columns) p[at + j] = T::held(v[j]);
    }
  }
};

// The sums of v over the wavefront, in every lane; one order of additions
template <int N>
__device__ __forceinline__ void wave_sum(float (&v)[N]) {
  // within a row of 16 lanes by cross-lane operands, then across rows and halves by swaps
  auto dpp = [&](auto ctrl) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v[i]), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  dpp(std::integral_constant<int, 0xb1>{});   // lanes 1 0 3 2 of four
  dpp(std::integral_constant<int, 0x4e>{});   // lanes 2 3 0 1 of four
  dpp(std::integral_constant<int, 0x141>{});  // the half row reversed
  dpp(std::integral_constant<int, 0x140>{});  // the row reversed
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t u = __float_as_uint(v[i]);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float s = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const uint32_t t = __float_as_uint(s);
    const auto q = __builtin_amdgcn_permlane32_swap(t, t, false, false);
    v[i] = __uint_as_float(q[0]) + __uint_as_float(q[1]);
  }
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

// Results of more bytes go past the caches (L2 has 32 MB, the memory-side cache 256 for inputs and results). Measured for the
// norms (afd_norm.hip); the sorted rows take the same number, of all pairs' rows, as those that are here are not known on the
// host (afd_sort.hip)
constexpr int64_t kPastBytes = int64_t(48) << 20;
// Workgroups in two dimensions (a dimension's threads are counted in 32 bits), and their number there
inline dim3 grid_of_many(int64_t blocks) {
  const int64_t row = int64_t(1) << 20;
  return blocks <= row ? dim3(static_cast<unsigned>(blocks)) : dim3(static_cast<unsigned>(row), static_cast<unsigned>((blocks + row - 1) / row));
}
__device__ __forceinline__ int64_t block_of_many() { return int64_t(blockIdx.y) * gridDim.x + blockIdx.x; }

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
