// A dense product with FP8-e4m3 weights that carry one fp32 scale per 128x128 block, on activations
// quantized to e4m3 with one fp32 scale per 1x128 (the block-FP8 format of the experts), on gfx950 MFMA:
//
//   y[t, o] = bf16( sum_kb  sx[t, kb] sw[o / 128, kb]  sum_{k in block kb} qx[t, k] qw[o, k] )
//   sx = max(amax_kb |x|, 1e-10) / 448,  qx = e4m3(x / sx)  (both quotients in fp32)
//
// Any n_out and k_in: both operands live in fragment images padded to 16 rows and 128 columns,
// [rows / 16][K / 64] pieces of 1 KiB, a piece's 16-byte chunk c (of 4) of row r at byte 256 c + 16 r. A
// piece is one contiguous wide load, whether a wavefront takes it straight into registers (lane l
// then holds chunk l / 16 of row l % 16: an operand of the 16-row MFMA) or copies it to LDS, where 16 consecutive
// rows of a chunk are 256 bytes, all banks once. Which K a lane's bytes stand for does not matter as
// long as both operands agree. Padding codes are 0; padding rows are never stored.
//
// The MFMA of e4m3 codes adds the products of 8 columns at a time, each cut towards zero at 2^-13 of the largest one's
// power of two, and these sums in fp32 (measured with single products beside a pair that cancels). Over N(0, 1) rows and
// weights 1.2% of the bf16 results are a neighbour of the exact result's rounding, where fp32 products leave 0.1%; the
// distance to 64 bits is the same (1.66e-3 root mean square, all of it bf16's).
// Every block's MFMA sum starts from 0 and is folded into the result with its scale sx sw by one fp32
// fused multiply-add. Scales may be 0, tiny or huge: where a product of two scales is no normal float, the results that it
// belongs to are made again in 64 bits (see odd_scale). A row of x with an infinity or a NaN in a block gets
// the scale NaN, which makes that row of y NaN and no other.
#include "afd_common.h"
#include "afd_gemm_dev.h"
#include "afd_internal.h"

namespace afd {
namespace linear {

constexpr int kPiece = 1024;  // 16 rows x 64 columns of e4m3
constexpr int kMaxDim = 65536;
constexpr int kMaxRows = 1 << 22;
// the activation scales are [K / 128][rows rounded up to kScaleRows]
constexpr int kScaleRows = 256;
// an x above this is read past the caches (the memory-side cache has 256 MB, shared with codes and weights)
constexpr int64_t kCachedBytes = int64_t(64) << 20;

inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

struct Args {
  const uint8_t* a;  // activation image [rows16][kt]
  const float* as;   // [kb][a_rows]
  const uint8_t* b;  // weight image [n_out / 16][kt]
  const float* bs;   // [n_out / 128][kb]
  uint16_t* y;
  int64_t ldy;
  int32_t n, n_out, kb;  // kb: K blocks of 128
  int32_t a_rows;
  bool wide;  // rows of y take 16-byte stores
};

__device__ __forceinline__ v8i join(v4i lo, v4i hi) {
  return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// ---------------------------------------------------------------- activations
// A wavefront's share of an activation image: 16 rows x one K block, lane l chunks l / 16 of both
// 64-column pieces of row l % 16. Raw: those 2 x 16 bf16 values, two a word.
struct Raw {
  uint32_t u[2][8];
};
// VEC: rows take 16-byte loads and k_in is a multiple of 16 (then a chunk is whole or missing). p: the
// row; c: the lane's chunk. What lies past k_in reads as 0.
template <bool VEC, bool NT = false>
__device__ __forceinline__ Raw load_raw(const uint16_t* p, int k_in, int b, int c) {
  Raw r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int k0 = b * 128 + h * 64 + c * 16;
    if constexpr (VEC) {
      const v4i* src = reinterpret_cast<const v4i*>(p + min(k0, k_in - 16));
      const v4i lo = NT ? __builtin_nontemporal_load(src) : src[0], hi = NT ? __builtin_nontemporal_load(src + 1) : src[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r.u[h][i] = k0 < k_in ? lo[i] : 0;
        r.u[h][4 + i] = k0 < k_in ? hi[i] : 0;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = k0 + 2 * i;
        const uint32_t lo = p[min(k, k_in - 1)], hi = p[min(k + 1, k_in - 1)];
        r.u[h][i] = (k < k_in ? lo : 0u) | (k + 1 < k_in ? hi << 16 : 0u);
      }
    }
  }
  return r;
}
// e4m3 codes of both pieces' chunks, and the row's scale of the K block (NaN of a row that is not finite)
__device__ __forceinline__ float quantize(const Raw& r, v4i (&q)[2]) {
  // the largest magnitude's bits, two columns at a time: infinities and NaN above every number
  typedef uint16_t v2u __attribute__((ext_vector_type(2)));
  v2u most = {0, 0};
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      most = __builtin_elementwise_max(most, __builtin_bit_cast(v2u, r.u[h][i] & 0x7fff7fffu));
  uint32_t top = uint32_t(max(most[0], most[1])) << 16;
  const auto r0 = __builtin_amdgcn_permlane16_swap(top, top, false, false);
  top = max(r0[0], r0[1]);
  const auto r1 = __builtin_amdgcn_permlane32_swap(top, top, false, false);
  top = max(r1[0], r1[1]);
  const bool finite = top < 0x7f800000u;
  const float sc = fmaxf(__uint_as_float(finite ? top : 0u), kFp8Eps) / kE4m3Max;
  const float rsc = 1.0f / sc;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t w = finite ? r.u[h][2 * i + j] : 0u;
        v[2 * j] = div_by(__uint_as_float(w << 16), sc, rsc);
        v[2 * j + 1] = div_by(__uint_as_float(w & 0xffff0000u), sc, rsc);
      }
      // quotients of a row's block stay below 448 (1 + 2^-23)
      q[h][i] = static_cast<int>(pk4_e4m3_near(v[0], v[1], v[2], v[3]));
    }
  return finite ? sc : __builtin_nanf("");
}

// bf16(silu(g) u) of a lane's gate and up values
__device__ __forceinline__ Raw silu_mul(const Raw& g, const Raw& u) {
  Raw r;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t a = g.u[h][i], b = u.u[h][i];
      r.u[h][i] = pk_bf16(act_swiglu(__uint_as_float(a << 16), __uint_as_float(b << 16)),
                          act_swiglu(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u)));
    }
  return r;
}

// One wavefront an item, one pass: bound by its bytes where x is large (16384 x 4096, 201 MB in all: 35 us, 5.7 TB/s).
// NT: non-temporal reads, for an x that no cache holds anyway.
// SILU: x's rows are [gate | up] of 2 k_in columns and what is quantized is bf16(silu(gate) up), which then
// never is in memory (the product of 16384 x 1536 x 4096 with it 134 us, 157 in two launches; 48 rows 9.1 against 9.9).
template <bool VEC, bool NT, bool SILU>
__global__ __launch_bounds__(256) void quant_kernel(const uint16_t* __restrict__ x, int64_t ldx, int n, int k_in,
                                                    uint8_t* __restrict__ q, float* __restrict__ s, int kb,
                                                    int a_rows) {
  const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (item >= ((int64_t(n) + 15) / 16) * kb) return;
  const int64_t r16 = item / kb;
  const int b = static_cast<int>(item % kb), lane = threadIdx.x & 63;
  const int64_t row = min(r16 * 16 + (lane & 15), int64_t(n) - 1);  // past the end: the last again
  v4i code[2];
  const uint16_t* p = x + row * ldx;
  Raw raw = load_raw<VEC, NT>(p, k_in, b, lane >> 4);
  if constexpr (SILU) raw = silu_mul(raw, load_raw<VEC, NT>(p + k_in, k_in, b, lane >> 4));
  const float sc = quantize(raw, code);
#pragma unroll
  for (int h = 0; h < 2; ++h)
    *reinterpret_cast<v4i*>(q + (r16 * (2 * kb) + 2 * b + h) * kPiece + lane * 16) = code[h];
  if (lane < 16) s[int64_t(b) * a_rows + r16 * 16 + lane] = sc;
}

// ---------------------------------------------------------------- scales whose product leaves the floats
// sx is between 1e-10 / 448 > 2^-43 and the largest bf16 / 448 < 2^120, so sx sw is a normal float for every x if sw is 0 or
// within 2^-83 .. 2^8. The kernels look at their weight scales, which are scalars, as they pass (a few scalar instructions a
// K block: 48 x 2048 x 4096 6.4 -> 6.6 us, 300 x 2000 x 1111 8.9 -> 9.2, 2900 x 4096 x 4096 46.6 -> 47.4, one row and 16384
// within the noise); where one lies outside, they look at the products themselves, and where one of those
// is no normal float the results are folded again in 64 bits: every sum and product is then in range (all of 16384 x 4096 x
// 4096 so: 1.6 ms for 0.27).
__device__ __forceinline__ bool odd_scale(float s) {
  const uint32_t u = __float_as_uint(s) & 0x7fffffffu;
  constexpr uint32_t kLow = (127u - 83u) << 23, kHigh = (127u + 8u) << 23, kInf = 0x7f800000u;
  // other than 0 and below infinity (which, as NaN, stays itself in any arithmetic), and not within the two; no branches
  return (u - 1 < kInf - 1) & (u - kLow > kHigh - kLow);
}
// Whether sx sw, of numbers other than 0, is no normal float
__device__ __forceinline__ bool odd_product(float sx, float sw) {
  const float s = fabsf(sx * sw);
  return odd_scale(sw) && sx == sx && !(s >= 0x1p-126f && s < __builtin_huge_valf());
}
// 16 outputs of 16 rows, as the MFMA gives them. fetch(b, q): K block b's activation fragment and (returned) its scale
template <typename F>
__device__ __forceinline__ v4f fold_f64(const Args& p, int64_t o16, int lane, F fetch) {
  const uint8_t* bw = p.b + o16 * (2 * p.kb) * kPiece + lane * 16;
  const float* sw = p.bs + o16 / 8 * p.kb;
  double acc[4] = {};
#pragma unroll 1
  for (int b = 0; b < p.kb; ++b) {
    v8i q;
    const float sx = fetch(b, q);
    const v8i fw = join(*reinterpret_cast<const v4i*>(bw + int64_t(2 * b) * kPiece),
                        *reinterpret_cast<const v4i*>(bw + int64_t(2 * b + 1) * kPiece));
    const v4f sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw, q, v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0 /*e4m3*/,
                                                                     0 /*e4m3*/, 0, 0, 0, 0);
    const double s = double(sx) * sw[b];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += sum[i] * s;
  }
  return v4f{static_cast<float>(acc[0]), static_cast<float>(acc[1]), static_cast<float>(acc[2]), static_cast<float>(acc[3])};
}
// K block b of row group r16 from the image
__device__ __forceinline__ float image_fragment(const Args& p, int64_t r16, int b, int lane, v8i& q) {
  const uint8_t* ax = p.a + (r16 * (2 * p.kb) + 2 * b) * kPiece + lane * 16;
  q = join(*reinterpret_cast<const v4i*>(ax), *reinterpret_cast<const v4i*>(ax + kPiece));
  return p.as[int64_t(b) * p.a_rows + r16 * 16 + (lane & 15)];
}

// ---------------------------------------------------------------- weights (load time)
__global__ __launch_bounds__(256) void pack_kernel(const uint8_t* __restrict__ w, int64_t ld, int n_out, int k_in,
                                                   int kb, uint8_t* __restrict__ out, int64_t pieces) {
  for (int64_t at = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); at < pieces; at += int64_t(gridDim.x) * 4) {
    const int lane = threadIdx.x & 63;
    const int64_t row = at / (2 * kb) * 16 + (lane & 15);
    const int k0 = static_cast<int>(at % (2 * kb)) * 64 + (lane >> 4) * 16;
    uint32_t d[4] = {};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t byte = row < n_out && k0 + i < k_in ? w[row * ld + k0 + i] : 0u;
      d[i / 4] |= byte << (8 * (i % 4));
    }
    *reinterpret_cast<v4i*>(out + at * kPiece + lane * 16) =
        v4i{static_cast<int>(d[0]), static_cast<int>(d[1]), static_cast<int>(d[2]), static_cast<int>(d[3])};
  }
}

// ---------------------------------------------------------------- few rows
// Calls of few rows are bound by reading the weights once and by latency. A workgroup owns 16 outputs over
// the whole K and 16 MT rows, its wavefronts every kRowWaves-th K block each: the weights straight into registers
// (non-temporal, DEPTH blocks ahead), the activations from the image likewise; the wavefronts' sums
// meet in LDS, in their order. 16 outputs a workgroup because 4096 of them then are one workgroup a CU with all
// of its weights on their way at once: 1 x 4096 x 4096 takes 5.8 us in a graph (16.8 MB), where a launch that does
// nothing takes 1.6; 48 x 2048 x 4096 8.8 us with its quantization (traced 6.6 and 3.3).
// FUSED: no launch before it. The workgroup quantizes its rows into LDS while its first weights are on
// their way (16 rows' K blocks a wavefront at a time, whichever rows they are of): n K elements, which every
// workgroup does again, so only where they are few and fit kFusedBytes. SILU: as the quantization's.
constexpr int kRowWaves = 8;
constexpr int kFusedBytes = 32768;

struct RowsIn {
  const uint16_t* x;  // FUSED
  int64_t ldx;
  int k_in;
};

template <int MT, bool FUSED, bool VEC, bool SILU>
__global__ __launch_bounds__(64 * kRowWaves) void rows_kernel(Args p, RowsIn in) {
  constexpr int kDepth = FUSED || MT <= 2 ? 4 : MT == 3 ? 3 : 2;
  constexpr int kPart = kRowWaves * MT * 64 * 16;
  constexpr int kCodes = FUSED ? kFusedBytes : 0;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kCodes > kPart ? kCodes : kPart];
  __shared__ float scales[FUSED ? kFusedBytes / 128 : 1];
  __shared__ bool odd_waves[kRowWaves];
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int o16 = blockIdx.x, g0 = blockIdx.y * MT;
  const int kt = 2 * p.kb, last = p.kb - 1;
  const int r16_last = (p.n + 15) / 16 - 1;
  v4f acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const uint8_t* bw = p.b + int64_t(o16) * kt * kPiece + lane * 16;
  const float* sw = p.bs + int64_t(o16 / 8) * p.kb;
  // what a K block needs; blocks past the end read the last one and are not added
  struct Block {
    v4i w[2];
    float s_w;
    v4i x[FUSED ? 1 : MT][2];
    float s_x[FUSED ? 1 : MT];
  };
  auto fetch = [&](int b) {
    Block k;
    const int c = min(b, last);
    k.w[0] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(bw + int64_t(2 * c) * kPiece));
    k.w[1] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(bw + int64_t(2 * c + 1) * kPiece));
    k.s_w = sw[c];
    if constexpr (!FUSED) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int64_t r16 = min(g0 + m, r16_last);
        const uint8_t* ax = p.a + (r16 * kt + 2 * c) * kPiece + lane * 16;
        k.x[m][0] = *reinterpret_cast<const v4i*>(ax);
        k.x[m][1] = *reinterpret_cast<const v4i*>(ax + kPiece);
        k.s_x[m] = p.as[int64_t(c) * p.a_rows + r16 * 16 + (lane & 15)];
      }
    }
    return k;
  };
  Block ring[kDepth];
#pragma unroll
  for (int d = 0; d < kDepth; ++d) ring[d] = fetch(w + d * kRowWaves);
  // FUSED: chunk c of half h of K block b of row r at ((2 b + h) 4 + c) 16 n + 16 r
  if constexpr (FUSED) {
    constexpr int kUp = SILU ? 2 : 4;  // items on their way at once
    const int items = p.n * p.kb, c = lane >> 4;
    for (int at = w * 16; at < items; at += kUp * kRowWaves * 16) {
      Raw raw[kUp], up[SILU ? kUp : 1];
      int r[kUp], b[kUp];
#pragma unroll
      for (int u = 0; u < kUp; ++u) {
        const int it = min(at + u * kRowWaves * 16 + (lane & 15), items - 1);
        r[u] = it / p.kb;
        b[u] = it - r[u] * p.kb;
        const uint16_t* x = in.x + r[u] * in.ldx;
        raw[u] = load_raw<VEC>(x, in.k_in, b[u], c);
        if constexpr (SILU) up[u] = load_raw<VEC>(x + in.k_in, in.k_in, b[u], c);
      }
#pragma unroll
      for (int u = 0; u < kUp; ++u) {
        if (u > 0 && at + u * kRowWaves * 16 >= items) break;
        v4i q[2];
        if constexpr (SILU) raw[u] = silu_mul(raw[u], up[u]);
        const float sc = quantize(raw[u], q);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<v4i*>(lds + (((2 * b[u] + h) * 4 + c) * p.n + r[u]) * 16) = q[h];
        scales[b[u] * p.n + r[u]] = sc;
      }
    }
    __syncthreads();
  }
  bool odd = false;
  for (int b0 = w; b0 <= last; b0 += kDepth * kRowWaves) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int b = b0 + d * kRowWaves;
      if (b > last) break;
      const Block k = ring[d];
      odd |= odd_scale(k.s_w);
      ring[d] = fetch(b + kDepth * kRowWaves);
      const v8i fw = join(k.w[0], k.w[1]);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        v4i q[2];
        float s;
        if constexpr (FUSED) {
          const int r = min(m * 16 + (lane & 15), p.n - 1);
          q[0] = *reinterpret_cast<const v4i*>(lds + ((8 * b + (lane >> 4)) * p.n + r) * 16);
          q[1] = *reinterpret_cast<const v4i*>(lds + ((8 * b + 4 + (lane >> 4)) * p.n + r) * 16);
          s = scales[b * p.n + r];
        } else {
          q[0] = k.x[m][0];
          q[1] = k.x[m][1];
          s = k.s_x[m];
        }
        s *= k.s_w;
        const v4f sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            fw, join(q[0], q[1]), v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0 /*e4m3*/, 0 /*e4m3*/, 0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][i] = __builtin_fmaf(sum[i], s, acc[m][i]);
      }
    }
  }
  if constexpr (FUSED) __syncthreads();  // the codes are read: the sums take their place
  v4f* part = reinterpret_cast<v4f*>(lds);
#pragma unroll
  for (int m = 0; m < MT; ++m) part[(w * MT + m) * 64 + lane] = acc[m];
  odd_waves[w] = odd;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRowWaves; ++i) odd |= odd_waves[i];
  // lane l: row l % 16 of x, outputs 4 (l / 16) .. + 3
  for (int m = w; m < MT; m += kRowWaves) {
    v4f y = part[m * 64 + lane];
    for (int i = 1; i < kRowWaves; ++i) y += part[(i * MT + m) * 64 + lane];
    if (odd) {
      const int r = min(m * 16 + (lane & 15), p.n - 1), r16 = min(g0 + m, r16_last);
      bool again = false;
      for (int b = 0; b <= last; ++b)
        again = again || odd_product(FUSED ? scales[b * p.n + r] : p.as[int64_t(b) * p.a_rows + r16 * 16 + (lane & 15)], sw[b]);
      if (__ballot(again))
        y = fold_f64(p, o16, lane, [&](int b, v8i& q) {
          if constexpr (FUSED) {  // the sums have taken the codes' place
            const uint16_t* x = in.x + r * in.ldx;
            Raw raw = load_raw<VEC>(x, in.k_in, b, lane >> 4);
            if constexpr (SILU) raw = silu_mul(raw, load_raw<VEC>(x + in.k_in, in.k_in, b, lane >> 4));
            v4i code[2];
            const float sc = quantize(raw, code);
            q = join(code[0], code[1]);
            return sc;
          } else {
            return image_fragment(p, r16, b, lane, q);
          }
        });
    }
    const int64_t row = int64_t(g0 + m) * 16 + (lane & 15);
    const int o = o16 * 16 + 4 * (lane >> 4);
    if (row >= p.n) continue;
    uint16_t* out = p.y + row * p.ldy + o;
    if (p.wide && o + 4 <= p.n_out) {
      *reinterpret_cast<uint2*>(out) = uint2{pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3])};
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (o + q < p.n_out) out[q] = f32_to_bf16(y[q]);
    }
  }
}

// ---------------------------------------------------------------- tiles
// BM rows of x by BN outputs, WM x WN wavefronts of TI x TJ MFMA tiles of 16x16 each (K 128 in one
// instruction, so a block's sum is one MFMA from 0 and its 4 values a lane are folded at once). A stage
// is one K block of both operands and the rows' scales, copied HBM -> LDS in 1 KiB pieces into S slots.
//
// A wavefront holds its TI activation fragments of a stage in registers and walks the TJ weight fragments, read two
// ahead, in an order kept as written (left alone, the compiler reads all of a stage first and then waits out every
// MFMA in turn: 322 us for 16384 x 4096 x 4096). When the last two are in registers (all of its reads of the
// stage done) it waits for its copies of the next stage and meets the others at the stage's one barrier: the
// next stage is there for all, and this one's slot is free for the copies of stage b + S. The MFMAs of the last two
// weight fragments run while the next stage's first fragments are read.
//
// 16384 x 4096 x 4096 takes 227 to 281 us (1.96 to 2.42 PFLOP/s; the library's product without block scales 230), at
// a clock of 1.4 to 1.7 GHz: power first, and within the cycles (MFMA busy in 65% of them) LDS, whose bytes for a
// 256 x 256 tile take as long as its MFMAs, and the folds' 4 FMAs an MFMA. 128 x 128 a wavefront would read
// a quarter less, but its 256 sums a lane leave no vector registers to fold with.
template <int BM_, int BN_, int WM_, int WN_, int S_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, S = S_;
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int TI = BM / WM / 16, TJ = BN / WN / 16;
  static constexpr int kAPieces = BM / 16 * 2, kBPieces = BN / 16 * 2;
  static constexpr int kAQ = kAPieces / kWaves, kBQ = kBPieces / kWaves;
  static constexpr int kBOff = kAPieces * kPiece, kSOff = kBOff + kBPieces * kPiece;
  static constexpr int kStage = kSOff + BM * 4;
  static constexpr int kLds = S * kStage;
  static constexpr int kCopies = 1 + kAQ + kBQ;  // a wavefront's copies of a stage
  static constexpr int kScaleWaves = BM / 64;  // each copies 64 rows' scales
  static_assert(TI * 16 * WM == BM && TJ * 16 * WN == BN && kAQ * kWaves == kAPieces && kBQ * kWaves == kBPieces, "tile");
  static_assert(TJ % 4 == 0 && BN / WN <= 128 && 128 % (BN / WN) == 0, "one weight scale per wavefront and K block");
  static_assert(kScaleWaves <= kWaves && BM <= kScaleRows && kLds <= 160 * 1024, "LDS");
  static_assert((S & (S - 1)) == 0 && (S - 1) * kCopies < 64, "slots by a mask; vmcnt is a 6-bit counter");
};

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

template <typename T>
__global__ __launch_bounds__(T::kThreads) void tile_kernel(Args p) {
  constexpr int TI = T::TI, TJ = T::TJ;
  __shared__ __attribute__((aligned(16))) uint8_t lds[T::kLds];
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = w / T::WN, wn = w % T::WN;
  const int mts = (p.n + T::BM - 1) / T::BM, nts = (p.n_out + T::BN - 1) / T::BN;
  const TileAt at = tile_at(blockIdx.x, mts, nts);
  if (at.mt < 0) return;
  // (the divisions run in vector registers; what follows from the tile is scalar)
  const int mt = __builtin_amdgcn_readfirstlane(at.mt), nt = __builtin_amdgcn_readfirstlane(at.nt);
  const int kt = 2 * p.kb, last = p.kb - 1;
  const int m0 = mt * T::BM, n0 = nt * T::BN;
  const int r16_last = (p.n + 15) / 16 - 1, o16_last = (p.n_out + 15) / 16 - 1;
  const uint32_t lds_base = __builtin_amdgcn_readfirstlane(lds_offset(lds));
  const uint32_t voff = static_cast<uint32_t>(lane) * 16;

  // this wavefront's pieces of a stage: piece q of an operand is row group q / 2, 64-column half q % 2.
  // Row groups past the end re-read the last one; their results are not stored.
  const uint8_t* a_src[T::kAQ];
  const uint8_t* b_src[T::kBQ];
#pragma unroll
  for (int i = 0; i < T::kAQ; ++i) {
    const int q = w * T::kAQ + i;
    a_src[i] = p.a + (int64_t(min(m0 / 16 + q / 2, r16_last)) * kt + q % 2) * kPiece;
  }
#pragma unroll
  for (int i = 0; i < T::kBQ; ++i) {
    const int q = w * T::kBQ + i;
    b_src[i] = p.b + (int64_t(min(n0 / 16 + q / 2, o16_last)) * kt + q % 2) * kPiece;
  }
  // copy number c of a stage: the scales, then the activation pieces, then the weight pieces
  constexpr int kCopies = T::kCopies, S = T::S;
  const int ws = w % T::kScaleWaves;
  const int s_row = min(m0 + 64 * ws, p.a_rows - 64);  // rows past the end take other rows' scales
  auto copy = [&](int b, auto c_c) {
    constexpr int c = decltype(c_c)::value;
    const uint32_t st = lds_base + static_cast<uint32_t>((b & (S - 1)) * T::kStage);
    const uint32_t off = voff + static_cast<uint32_t>(b) * (2 * kPiece);
    if constexpr (c == 0) {
      // (every wavefront: two may write the same bytes, and the steps stay one block of code)
      lds_dma4(st + T::kSOff + ws * 256, p.as + int64_t(b) * p.a_rows + s_row, lane * 4u);
    } else if constexpr (c <= T::kAQ) {
      lds_dma16(st + (w * T::kAQ + c - 1) * kPiece, a_src[c - 1], off);
    } else {
      constexpr int i = c - 1 - T::kAQ;
      lds_dma16(st + T::kBOff + (w * T::kBQ + i) * kPiece, b_src[i], off);
    }
  };
  auto issue = [&](int b) { static_for<kCopies>([&](auto c) { copy(b, c); }); };

  v4f acc[TI][TJ];
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  const int sw_row = min((n0 + wn * (T::BN / T::WN)) / 128, (p.n_out - 1) / 128);
  const float* sw = p.bs + int64_t(sw_row) * p.kb;
  float s_w = load_uniform(sw);  // of the stage; the next one's is read where no LDS read is in flight
  bool odd = odd_scale(s_w);
  const uint8_t* a_lds = lds + wm * TI * 2 * kPiece + lane * 16;
  const uint8_t* b_lds = lds + T::kBOff + wn * TJ * 2 * kPiece + lane * 16;
  const uint8_t* s_lds = lds + T::kSOff + (wm * TI * 16 + (lane & 15)) * 4;
  v8i fa[TI], fb[4];
  float sx[TI], s[TI];
  auto read = [&](const uint8_t* f) {
    return join(*reinterpret_cast<const v4i*>(f), *reinterpret_cast<const v4i*>(f + kPiece));
  };
  auto read_a = [&](int b, int i) {
    fa[i] = read(a_lds + (b & (S - 1)) * T::kStage + i * 2 * kPiece);
    sx[i] = *reinterpret_cast<const float*>(s_lds + (b & (S - 1)) * T::kStage + i * 64);
  };
  auto read_b = [&](int b, int j) { return read(b_lds + (b & (S - 1)) * T::kStage + j * 2 * kPiece); };

  // An MFMA's result is folded kLate steps after it was issued (its latency is one step of its own and
  // one of the other wavefront's); the last ones of a stage in the next stage's first steps.
  constexpr int kSteps = TI * TJ, kLate = 3, kSums = 4;
  static_assert(kLate <= kSteps && kSteps % kSums == 0 && kLate < kSums, "a sum is folded before its registers take another");
  v4f sum[kSums];
#pragma unroll
  for (int i = 0; i < kSums; ++i) sum[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < TI; ++i) s[i] = 0.0f;
  auto fold = [&](auto m_c) {
    constexpr int m = decltype(m_c)::value, i = m % TI, j = m / TI;
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[i][j][q] = __builtin_fmaf(sum[m % kSums][q], s[i], acc[i][j][q]);
  };

  static_for<S>([&](auto c) { issue(min(static_cast<int>(decltype(c)::value), last)); });
  wait_vmcnt<(S - 1) * kCopies>();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < TI; ++i) read_a(0, i);
  fb[0] = read_b(0, 0);
  fb[1] = read_b(0, 1);
  for (int b = 0; b <= last; ++b) {
    float s_w_next = 0.0f;
    const int ahead = min(b + S, last);  // past the end: the last stage over itself, the same bytes
    static_for<kSteps>([&](auto mc) {
      constexpr int m = decltype(mc)::value, i = m % TI, j = m / TI;
      constexpr int kFree = (TJ - 2) * TI;  // the first step at which the stage's slot is free
      if constexpr (m == kFree) {
        wait_vmcnt_lds<(S - 2) * kCopies>();  // copies land in the order they were issued in
        __syncthreads();
        s_w_next = load_uniform(sw + min(b + 1, last));
      }
      if constexpr (i == 0) {
        if constexpr (j < TJ - 2)
          fb[(j + 2) % 4] = read_b(b, j + 2);
        else
          fb[(j + 2) % 4] = read_b(b + 1, j + 2 - TJ);
      }
      sum[m % kSums] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
          fb[j % 4], fa[i], v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0 /*e4m3*/, 0 /*e4m3*/, 0, 0, 0, 0);
      if constexpr (m >= kLate)
        fold(std::integral_constant<int, m - kLate>{});
      else
        fold(std::integral_constant<int, kSteps + m - kLate>{});
      if constexpr (m == kLate - 1) {
#pragma unroll
        for (int x = 0; x < TI; ++x) s[x] = sx[x] * s_w;
      }
      if constexpr (m >= kFree) {  // the copies of the stage after next, dealt to the steps that are left
        constexpr int kLeft = kSteps - kFree, at = m - kFree;
        constexpr int c0 = kCopies * at / kLeft, c1 = kCopies * (at + 1) / kLeft;
        static_for<c1 - c0>([&](auto c) { copy(ahead, std::integral_constant<int, c0 + decltype(c)::value>{}); });
      }
      if constexpr (j == TJ - 1) read_a(b + 1, i);
      __builtin_amdgcn_sched_barrier(0);
    });
    s_w = s_w_next;
    odd |= odd_scale(s_w);
  }
  static_for<kLate>([&](auto c) { fold(std::integral_constant<int, kSteps - kLate + decltype(c)::value>{}); });
  wait_vmcnt<0>();

  if (odd) {
    bool again = false;
    for (int b = 0; b <= last; ++b)
#pragma unroll 1
      for (int i = 0; i < TI; ++i)
        again = again || odd_product(p.as[int64_t(b) * p.a_rows + min(m0 + (wm * TI + i) * 16 + (lane & 15), p.n - 1)], sw[b]);
    if (__ballot(again)) {
#pragma unroll 1
      for (int ij = 0; ij < TI * TJ; ++ij) {
        const int r16 = m0 / 16 + wm * TI + ij / TJ, o16 = n0 / 16 + wn * TJ + ij % TJ;
        if (r16 > r16_last || o16 > o16_last) continue;
        const v4f y = fold_f64(p, o16, lane, [&](int b, v8i& q) { return image_fragment(p, r16, b, lane, q); });
        const int64_t row = int64_t(r16) * 16 + (lane & 15);
        for (int q = 0; q < 4; ++q)
          if (row < p.n && o16 * 16 + 4 * (lane >> 4) + q < p.n_out)
            p.y[row * p.ldy + o16 * 16 + 4 * (lane >> 4) + q] = f32_to_bf16(y[q]);
      }
      return;
    }
  }

  // lane l holds, of row l % 16 of an activation tile, outputs 4 (l / 16) .. + 3 of each weight tile. Two
  // neighbouring weight tiles trade halves so that a lane holds 8 outputs: lane groups 0 and 2 those of tile
  // j, 1 and 3 of tile j + 1, 64 contiguous bytes of a row from its four lanes.
  const int lg = lane >> 4;
#pragma unroll
  for (int i = 0; i < TI; ++i) {
    const int row = m0 + (wm * TI + i) * 16 + (lane & 15);
#pragma unroll
    for (int j = 0; j < TJ; j += 2) {
      const uint32_t x0 = pk_bf16(acc[i][j][0], acc[i][j][1]), x1 = pk_bf16(acc[i][j][2], acc[i][j][3]);
      const uint32_t y0 = pk_bf16(acc[i][j + 1][0], acc[i][j + 1][1]);
      const uint32_t y1 = pk_bf16(acc[i][j + 1][2], acc[i][j + 1][3]);
      const auto d0 = __builtin_amdgcn_permlane16_swap(x0, y0, false, false);
      const auto d1 = __builtin_amdgcn_permlane16_swap(x1, y1, false, false);
      const v4i chunk = {static_cast<int>(d0[0]), static_cast<int>(d1[0]), static_cast<int>(d0[1]),
                         static_cast<int>(d1[1])};
      const int o = n0 + (wn * TJ + j + (lg & 1)) * 16 + (lg >> 1) * 8;
      if (row >= p.n) continue;
      uint16_t* out = p.y + row * p.ldy + o;
      if (p.wide && o + 8 <= p.n_out) {
        *reinterpret_cast<v4i*>(out) = chunk;
      } else {
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (o + q < p.n_out)
            out[q] = static_cast<uint16_t>(static_cast<uint32_t>(chunk[q / 2]) >> (16 * (q % 2)));
      }
    }
  }
}

// ---------------------------------------------------------------- host
// Tile shapes. With a tile on each of 256 CUs a K block takes 0.35, 0.49, 0.72, 1.16, 1.48 and 1.86 us (4096
// inputs), that is 0.35, 0.25, 0.18, 0.15, 0.12 and 0.12 for every 64 x 64 outputs: the larger the tile, the less of its
// time goes into moving operands, and the fewer of them there are to fill the CUs. The ring is as deep as the
// LDS allows with the fragments' order in mind: small tiles wait for latency, large ones do not.
using T64 = Shape<64, 64, 4, 1, 4>;
using T64x128 = Shape<64, 128, 2, 2, 4>;
using T128 = Shape<128, 128, 2, 2, 4>;
using T256x128 = Shape<256, 128, 4, 2, 2>;
using T192x256 = Shape<192, 256, 2, 4, 2>;
using T256 = Shape<256, 256, 4, 2, 2>;

struct Plan {
  int kb, a_rows;
  int64_t q_bytes, total;
};
static Plan plan(int32_t n, int32_t k_in) {
  Plan p;
  p.kb = (k_in + 127) / 128;
  p.a_rows = static_cast<int>(round_up(n, kScaleRows));
  p.q_bytes = round_up(n, 16) * p.kb * 128;
  p.total = p.q_bytes + int64_t(p.kb) * p.a_rows * 4;
  return p;
}
static int check_dims(int32_t n_out, int32_t k_in) {
  return n_out < 1 || n_out > kMaxDim || k_in < 1 || k_in > kMaxDim ? AFD_ERR_SHAPE : AFD_OK;
}

template <typename T>
static int launch_tiles(const Args& p, hipStream_t s) {
  const int64_t mts = (p.n + T::BM - 1) / T::BM, nts = (p.n_out + T::BN - 1) / T::BN;
  hipLaunchKernelGGL(tile_kernel<T>, dim3(static_cast<unsigned>(tile_grid(mts, nts))), dim3(T::kThreads), 0, s, p);
  AFD_CHECK_LAUNCH();
  return AFD_OK;
}
template <int MT, bool FUSED, bool SILU>
static int launch_rows(const Args& p, const RowsIn& in, bool vec, hipStream_t s) {
  const dim3 grid((p.n_out + 15) / 16, (p.n + 16 * MT - 1) / (16 * MT)), block(64 * kRowWaves);
  if (!FUSED || vec)
    hipLaunchKernelGGL((rows_kernel<MT, FUSED, true, SILU>), grid, block, 0, s, p, in);
  else
    hipLaunchKernelGGL((rows_kernel<MT, FUSED, !FUSED, SILU>), grid, block, 0, s, p, in);
  AFD_CHECK_LAUNCH();
  return AFD_OK;
}
template <bool SILU>
static int launch_fused_rows(const Args& p, const RowsIn& in, bool vec, hipStream_t s) {
  if (p.n <= 16) return launch_rows<1, true, SILU>(p, in, vec, s);
  if (p.n <= 32) return launch_rows<2, true, SILU>(p, in, vec, s);
  return launch_rows<4, true, SILU>(p, in, vec, s);
}

// The shape whose rounds over the CUs take least: rounds x the measured time of one K block (T64 .. T256
// above). At 4096 x 4096, measured best and chosen: 512 rows T64x128 (20.7 us, T128 25.6), 1024 T128 (28.9, T256x128
// 40), 1500 T256x128 (43, T128 46), 2900 T192x256 (57.8, T256 60.3, T256x128 72), 5800 T192x256 (106, T256 114),
// 8192 T256 (136, T192x256 152). Measured at 32 K blocks alone: at one to four a tile's first copies and its epilogue are
// most of its time, which the rule does not know.
enum { kT64, kT64x128, kT128, kT256x128, kT192x256, kT256, kShapes };
static int best_shape(int64_t n, int64_t n_out, int cus) {
  static const int bm[kShapes] = {64, 64, 128, 256, 192, 256}, bn[kShapes] = {64, 128, 128, 128, 256, 256};
  static const int cost[kShapes] = {35, 49, 72, 116, 148, 186};
  int best = 0;
  int64_t least = 0;
  for (int i = 0; i < kShapes; ++i) {
    const int64_t tiles = ((n + bm[i] - 1) / bm[i]) * ((n_out + bn[i] - 1) / bn[i]);
    const int64_t time = (tiles + cus - 1) / cus * cost[i];
    if (i == 0 || time < least) {
      best = i;
      least = time;
    }
  }
  return best;
}

// y = q(x) W^T, or with silu of the activation of x's rows [gate | up]
static int run(const afd_linear_weights* weights, const uint16_t* x, int64_t ldx, int32_t n, bool silu, void* ws,
               uint64_t ws_bytes, uint16_t* y, int64_t ldy, hipStream_t s) {
  if (!weights || n < 0 || n > kMaxRows) return AFD_ERR_ARG;
  const int st = check_dims(weights->n_out, weights->k_in);
  if (st != AFD_OK) return st;
  if (ldx < int64_t(silu ? 2 : 1) * weights->k_in || ldy < weights->n_out) return AFD_ERR_SHAPE;
  if (n == 0) return AFD_OK;
  if (!weights->image || !weights->scales || !x || !ws || !y) return AFD_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(weights->image) % 16) return AFD_ERR_SHAPE;
  const Plan pl = plan(n, weights->k_in);
  if (ws_bytes < static_cast<uint64_t>(pl.total) || reinterpret_cast<uintptr_t>(ws) % 16) return AFD_ERR_WORKSPACE;
  uint8_t* q = static_cast<uint8_t*>(ws);
  float* sx = reinterpret_cast<float*>(q + pl.q_bytes);
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 8 == 0 && weights->k_in % 16 == 0;
  Args p = {};
  p.a = q;
  p.as = sx;
  p.b = static_cast<const uint8_t*>(weights->image);
  p.bs = weights->scales;
  p.y = y;
  p.ldy = ldy;
  p.n = n;
  p.n_out = weights->n_out;
  p.kb = pl.kb;
  p.a_rows = pl.a_rows;
  p.wide = reinterpret_cast<uintptr_t>(y) % 16 == 0 && ldy % 8 == 0;
  const RowsIn in = {x, ldx, weights->k_in};
  // the rows kernel's own quantization is faster up to 32 K elements (4096 x 4096: 4 rows 6.7 against 8.8 us,
  // 16 rows 10.8 against 9.0; 1024 x 1000: 32 rows 6.4 against 7.1, 64 rows 9.5 against 7.4), a third
  // of that where the rows do not take wide loads (300 x 3000: 32 rows 6.7 against 7.3, 64 rows 10.0 against 7.5)
  const int64_t elements = int64_t(n) * pl.kb * 128;
  if (n <= 64 && elements <= (vec ? kFusedBytes : kFusedBytes / 3))
    return silu ? launch_fused_rows<true>(p, in, vec, s) : launch_fused_rows<false>(p, in, vec, s);
  const int64_t items = (int64_t(n) + 15) / 16 * pl.kb;
  const dim3 grid(static_cast<unsigned>((items + 3) / 4));
  // (134 MB of x: 36 us non-temporal, 42 through the caches; 24 MB, which they hold: 9.3 against 8.0)
  const bool nt = int64_t(n) * weights->k_in * (silu ? 4 : 2) > kCachedBytes;
  auto quant = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, x, ldx, n, weights->k_in, q, sx, pl.kb, pl.a_rows);
  };
  auto quant_any = [&](auto silu_c) {
    constexpr bool kSilu = decltype(silu_c)::value;
    if (vec && nt)
      quant(quant_kernel<true, true, kSilu>);
    else if (vec)
      quant(quant_kernel<true, false, kSilu>);
    else
      quant(quant_kernel<false, false, kSilu>);
  };
  if (silu)
    quant_any(std::true_type{});
  else
    quant_any(std::false_type{});
  AFD_CHECK_LAUNCH();
  // up to 64 rows the weights are read once; above, tiles (4096 x 4096: 64 rows 12.8 against 13.5 us, 128
  // rows 14.7 against 13.9)
  if (n <= 16) return launch_rows<1, false, false>(p, in, vec, s);
  if (n <= 32) return launch_rows<2, false, false>(p, in, vec, s);
  if (n <= 48) return launch_rows<3, false, false>(p, in, vec, s);
  if (n <= 64) return launch_rows<4, false, false>(p, in, vec, s);
  switch (best_shape(n, p.n_out, device_cu_count())) {
    case kT64: return launch_tiles<T64>(p, s);
    case kT64x128: return launch_tiles<T64x128>(p, s);
    case kT128: return launch_tiles<T128>(p, s);
    case kT192x256: return launch_tiles<T192x256>(p, s);
    case kT256x128: return launch_tiles<T256x128>(p, s);
    default: return launch_tiles<T256>(p, s);
  }
}

}  // namespace linear
}  // namespace afd

using namespace afd;

extern "C" int afd_linear_layout(int32_t n_out, int32_t k_in, uint64_t* image_bytes) {
  if (!image_bytes) return AFD_ERR_ARG;
  const int st = linear::check_dims(n_out, k_in);
  if (st != AFD_OK) return st;
  *image_bytes = static_cast<uint64_t>(linear::round_up(n_out, 16) * linear::round_up(k_in, 128));
  return AFD_OK;
}

extern "C" int afd_linear_pack(const uint8_t* codes, int64_t ld, int32_t n_out, int32_t k_in, uint8_t* image,
                               afd_stream_t stream) {
  if (!codes || !image) return AFD_ERR_ARG;
  const int st = linear::check_dims(n_out, k_in);
  if (st != AFD_OK) return st;
  if (ld < k_in || reinterpret_cast<uintptr_t>(image) % 16) return AFD_ERR_SHAPE;
  const int kb = (k_in + 127) / 128;
  const int64_t pieces = linear::round_up(n_out, 16) / 16 * 2 * kb;
  const int64_t grid = (pieces + 3) / 4;
  hipLaunchKernelGGL(linear::pack_kernel, dim3(static_cast<unsigned>(grid < 8192 ? grid : 8192)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), codes, ld, n_out, k_in, kb, image, pieces);
  AFD_CHECK_LAUNCH();
  return AFD_OK;
}

extern "C" int afd_linear_workspace(int32_t n, int32_t k_in, uint64_t* bytes) {
  if (!bytes || n < 0 || n > linear::kMaxRows) return AFD_ERR_ARG;
  const int st = linear::check_dims(1, k_in);
  if (st != AFD_OK) return st;
  *bytes = static_cast<uint64_t>(linear::plan(n, k_in).total);
  return AFD_OK;
}

extern "C" int afd_linear(const afd_linear_weights* weights, const uint16_t* x, int64_t ldx, int32_t n, void* ws,
                          uint64_t ws_bytes, uint16_t* y, int64_t ldy, afd_stream_t stream) {
  return linear::run(weights, x, ldx, n, false, ws, ws_bytes, y, ldy, static_cast<hipStream_t>(stream));
}

extern "C" int afd_linear_silu_mul(const afd_linear_weights* weights, const uint16_t* gate_up, int64_t ld, int32_t n,
                                   void* ws, uint64_t ws_bytes, uint16_t* y, int64_t ldy, afd_stream_t stream) {
  return linear::run(weights, gate_up, ld, n, true, ws, ws_bytes, y, ldy, static_cast<hipStream_t>(stream));
}
