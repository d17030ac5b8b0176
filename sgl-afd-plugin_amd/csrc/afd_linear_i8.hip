// A dense product with int8 weights that carry one fp32 scale per output channel, on activations quantized to int8 with
// one fp32 scale per token, on gfx950 MFMA:
//
//   y[t, o] = bf16( sx[t] sw[o] sum_k qx[t, k] qw[o, k] )
//   sx = max(amax_k |x|, 1e-10) / 127,  qx = rint(x / sx)  (both quotients in fp32)
//
// The sums are exact: 65536 products of at most 127 x 128 stay below 2^31. So they may be made in any order and cut
// in any way with the same result, and nothing is rounded but the scales' product, the sum as a float, their product
// (each by at most 2^-24 of it) and the result.
//
// Operands live in the fragment images of the e4m3 product (afd_linear.hip): 16 rows x 64 columns = 1 KiB pieces,
// chunk c (of 4) of row r at byte 256 c + 16 r, K padded to 128 with zeros. A piece is an operand of the 16x16x64
// MFMA as it stands.
// A row of x with an infinity or a NaN gets the scale NaN, which makes that row of y NaN and no other.
#include "afd_common.h"
#include "afd_gemm_dev.h"
#include "afd_internal.h"
#include "afd_linear_dev.h"

namespace afd {
namespace linear8 {

using namespace linear;

constexpr float kI8Max = 127.0f;
constexpr float kI8Eps = 1e-10f;

struct Args {
  const uint8_t* a;  // activation image [rows16][kt]
  const float* as;   // [a_rows]
  const uint8_t* b;  // weight image [n_out / 16][kt]
  const float* bs;   // [n_out]
  uint16_t* y;
  int64_t ldy;
  int32_t n, n_out, kb;  // kb: K blocks of 128
};

__device__ __forceinline__ v4i mfma(v4i w, v4i x, v4i c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, c, 0, 0, 0); }

// ---------------------------------------------------------------- activations
// The largest magnitude's bits of a lane's values (infinities and NaN above every number)
__device__ __forceinline__ uint32_t largest(const Half& r) {
  typedef uint16_t v2u __attribute__((ext_vector_type(2)));
  v2u most = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(v2u, r.u[i] & 0x7fff7fffu));
  return uint32_t(max(most[0], most[1])) << 16;
}
// The largest of a row's lanes: those l with the same l % ROWS
template <int ROWS>
__device__ __forceinline__ uint32_t largest_of_row(uint32_t top) {
  if constexpr (ROWS <= 4)
    top = max(top, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0x124 /*row_ror:4*/, 0xf, 0xf, false)));
  if constexpr (ROWS <= 8)
    top = max(top, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0x128 /*row_ror:8*/, 0xf, 0xf, false)));
  const auto r0 = __builtin_amdgcn_permlane16_swap(top, top, false, false);
  top = max(r0[0], r0[1]);
  const auto r1 = __builtin_amdgcn_permlane32_swap(top, top, false, false);
  return max(r1[0], r1[1]);
}
struct RowScale {
  float s, inv;
  bool finite;
  __device__ __forceinline__ explicit RowScale(uint32_t top) {
    finite = top < 0x7f800000u;
    s = fmaxf(__uint_as_float(finite ? top : 0u), kI8Eps) / kI8Max;
    inv = 1.0f / s;
  }
  __device__ __forceinline__ float held() const { return finite ? s : __builtin_nanf(""); }
};
// the code of v in the low byte: 1.5 2^23 + v rounds v to the nearest integer, ties to even, in two's complement
__device__ __forceinline__ uint32_t code_of(float v) { return __float_as_uint(v + 12582912.0f); }
// int8 codes of 16 values; quotients of a row stay below 127 (1 + 2^-23)
__device__ __forceinline__ v4i quantize(const Half& r, const RowScale& sc) {
  v4i q;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t pair[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t w = sc.finite ? r.u[2 * i + j] : 0u;
      const uint32_t lo = code_of(div_by(__uint_as_float(w << 16), sc.s, sc.inv));
      const uint32_t hi = code_of(div_by(__uint_as_float(w & 0xffff0000u), sc.s, sc.inv));
      pair[j] = __builtin_amdgcn_perm(hi, lo, 0x0c0c0400u);
    }
    q[i] = static_cast<int>(__builtin_amdgcn_perm(pair[1], pair[0], 0x05040100u));
  }
  return q;
}

// A workgroup of WAVES wavefronts takes ROWS rows. A wavefront's unit is 16 columns a lane, 1024 / ROWS of its rows', and it
// takes every WAVES-th. D: the units that it holds in registers between the rows' maximum and the codes (x is read once);
// 0: x is read again for the codes, any K. NT: non-temporal reads, for an x that no cache holds anyway.
// SILU: x's rows are [gate | up] of 2 k_in columns and what is quantized is bf16(silu(gate) up).
template <int ROWS, int WAVES, int D, bool VEC, bool NT, bool SILU>
__global__ __launch_bounds__(64 * WAVES) void quant_kernel(const uint16_t* __restrict__ x, int64_t ldx, int n, int k_in,
                                                           uint8_t* __restrict__ q, float* __restrict__ s, int kb) {
  __shared__ uint32_t tops[WAVES][ROWS];
  constexpr int kLanes = 64 / ROWS;  // of a row
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int chunks = 8 * kb, units = (chunks + kLanes - 1) / kLanes;
  const int at = blockIdx.x * ROWS + lane % ROWS;
  const uint16_t* p = x + int64_t(min(at, n - 1)) * ldx;  // past the end: the last row again
  auto fetch = [&](int unit) {
    const int k0 = (unit * kLanes + lane / ROWS) * 16;
    Half raw = load_half<VEC, NT>(p, k_in, k0);
    if constexpr (SILU) raw = silu_mul(raw, load_half<VEC, NT>(p + k_in, k_in, k0));
    return raw;
  };
  constexpr int kHeld = D > 0 ? D : 1;
  Half raw[kHeld];
  uint32_t top = 0;
  if constexpr (D > 0) {
#pragma unroll
    for (int d = 0; d < D; ++d) raw[d] = fetch(min(w + d * WAVES, units - 1));
#pragma unroll
    for (int d = 0; d < D; ++d) top = max(top, largest(raw[d]));
  } else {
    for (int u = w; u < units; u += WAVES) top = max(top, largest(fetch(u)));
  }
  top = largest_of_row<ROWS>(top);
  if (lane < ROWS) tops[w][lane] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WAVES; ++i) top = max(top, tops[i][lane % ROWS]);
  const RowScale sc(top);
  // chunk c of a row lies in piece c / 4, at its row's place
  uint8_t* out = q + int64_t(at / 16) * (2 * kb) * kPiece + at % 16 * 16;
  auto store = [&](int unit, const Half& v) {
    const int c = unit * kLanes + lane / ROWS;
    const v4i code = quantize(v, sc);
    if (c < chunks) *reinterpret_cast<v4i*>(out + int64_t(c / 4) * kPiece + c % 4 * 256) = code;
  };
  if constexpr (D > 0) {
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (w + d * WAVES < units) store(w + d * WAVES, raw[d]);
  } else {
    for (int u = w; u < units; u += WAVES) store(u, fetch(u));
  }
  if (w == 0 && lane < ROWS) s[at] = sc.held();
}

// ---------------------------------------------------------------- results
// sx is between 1e-10 / 127 > 2^-41 and the largest bf16 / 127 < 2^122, so sx sw is a normal float for every x if sw is 0 or
// within 2^-85 .. 2^6. Where a channel's lies outside, its results are made in 64 bits.
__device__ __forceinline__ bool odd_scale(float s) {
  const uint32_t u = __float_as_uint(s) & 0x7fffffffu;
  constexpr uint32_t kLow = (127u - 85u) << 23, kHigh = (127u + 6u) << 23, kInf = 0x7f800000u;
  // other than 0 and below infinity (which, as NaN, stays itself in any arithmetic), and not within the two
  return (u - 1 < kInf - 1) & (u - kLow > kHigh - kLow);
}
__device__ __forceinline__ float scaled(int sum, float sx, float sw, bool odd) {
  if (odd) return static_cast<float>(double(sum) * (double(sx) * double(sw)));
  return static_cast<float>(sum) * (sx * sw);
}

// ---------------------------------------------------------------- few rows
// Calls of few rows are bound by reading the weights once and by latency. A workgroup owns 16 outputs over
// the whole K and 16 MT rows, its wavefronts every kRowWaves-th K block each: the weights straight into registers
// (non-temporal, DEPTH blocks ahead), the activations from the image likewise; the wavefronts' sums
// meet in LDS. FUSED: no launch before it; the workgroup quantizes its rows into LDS while its first weights are on
// their way (16 rows' K blocks a wavefront at a time, whichever rows they are of): n K elements, which every
// workgroup does again, so only where they are few and fit kFusedBytes. SILU: as the quantization's.
constexpr int kRowWaves = 8;
constexpr int kFusedBytes = 32768;
constexpr int kFusedRows = 64;

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
  __shared__ uint32_t tops[FUSED ? kFusedRows : 1];
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int o16 = blockIdx.x, g0 = blockIdx.y * MT;
  const int kt = 2 * p.kb, last = p.kb - 1;
  const int r16_last = (p.n + 15) / 16 - 1;
  v4i acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = v4i{0, 0, 0, 0};
  const uint8_t* bw = p.b + int64_t(o16) * kt * kPiece + lane * 16;
  // what a K block needs; blocks past the end read the last one and are not added
  struct Block {
    v4i w[2];
    v4i x[FUSED ? 1 : MT][2];
  };
  auto fetch = [&](int b) {
    Block k;
    const int c = min(b, last);
    k.w[0] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(bw + int64_t(2 * c) * kPiece));
    k.w[1] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(bw + int64_t(2 * c + 1) * kPiece));
    if constexpr (!FUSED) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint8_t* ax = p.a + (int64_t(min(g0 + m, r16_last)) * kt + 2 * c) * kPiece + lane * 16;
        k.x[m][0] = *reinterpret_cast<const v4i*>(ax);
        k.x[m][1] = *reinterpret_cast<const v4i*>(ax + kPiece);
      }
    }
    return k;
  };
  Block ring[kDepth];
#pragma unroll
  for (int d = 0; d < kDepth; ++d) ring[d] = fetch(w + d * kRowWaves);
  // the scales of a lane's outputs 4 (l / 16) .. + 3, and of its rows
  float sw[4], sx[MT];
#pragma unroll
  for (int q = 0; q < 4; ++q) sw[q] = p.bs[min(o16 * 16 + 4 * (lane >> 4) + q, p.n_out - 1)];
#pragma unroll
  for (int m = 0; m < MT; ++m) sx[m] = FUSED ? 0.0f : p.as[min((g0 + m) * 16 + (lane & 15), p.n - 1)];
  // FUSED: chunk c of half h of K block b of row r at ((2 b + h) 4 + c) 16 n + 16 r
  if constexpr (FUSED) {
    // items: a row's K block, 16 of them a wavefront at a time; at most kFusedBytes / 128 of them
    constexpr int kUp = kFusedBytes / 128 / 16 / kRowWaves;
    const int items = p.n * p.kb, c = lane >> 4;
    Raw raw[kUp];
    int r[kUp], b[kUp];
    if (t < kFusedRows) tops[t] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kUp; ++u) {
      const int it = min((w + u * kRowWaves) * 16 + (lane & 15), items - 1);  // past the end: the last again
      r[u] = it / p.kb;
      b[u] = it - r[u] * p.kb;
      const uint16_t* x = in.x + r[u] * in.ldx;
      if ((w + u * kRowWaves) * 16 >= items) continue;
      raw[u] = load_raw<VEC>(x, in.k_in, b[u], c);
      if constexpr (SILU) raw[u] = silu_mul(raw[u], load_raw<VEC>(x + in.k_in, in.k_in, b[u], c));
    }
#pragma unroll
    for (int u = 0; u < kUp; ++u) {
      if ((w + u * kRowWaves) * 16 >= items) continue;
      atomicMax(&tops[r[u]], largest_of_row<16>(max(largest(raw[u].h[0]), largest(raw[u].h[1]))));
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kUp; ++u) {
      if ((w + u * kRowWaves) * 16 >= items) continue;
      const RowScale sc(tops[r[u]]);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<v4i*>(lds + (((2 * b[u] + h) * 4 + c) * p.n + r[u]) * 16) = quantize(raw[u].h[h], sc);
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m) sx[m] = RowScale(tops[min(m * 16 + (lane & 15), p.n - 1)]).held();
  }
  for (int b0 = w; b0 <= last; b0 += kDepth * kRowWaves) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int b = b0 + d * kRowWaves;
      if (b > last) break;
      const Block k = ring[d];
      ring[d] = fetch(b + kDepth * kRowWaves);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          v4i x;
          if constexpr (FUSED)
            x = *reinterpret_cast<const v4i*>(
                lds + ((8 * b + 4 * h + (lane >> 4)) * p.n + min(m * 16 + (lane & 15), p.n - 1)) * 16);
          else
            x = k.x[m][h];
          acc[m] = mfma(k.w[h], x, acc[m]);
        }
    }
  }
  if constexpr (FUSED) __syncthreads();  // the codes are read: the sums take their place
  v4i* part = reinterpret_cast<v4i*>(lds);
#pragma unroll
  for (int m = 0; m < MT; ++m) part[(w * MT + m) * 64 + lane] = acc[m];
  __syncthreads();
  // lane l: row l % 16 of x, outputs 4 (l / 16) .. + 3
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (w != m) continue;  // MT <= kRowWaves
    v4i sum = part[m * 64 + lane];
    for (int i = 1; i < kRowWaves; ++i) sum += part[(i * MT + m) * 64 + lane];
    const int64_t row = int64_t(g0 + m) * 16 + (lane & 15);
    const int o = o16 * 16 + 4 * (lane >> 4);
    if (row >= p.n) continue;
    float y[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) y[q] = scaled(sum[q], sx[m], sw[q], odd_scale(sw[q]));
    uint16_t* out = p.y + row * p.ldy + o;
    if (o + 4 <= p.n_out) {
      typedef int v2i_any __attribute__((ext_vector_type(2), aligned(2)));
      *reinterpret_cast<v2i_any*>(out) = v2i_any{static_cast<int>(pk_bf16(y[0], y[1])), static_cast<int>(pk_bf16(y[2], y[3]))};
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (o + q < p.n_out) out[q] = f32_to_bf16(y[q]);
    }
  }
}

// ---------------------------------------------------------------- tiles
// BM rows of x by BN outputs, WM x WN x WK wavefronts of TI x TJ MFMA tiles of 16x16 each; the WK groups share the tile and
// take K in turns, their sums meet in LDS at the end. A stage is 64 columns of both operands for each group, copied
// HBM -> LDS in 1 KiB pieces into S slots.
//
// A wavefront holds its TI activation fragments of a stage in registers and walks the TJ weight fragments, read two
// ahead, in an order kept as written. When the last two are in registers (all of its reads of the
// stage done) it waits for its copies of the next stage and meets the others at the stage's one barrier: the
// next stage is there for all, and this one's slot is free for the copies of stage b + S. The MFMAs of the last two
// weight fragments run while the next stage's first fragments are read.
//
// 16384 x 4096 x 4096 takes 204 to 211 us (2.6 to 2.7 POP/s; a library's product without scales 252): in the loop over K 3.2
// POP/s, MFMA busy in 64% of all cycles at 1.95 GHz, and 8 to 10 us a round of tiles for its first copies and its results.
// Operands move at 16 to 18 bytes a cycle and CU, which is what bounds the loop (without copies 196 us for 239, without LDS
// reads 234; deeper rings, cache hints and workgroups that stay resident and start the next tile's copies early change
// nothing or lose). Stages of 64 columns free their slots sooner than of 128 (231 for 241), and wavefronts of 128 x 64
// hold more of what the long side needs than of 64 x 128 (222 for 231).
template <int BM_, int BN_, int WM_, int WN_, int WK_, int S_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, WK = WK_, S = S_;
  static constexpr int kWaves = WM * WN * WK, kThreads = 64 * kWaves;
  static constexpr int TI = BM / WM / 16, TJ = BN / WN / 16;
  static constexpr int kAPieces = BM / 16, kBPieces = BN / 16, kGroup = kAPieces + kBPieces, kPieces = WK * kGroup;
  static constexpr int kStage = kPieces * kPiece;
  static constexpr int kRing = S * kStage, kSums = (WK - 1) * WM * WN * TI * TJ * 1024;
  static constexpr int kLds = kRing > kSums ? kRing : kSums;
  static constexpr int kCopies = (kPieces + kWaves - 1) / kWaves;  // a wavefront's copies of a stage
  static_assert(TI * 16 * WM == BM && TJ * 16 * WN == BN, "tile");
  static constexpr int kRingB = TJ % 4 == 0 ? 4 : 3;  // weight fragments in registers
  static_assert(TJ % kRingB == 0 && TJ % 2 == 0 && kLds <= 160 * 1024, "fragments by their number; pairs of results; LDS");
  static_assert(S >= 2 && (S - 1) * kCopies < 64, "vmcnt is a 6-bit counter");
};

// NT: results are stored past the caches, for rows whose 64-byte pieces are aligned (through L2 the 134 MB of 16384 x 4096 x
// 4096 cost 23 us more: 227 us, with no stores at all 198, so 204; 6000 x 2048 x 3584 57.1 against 54.0; where pieces lie
// across lines it is the other way: 6000 x 2048 x 3500 59.5 against 78.4).
template <typename T, bool NT>
__global__ __launch_bounds__(T::kThreads) __attribute__((amdgpu_waves_per_eu(2))) void tile_kernel(Args p) {
  constexpr int TI = T::TI, TJ = T::TJ, WK = T::WK, kCopies = T::kCopies, S = T::S, kRingB = T::kRingB;
  __shared__ __attribute__((aligned(16))) uint8_t lds[T::kLds];
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wk = w / (T::WM * T::WN), wm = w / T::WN % T::WM, wn = w % T::WN;
  const int mts = (p.n + T::BM - 1) / T::BM, nts = (p.n_out + T::BN - 1) / T::BN;
  const TileAt at = tile_at(blockIdx.x, mts, nts);
  if (at.mt < 0) return;
  // (the divisions run in vector registers; what follows from the tile is scalar)
  const int mt = __builtin_amdgcn_readfirstlane(at.mt), nt = __builtin_amdgcn_readfirstlane(at.nt);
  const int kt = 2 * p.kb, last = (kt + WK - 1) / WK - 1;
  const int m0 = mt * T::BM, n0 = nt * T::BN;
  const int r16_last = (p.n + 15) / 16 - 1, o16_last = (p.n_out + 15) / 16 - 1;
  const uint32_t lds_base = __builtin_amdgcn_readfirstlane(lds_offset(lds));
  const uint32_t voff = static_cast<uint32_t>(lane) * 16;

  // this wavefront's pieces of a stage: every kWaves-th, of group q / kGroup its activations' row groups, then its
  // weights'. Past the last piece the last again (the same bytes), past the last row group the last one, whose
  // results are not stored.
  const uint8_t* src[kCopies];
  int ks[kCopies], dst[kCopies];
#pragma unroll
  for (int c = 0; c < kCopies; ++c) {
    const int q = min(c * T::kWaves + w, T::kPieces - 1), r = q % T::kGroup;
    src[c] = r < T::kAPieces ? p.a + int64_t(min(m0 / 16 + r, r16_last)) * kt * kPiece
                             : p.b + int64_t(min(n0 / 16 + r - T::kAPieces, o16_last)) * kt * kPiece;
    ks[c] = q / T::kGroup;
    dst[c] = q * kPiece;
  }
  // copy c of stage b into a slot; past the end of K the last piece (a group that has none left adds nothing)
  auto copy = [&](int b, int slot, auto c_c) {
    constexpr int c = decltype(c_c)::value;
    const int k = WK == 1 ? b : min(b * WK + ks[c], kt - 1);
    lds_dma16(lds_base + static_cast<uint32_t>(slot * T::kStage + dst[c]), src[c], voff + static_cast<uint32_t>(k) * kPiece);
  };

  v4i acc[TI][TJ];
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j) acc[i][j] = v4i{0, 0, 0, 0};

  const uint8_t* a_lds = lds + (wk * T::kGroup + wm * TI) * kPiece + lane * 16;
  const uint8_t* b_lds = lds + (wk * T::kGroup + T::kAPieces + wn * TJ) * kPiece + lane * 16;
  v4i fa[TI], fb[kRingB];
  auto read_a = [&](int slot, int i) { fa[i] = *reinterpret_cast<const v4i*>(a_lds + slot * T::kStage + i * kPiece); };
  auto read_b = [&](int slot, int j, int to) { fb[to] = *reinterpret_cast<const v4i*>(b_lds + slot * T::kStage + j * kPiece); };

  static_for<S>([&](auto s) {
    static_for<kCopies>([&](auto c) { copy(min(static_cast<int>(decltype(s)::value), last), decltype(s)::value, c); });
  });
  wait_vmcnt<(S - 1) * kCopies>();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < TI; ++i) read_a(0, i);
  read_b(0, 0, 0);
  read_b(0, 1, 1);
  constexpr int kSteps = TI * TJ;
  int slot = 0;
  // (kt is even: only with more than two groups can some have nothing in the last stage)
  const int mine = WK > 2 && last * WK + wk >= kt ? last - 1 : last;
  for (int b = 0; b <= last; ++b) {
    const int ahead = min(b + S, last);  // past the end: the last stage over itself, the same bytes
    const int slot1 = slot + 1 == S ? 0 : slot + 1;
    if constexpr (WK > 2)
      if (b > mine) {
#pragma unroll
        for (int i = 0; i < TI; ++i) fa[i] = v4i{0, 0, 0, 0};
      }
    static_for<kSteps>([&](auto mc) {
      constexpr int m = decltype(mc)::value, i = m % TI, j = m / TI;
      constexpr int kFree = (TJ - 2) * TI;  // the first step at which the stage's slot is free
      if constexpr (m == kFree) {
        wait_vmcnt_lds<(S - 2) * kCopies>();  // copies land in the order they were issued in
        __syncthreads();
      }
      if constexpr (i == 0) {
        if constexpr (j < TJ - 2)
          read_b(slot, j + 2, (j + 2) % kRingB);
        else
          read_b(slot1, j + 2 - TJ, (j + 2) % kRingB);
      }
      acc[i][j] = mfma(fb[j % kRingB], fa[i], acc[i][j]);
      if constexpr (m >= kFree) {  // the copies of the stage that takes this one's slot, dealt to the steps that are left
        constexpr int kLeft = kSteps - kFree, at = m - kFree;
        constexpr int c0 = kCopies * at / kLeft, c1 = kCopies * (at + 1) / kLeft;
        static_for<c1 - c0>([&](auto c) { copy(ahead, slot, std::integral_constant<int, c0 + decltype(c)::value>{}); });
      }
      if constexpr (j == TJ - 1) read_a(slot1, i);
      __builtin_amdgcn_sched_barrier(0);
    });
    slot = slot1;
  }
  wait_vmcnt<0>();

  if constexpr (WK > 1) {
    __syncthreads();  // the last copies have landed: the sums take the ring's place
    v4i* part = reinterpret_cast<v4i*>(lds);
    const int u = w % (T::WM * T::WN);
    if (wk > 0) {
#pragma unroll
      for (int ij = 0; ij < TI * TJ; ++ij)
        part[(((wk - 1) * T::WM * T::WN + u) * TI * TJ + ij) * 64 + lane] = acc[ij / TJ][ij % TJ];
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int g = 0; g < WK - 1; ++g)
#pragma unroll
      for (int ij = 0; ij < TI * TJ; ++ij) acc[ij / TJ][ij % TJ] += part[((g * T::WM * T::WN + u) * TI * TJ + ij) * 64 + lane];
  }

  // lane l holds, of row l % 16 of an activation tile, outputs 4 (l / 16) .. + 3 of each weight tile. Two
  // neighbouring weight tiles trade halves so that a lane holds 8 outputs: lane groups 0 and 2 those of tile
  // j, 1 and 3 of tile j + 1, 64 contiguous bytes of a row from its four lanes.
  const int lg = lane >> 4;
  float sx[TI];
#pragma unroll
  for (int i = 0; i < TI; ++i) sx[i] = p.as[min(m0 + (wm * TI + i) * 16 + (lane & 15), p.n - 1)];
#pragma unroll
  for (int j = 0; j < TJ; j += 2) {
    float sw[2][4];
    uint32_t odd = 0;  // a bit for each of the lane's eight channels: a channel's way does not depend on those beside it
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        sw[u][q] = p.bs[min(n0 + (wn * TJ + j + u) * 16 + 4 * lg + q, p.n_out - 1)];
        odd |= static_cast<uint32_t>(odd_scale(sw[u][q])) << (4 * u + q);
      }
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      float y[2][4];
      if (odd) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int q = 0; q < 4; ++q) y[u][q] = scaled(acc[i][j + u][q], sx[i], sw[u][q], odd >> (4 * u + q) & 1);
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int q = 0; q < 4; ++q) y[u][q] = scaled(acc[i][j + u][q], sx[i], sw[u][q], false);
      }
      const auto d0 = __builtin_amdgcn_permlane16_swap(pk_bf16(y[0][0], y[0][1]), pk_bf16(y[1][0], y[1][1]), false, false);
      const auto d1 = __builtin_amdgcn_permlane16_swap(pk_bf16(y[0][2], y[0][3]), pk_bf16(y[1][2], y[1][3]), false, false);
      const v4i chunk = {static_cast<int>(d0[0]), static_cast<int>(d1[0]), static_cast<int>(d0[1]),
                         static_cast<int>(d1[1])};
      const int64_t row = m0 + (wm * TI + i) * 16 + (lane & 15);
      const int o = n0 + (wn * TJ + j + (lg & 1)) * 16 + (lg >> 1) * 8;
      if (row >= p.n) continue;
      uint16_t* out = p.y + row * p.ldy + o;
      if (o + 8 <= p.n_out) {
        if constexpr (NT)
          __builtin_nontemporal_store(chunk, reinterpret_cast<v4i*>(out));
        else
          *reinterpret_cast<v4i_any*>(out) = chunk;
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
// Tile shapes. A tile's time is a fixed part (its first copies, its results) and one for each K block, measured
// with every CU at work (in 10 ns): the larger the tile, the less of its time goes into moving operands, and the fewer of them
// there are to fill the CUs. Small tiles have few MFMAs a stage, so that its barrier and its copies' latency are what takes time:
// their wavefronts split K, and a stage is two or four groups' 64 columns (300 x 2000 x 1111, 64 x 64: one group 7.7 us, two 7.6
// with half the LDS; 32 x 64 with four 6.7).
using T32x64 = Shape<32, 64, 2, 1, 4, 4>;
using T64 = Shape<64, 64, 4, 1, 2, 4>;
using T64x128 = Shape<64, 128, 2, 2, 2, 4>;
using T128 = Shape<128, 128, 4, 2, 1, 4>;
using T256x128 = Shape<256, 128, 4, 2, 1, 4>;
using T192x128 = Shape<192, 128, 4, 2, 1, 4>;
using T192 = Shape<192, 192, 4, 2, 1, 3>;
using T192x256 = Shape<192, 256, 2, 4, 1, 3>;
using T256 = Shape<256, 256, 2, 4, 1, 3>;
struct ShapeCost {
  int bm, bn, fixed, block;
};
constexpr ShapeCost kCosts[] = {{32, 64, 240, 15},    {64, 64, 220, 20},   {64, 128, 310, 30},  {128, 128, 270, 40}, {192, 128, 350, 55},
                                {256, 128, 420, 74}, {192, 192, 450, 84}, {192, 256, 500, 94}, {256, 256, 800, 130}};
enum { kT32x64, kT64, kT64x128, kT128, kT192x128, kT256x128, kT192, kT192x256, kT256, kShapes };

struct Plan {
  int kb;
  int64_t q_bytes, total;
};
static Plan plan(int32_t n, int32_t k_in) {
  Plan p;
  p.kb = (k_in + 127) / 128;
  p.q_bytes = round_up(n, 16) * p.kb * 128;
  p.total = p.q_bytes + round_up(n, 16) * 4;
  return p;
}

template <typename T>
static int launch_tiles(const Args& p, hipStream_t s) {
  const int64_t mts = (p.n + T::BM - 1) / T::BM, nts = (p.n_out + T::BN - 1) / T::BN;
  const dim3 grid(static_cast<unsigned>(tile_grid(mts, nts)));
  if (reinterpret_cast<uintptr_t>(p.y) % 64 == 0 && p.ldy % 32 == 0)
    hipLaunchKernelGGL((tile_kernel<T, true>), grid, dim3(T::kThreads), 0, s, p);
  else
    hipLaunchKernelGGL((tile_kernel<T, false>), grid, dim3(T::kThreads), 0, s, p);
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
template <int ROWS, bool VEC, bool NT, bool SILU>
static int launch_quant(const Args& p, const RowsIn& in, uint8_t* q, float* sx, hipStream_t s) {
  const dim3 grid((p.n + ROWS - 1) / ROWS);
  auto go = [&](auto kernel, int waves) {
    hipLaunchKernelGGL(kernel, grid, dim3(64 * waves), 0, s, in.x, in.ldx, p.n, in.k_in, q, sx, p.kb);
  };
  // units: 8 kb chunks of 64 / ROWS lanes
  const int units = (8 * p.kb * ROWS + 63) / 64;
  if (units <= 8)
    go(quant_kernel<ROWS, 4, 2, VEC, NT, SILU>, 4);
  else if (units <= 16)
    go(quant_kernel<ROWS, 8, 2, VEC, NT, SILU>, 8);
  else if (units <= 32)
    go(quant_kernel<ROWS, 8, 4, VEC, NT, SILU>, 8);
  else if (units <= 64)
    go(quant_kernel<ROWS, 16, 4, VEC, NT, SILU>, 16);
  else
    go(quant_kernel<ROWS, 16, 0, VEC, NT, SILU>, 16);
  AFD_CHECK_LAUNCH();
  return AFD_OK;
}

// The shape whose rounds over the CUs take least
static int best_shape(int64_t n, int64_t n_out, int kb, int cus) {
  int best = 0;
  int64_t least = 0;
  for (int i = 0; i < kShapes; ++i) {
    const ShapeCost& c = kCosts[i];
    const int64_t tiles = ((n + c.bm - 1) / c.bm) * ((n_out + c.bn - 1) / c.bn);
    const int64_t time = (tiles + cus - 1) / cus * (c.fixed + int64_t(kb) * c.block);
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
  int st = check_dims(weights->n_out, weights->k_in);
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
  const RowsIn in = {x, ldx, weights->k_in};
  // the rows kernel's own quantization, up to 32 K elements: a launch less, which a call from Python has 3 us of, and in a graph no
  // slower than two but for many short rows (4096 x 4096, with and without: 1 row 6.3 and 8.7 us, 4 rows 7.3 and 9.2, 8 rows 9.4
  // and 9.5; 64 x 512 7.0 and 6.2); half of that where rows are not aligned (4 x 4001 7.7 and 9.4, 8 x 4001 11.5 and 9.7)
  const int64_t elements = int64_t(n) * pl.kb * 128;
  if (n <= kFusedRows && elements <= (vec ? kFusedBytes : kFusedBytes / 2))
    return silu ? launch_fused_rows<true>(p, in, vec, s) : launch_fused_rows<false>(p, in, vec, s);
  const bool nt = int64_t(n) * weights->k_in * (silu ? 4 : 2) > kCachedBytes;
  auto quant = [&](auto silu_c) {
    constexpr bool kSilu = decltype(silu_c)::value;
    // Four rows a workgroup while those are few for the CUs, eight above (4096 columns in a graph, 4 / 8 / 16 rows: 300 tokens
    // 3.5 / 4.8 / 7.5 us, 2900 7.8 / 9.0 / 9.5, 8192 22.2 / 20.5 / 21.3, 16384 41.0 / 38.6 / 37.8)
    auto rows = [&](auto rows_c) {
      constexpr int R = decltype(rows_c)::value;
      if (vec && nt) return launch_quant<R, true, true, kSilu>(p, in, q, sx, s);
      if (vec) return launch_quant<R, true, false, kSilu>(p, in, q, sx, s);
      return launch_quant<R, false, false, kSilu>(p, in, q, sx, s);
    };
    return n <= 16 * device_cu_count() ? rows(std::integral_constant<int, 4>{}) : rows(std::integral_constant<int, 8>{});
  };
  st = silu ? quant(std::true_type{}) : quant(std::false_type{});
  if (st != AFD_OK) return st;
  // up to 64 rows the weights are read once; above, tiles (4096 x 4096 without the quantization: 64 rows 8.7 us against 8.6 with
  // tiles of 32 x 64, 48 x 2048 x 4096 4.8 against 5.9, 100 rows 15.1 against 8.6)
  if (n <= 16) return launch_rows<1, false, false>(p, in, vec, s);
  if (n <= 32) return launch_rows<2, false, false>(p, in, vec, s);
  if (n <= 48) return launch_rows<3, false, false>(p, in, vec, s);
  if (n <= 64) return launch_rows<4, false, false>(p, in, vec, s);
  switch (best_shape(n, p.n_out, p.kb, device_cu_count())) {
    case kT32x64: return launch_tiles<T32x64>(p, s);
    case kT64: return launch_tiles<T64>(p, s);
    case kT64x128: return launch_tiles<T64x128>(p, s);
    case kT128: return launch_tiles<T128>(p, s);
    case kT192x128: return launch_tiles<T192x128>(p, s);
    case kT192: return launch_tiles<T192>(p, s);
    case kT192x256: return launch_tiles<T192x256>(p, s);
    case kT256x128: return launch_tiles<T256x128>(p, s);
    default: return launch_tiles<T256>(p, s);
  }
}

}  // namespace linear8
}  // namespace afd

using namespace afd;

extern "C" int afd_linear_i8_workspace(int32_t n, int32_t k_in, uint64_t* bytes) {
  if (!bytes || n < 0 || n > linear::kMaxRows) return AFD_ERR_ARG;
  const int st = linear::check_dims(1, k_in);
  if (st != AFD_OK) return st;
  *bytes = static_cast<uint64_t>(linear8::plan(n, k_in).total);
  return AFD_OK;
}

extern "C" int afd_linear_i8(const afd_linear_weights* weights, const uint16_t* x, int64_t ldx, int32_t n, void* ws,
                             uint64_t ws_bytes, uint16_t* y, int64_t ldy, afd_stream_t stream) {
  return linear8::run(weights, x, ldx, n, false, ws, ws_bytes, y, ldy, static_cast<hipStream_t>(stream));
}

extern "C" int afd_linear_i8_silu_mul(const afd_linear_weights* weights, const uint16_t* gate_up, int64_t ld, int32_t n,
                                      void* ws, uint64_t ws_bytes, uint16_t* y, int64_t ldy, afd_stream_t stream) {
  return linear8::run(weights, gate_up, ld, n, true, ws, ws_bytes, y, ldy, static_cast<hipStream_t>(stream));
}
