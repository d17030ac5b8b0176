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
// Every block's MFMA sum starts from 0 and is folded into the result with its scale by one fp32
// fused multiply-add, so scales may be 0, tiny or huge. A row of x with an infinity or a NaN in a block gets
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
// A wavefront quantizes 16 rows x one K block: lane l chunks l / 16 of both 64-column pieces of row
// l % 16. vec: 16-byte loads of whole chunks.
__global__ __launch_bounds__(256) void quant_kernel(const uint16_t* __restrict__ x, int64_t ldx, int n, int k_in,
                                                    uint8_t* __restrict__ q, float* __restrict__ s, int kb,
                                                    int a_rows, bool vec) {
  const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (item >= ((int64_t(n) + 15) / 16) * kb) return;
  const int64_t r16 = item / kb;
  const int b = static_cast<int>(item % kb);
  const int lane = threadIdx.x & 63, c = lane >> 4;
  const int64_t row = r16 * 16 + (lane & 15);
  float v[2][16];
  uint32_t top = 0;  // bits of the largest magnitude: infinities and NaN above every number
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int k0 = b * 128 + h * 64 + c * 16;
    const uint16_t* p = x + row * ldx + k0;
    if (vec && row < n && k0 + 16 <= k_in) {
      const v4i lo = *reinterpret_cast<const v4i*>(p), hi = *reinterpret_cast<const v4i*>(p + 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = static_cast<uint32_t>(i < 4 ? lo[i & 3] : hi[i & 3]);
        v[h][2 * i] = __uint_as_float(w << 16);
        v[h][2 * i + 1] = __uint_as_float(w & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[h][i] = row < n && k0 + i < k_in ? bf16_to_f32(p[i]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[h][i]) & 0x7fffffffu);
  }
  const auto r0 = __builtin_amdgcn_permlane16_swap(top, top, false, false);
  top = max(r0[0], r0[1]);
  const auto r1 = __builtin_amdgcn_permlane32_swap(top, top, false, false);
  top = max(r1[0], r1[1]);
  const bool finite = top < 0x7f800000u;
  const float sc = fmaxf(__uint_as_float(top), kFp8Eps) / kE4m3Max;
  const float rsc = 1.0f / sc;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    v4i out;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      out[i] = finite ? static_cast<int>(pk4_e4m3(div_by(v[h][4 * i], sc, rsc), div_by(v[h][4 * i + 1], sc, rsc),
                                                  div_by(v[h][4 * i + 2], sc, rsc), div_by(v[h][4 * i + 3], sc, rsc)))
                      : 0;
    *reinterpret_cast<v4i*>(q + (r16 * (2 * kb) + 2 * b + h) * kPiece + lane * 16) = out;
  }
  if (c == 0 && row < n) s[int64_t(b) * a_rows + row] = finite ? sc : __builtin_nanf("");
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
// Up to 16 MT rows of x: a call is bound by reading the weights once. A workgroup owns 16 outputs over the
// whole K, its wavefronts a share of the K blocks each, weights and activations straight into
// registers; the wavefronts' sums meet in LDS, in their order.
constexpr int kRowWaves = 8;

template <int MT>
__global__ __launch_bounds__(64 * kRowWaves) void rows_kernel(Args p) {
  __shared__ v4f part[kRowWaves][MT][64];
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int o16 = blockIdx.x;
  const int kt = 2 * p.kb;
  const int r16s = (p.n + 15) / 16;
  v4f acc[MT] = {};
  const uint8_t* bw = p.b + int64_t(o16) * kt * kPiece + lane * 16;
  const float* sw = p.bs + int64_t(o16 / 8) * p.kb;
  for (int b = w; b < p.kb; b += kRowWaves) {
    const v4i lo = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(bw + int64_t(2 * b) * kPiece));
    const v4i hi = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(bw + int64_t(2 * b + 1) * kPiece));
    const v8i fw = join(lo, hi);
    const float s_w = load_uniform(sw + b);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r16 = min(m, r16s - 1);
      const uint8_t* ax = p.a + (int64_t(r16) * kt + 2 * b) * kPiece + lane * 16;
      const v8i fx = join(*reinterpret_cast<const v4i*>(ax), *reinterpret_cast<const v4i*>(ax + kPiece));
      const float s = p.as[int64_t(b) * p.a_rows + r16 * 16 + (lane & 15)] * s_w;
      const v4f sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw, fx, v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0,
                                                                     127, 0, 127);
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[m][q] = __builtin_fmaf(sum[q], s, acc[m][q]);
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) part[w][m][lane] = acc[m];
  __syncthreads();
  // lane l: row l % 16 of x, outputs 4 (l / 16) .. + 3
  if (w >= MT) return;
  for (int m = w; m < MT; m += kRowWaves) {
    v4f y = part[0][m][lane];
    for (int i = 1; i < kRowWaves; ++i) y += part[i][m][lane];
    const int row = m * 16 + (lane & 15), o = o16 * 16 + 4 * (lane >> 4);
    if (row >= p.n) continue;
    uint16_t* out = p.y + row * p.ldy + o;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (o + q < p.n_out) out[q] = f32_to_bf16(y[q]);
  }
}

// ---------------------------------------------------------------- tiles
// BM rows of x by BN outputs, WM x WN wavefronts of TI x TJ MFMA tiles of 16x16 each (K 128 in one
// instruction, so a block's sum is one MFMA from 0 and its 4 values a lane are folded at once). A stage
// is one K block of both operands and the rows' scales, copied HBM -> LDS in 1 KiB pieces into two slots.
//
// A wavefront holds its TI activation fragments of a stage in registers and walks the TJ weight fragments,
// read two ahead, in an order kept as written (left alone, the compiler reads all of a stage first and then
// waits out every MFMA in turn: 322 us for 16384 x 4096 x 4096). When the last two are in registers (all of its reads of the stage done) it waits for
// its copies of the next stage and meets the others at the stage's one barrier: the next stage
// is there for all, and this one's slot is free for the copies of the stage after. The MFMAs of the
// last two weight fragments run while the next stage's first fragments are read.
template <int BM_, int BN_, int WM_, int WN_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int TI = BM / WM / 16, TJ = BN / WN / 16;
  static constexpr int kAPieces = BM / 16 * 2, kBPieces = BN / 16 * 2;
  static constexpr int kAQ = kAPieces / kWaves, kBQ = kBPieces / kWaves;
  static constexpr int kBOff = kAPieces * kPiece, kSOff = kBOff + kBPieces * kPiece;
  static constexpr int kStage = kSOff + BM * 4;
  static constexpr int kLds = 2 * kStage;
  static constexpr int kScaleWaves = BM / 64;  // each copies 64 rows' scales
  static_assert(TI * 16 * WM == BM && TJ * 16 * WN == BN && kAQ * kWaves == kAPieces && kBQ * kWaves == kBPieces, "tile");
  static_assert(TJ % 4 == 0 && BN / WN <= 128 && 128 % (BN / WN) == 0, "one weight scale per wavefront and K block");
  static_assert(kScaleWaves <= kWaves && BM <= kScaleRows && kLds <= 160 * 1024, "LDS");
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
  constexpr int kCopies = 1 + T::kAQ + T::kBQ;
  const int ws = w % T::kScaleWaves;
  auto copy = [&](int b, auto c_c) {
    constexpr int c = decltype(c_c)::value;
    const uint32_t st = lds_base + static_cast<uint32_t>((b & 1) * T::kStage);
    const uint32_t off = voff + static_cast<uint32_t>(b) * (2 * kPiece);
    if constexpr (c == 0) {
      // (every wavefront: two may write the same bytes, and the steps stay one block of code)
      lds_dma4(st + T::kSOff + ws * 256, p.as + int64_t(b) * p.a_rows + m0 + 64 * ws, lane * 4u);
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
  const uint8_t* a_lds = lds + wm * TI * 2 * kPiece + lane * 16;
  const uint8_t* b_lds = lds + T::kBOff + wn * TJ * 2 * kPiece + lane * 16;
  const uint8_t* s_lds = lds + T::kSOff + (wm * TI * 16 + (lane & 15)) * 4;
  v8i fa[TI], fb[4];
  float sx[TI], s[TI];
  auto read = [&](const uint8_t* f) {
    return join(*reinterpret_cast<const v4i*>(f), *reinterpret_cast<const v4i*>(f + kPiece));
  };
  auto read_a = [&](int b, int i) {
    fa[i] = read(a_lds + (b & 1) * T::kStage + i * 2 * kPiece);
    sx[i] = *reinterpret_cast<const float*>(s_lds + (b & 1) * T::kStage + i * 64);
  };
  auto read_b = [&](int b, int j) { return read(b_lds + (b & 1) * T::kStage + j * 2 * kPiece); };

  // An MFMA's result is folded kLate steps after it was issued (its latency is one step of its own and
  // one of the other wavefront's); the last ones of a stage in the next stage's first steps.
  constexpr int kSteps = TI * TJ, kLate = 3, kSums = 4;
  static_assert(kSteps % kSums == 0 && kLate < kSums, "a sum is folded before its registers take another");
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

  issue(0);
  wait_vmcnt<0>();
  __syncthreads();
  issue(min(1, last));
#pragma unroll
  for (int i = 0; i < TI; ++i) read_a(0, i);
  fb[0] = read_b(0, 0);
  fb[1] = read_b(0, 1);
  for (int b = 0; b <= last; ++b) {
    const int ahead = min(b + 2, last);  // past the end: the last stage over itself, the same bytes
    static_for<kSteps>([&](auto mc) {
      constexpr int m = decltype(mc)::value, i = m % TI, j = m / TI;
      constexpr int kFree = (TJ - 2) * TI;  // the first step at which the stage's slot is free
      if constexpr (m == kFree) {
        wait_vmcnt_lds<0>();
        __syncthreads();
        s_w = load_uniform(sw + min(b + 1, last));
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
  }
  static_for<kLate>([&](auto c) { fold(std::integral_constant<int, kSteps - kLate + decltype(c)::value>{}); });
  wait_vmcnt<0>();

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
using Large = Shape<256, 256, 4, 2>;
using Mid = Shape<128, 128, 2, 2>;

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
template <int MT>
static int launch_rows(const Args& p, hipStream_t s) {
  hipLaunchKernelGGL(rows_kernel<MT>, dim3((p.n_out + 15) / 16), dim3(64 * kRowWaves), 0, s, p);
  AFD_CHECK_LAUNCH();
  return AFD_OK;
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
  if (!weights || n < 0 || n > linear::kMaxRows) return AFD_ERR_ARG;
  const int st = linear::check_dims(weights->n_out, weights->k_in);
  if (st != AFD_OK) return st;
  if (ldx < weights->k_in || ldy < weights->n_out) return AFD_ERR_SHAPE;
  if (n == 0) return AFD_OK;
  if (!weights->image || !weights->scales || !x || !ws || !y) return AFD_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(weights->image) % 16) return AFD_ERR_SHAPE;
  const linear::Plan pl = linear::plan(n, weights->k_in);
  if (ws_bytes < static_cast<uint64_t>(pl.total) || reinterpret_cast<uintptr_t>(ws) % 16) return AFD_ERR_WORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint8_t* q = static_cast<uint8_t*>(ws);
  float* sx = reinterpret_cast<float*>(q + pl.q_bytes);
  const int64_t items = (int64_t(n) + 15) / 16 * pl.kb;
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 8 == 0;
  hipLaunchKernelGGL(linear::quant_kernel, dim3(static_cast<unsigned>((items + 3) / 4)), dim3(256), 0, s, x, ldx, n,
                     weights->k_in, q, sx, pl.kb, pl.a_rows, vec);
  AFD_CHECK_LAUNCH();
  linear::Args p = {};
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
  if (n <= 16) return linear::launch_rows<1>(p, s);
  if (n <= 32) return linear::launch_rows<2>(p, s);
  if (n <= 64) return linear::launch_rows<4>(p, s);
  const int64_t large = ((int64_t(n) + 255) / 256) * ((int64_t(p.n_out) + 255) / 256);
  if (large >= device_cu_count()) return linear::launch_tiles<linear::Large>(p, s);
  return linear::launch_tiles<linear::Mid>(p, s);
}
