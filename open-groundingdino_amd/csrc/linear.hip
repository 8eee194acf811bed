// A linear layer with its epilogue, and its gradients, for gfx950:
//
//   z = x W^T + b     y = act(z) + r          x [M, K], W [N, K], bf16 / fp16
//   dz = dy * act'(z)     dx = dz W     dW = dz^T x     db = sum_m dz     (dr = dy)
//
// All three products are one kernel, C[m][n] = sum_r A(m, r) B(n, r), whose
// operands lie in memory either with r contiguous ("rows": x, W, dz in the
// forward and dx) or with m / n contiguous ("columns": W in dx, dz and x in dW).
// Products of 16-bit values are exact in fp32 and the accumulators are fp32
// matrix-core registers; bias, activation and residual are applied to them in
// fp32 and the result is rounded once.  The backward rounds dz to 16 bits, as the
// matrix instructions take it, and needs act'(z): the forward writes z rounded to
// 16 bits beside y (for ReLU without a residual y itself tells where z > 0).
//
// Where the output has too few tiles to fill 256 CUs the sum over r is split: the
// parts go to a workspace in fp32 and a finishing kernel adds them in a fixed
// order and applies the epilogue.  There are no atomics: results repeat bit
// by bit.
#include "gd_common.h"

#include <cmath>
#include <type_traits>

namespace gd {
namespace {

enum Act : int { kNone = 0, kRelu = 1, kGelu = 2, kGeluTanh = 3, kSilu = 4 };

typedef short gd_i16x8 __attribute__((ext_vector_type(8)));
typedef short gd_i16x4 __attribute__((ext_vector_type(4)));
typedef float gd_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 gd_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 gd_f16x8 __attribute__((ext_vector_type(8)));

// acc += a b with acc held in accumulation registers, which 256 of the compiler's own products would move
// back and forth; their results are read only after GD_MMA_WAIT8 (a matrix instruction's result takes up to 18
// cycles, which the compiler does not see in assembly)
#ifndef GD_MMA_IN_PLACE
#define GD_MMA_IN_PLACE(name, acc, a, b, E) asm volatile(name " %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b))
#define GD_MMA_WAIT8(nops, r)                                                                              \
  asm volatile(nops : "+a"((r)[0]), "+a"((r)[1]), "+a"((r)[2]), "+a"((r)[3]), "+a"((r)[4]), "+a"((r)[5]), \
                     "+a"((r)[6]), "+a"((r)[7]))
#endif

// the two 16-bit types
struct Bf16 {
  static __device__ __forceinline__ float up(uint16_t h) { return bf16_to_f32(h); }
  static __device__ __forceinline__ uint16_t down(float f) { return f32_to_bf16(f); }
  static __device__ __forceinline__ gd_f32x4 mma(gd_i16x8 a, gd_i16x8 b, gd_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gd_bf16x8, a), __builtin_bit_cast(gd_bf16x8, b),
                                                   c, 0, 0, 0);
  }
  static __device__ __forceinline__ void mma_in(gd_f32x4& c, gd_i16x8 a, gd_i16x8 b) {
    GD_MMA_IN_PLACE("v_mfma_f32_16x16x32_bf16", c, a, b, Bf16);
  }
};
struct Fp16 {
  static __device__ __forceinline__ float up(uint16_t h) { return float(__builtin_bit_cast(_Float16, h)); }
  static __device__ __forceinline__ uint16_t down(float f) {
    const _Float16 h = (_Float16)f;
    return __builtin_bit_cast(uint16_t, h);
  }
  static __device__ __forceinline__ gd_f32x4 mma(gd_i16x8 a, gd_i16x8 b, gd_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(gd_f16x8, a), __builtin_bit_cast(gd_f16x8, b), c,
                                                  0, 0, 0);
  }
  static __device__ __forceinline__ void mma_in(gd_f32x4& c, gd_i16x8 a, gd_i16x8 b) {
    GD_MMA_IN_PLACE("v_mfma_f32_16x16x32_f16", c, a, b, Fp16);
  }
};

// ---- activations ------------------------------------------------------------
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// The normal distribution's Phi(z), and exp(-z^2 / 2) for its density: Abramowitz and Stegun 7.1.26,
// erfc(x) = t (a1 + t (a2 + ...)) exp(-x^2), t = 1 / (1 + p x), off by 1.5e-7 at most; on -|z|, so that the tail
// keeps its sign and does not cancel.
__device__ __forceinline__ float normal_cdf(float z, float* bell) {
  const float x = fabsf(z) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * x);
  const float e = exp_of(-0.5f * z * z);
  const float q = t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
  const float tail = 0.5f * q * e;
  *bell = e;
  return z > 0.f ? 1.f - tail : (z <= 0.f ? tail : z);
}

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + exp_of(-z)); }

constexpr float kTanhC = 0.79788456080286536f, kTanhA = 0.044715f;

// (the switch around the 8 values: a uniform branch each, not eight)
__device__ __forceinline__ void activate8(float v[8], int act) {
  switch (act) {
    case kRelu:
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];  // (NaN stays)
      break;
    case kGelu:
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float bell;
        v[j] *= normal_cdf(v[j], &bell);
      }
      break;
    case kGeluTanh:  // (1 + tanh u) / 2 = sigmoid(2 u)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= sigmoid(2.f * kTanhC * (v[j] + kTanhA * v[j] * v[j] * v[j]));
      break;
    case kSilu:
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= sigmoid(v[j]);
      break;
    default: break;
  }
}

// d[j] *= act'(z[j])
__device__ __forceinline__ void slope8(float d[8], const float z[8], int act) {
  switch (act) {
    case kRelu:
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = z[j] > 0.f ? d[j] : 0.f;
      break;
    case kGelu:
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float bell;
        const float c = normal_cdf(z[j], &bell);
        d[j] *= c + z[j] * bell * 0.39894228040143268f;
      }
      break;
    case kGeluTanh:
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float q = sigmoid(2.f * kTanhC * (z[j] + kTanhA * z[j] * z[j] * z[j]));
        d[j] *= q + 2.f * z[j] * q * (1.f - q) * kTanhC * (1.f + 3.f * kTanhA * z[j] * z[j]);
      }
      break;
    case kSilu:
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float q = sigmoid(z[j]);
        d[j] *= q * (1.f + z[j] * (1.f - q));
      }
      break;
    default: break;
  }
}

// ---- 8 consecutive 16-bit or fp32 values, the first `left` of them valid ------
template <typename E>
__device__ __forceinline__ void ld8(const void* p, int64_t at, bool f32, bool vec, int left, float v[8]) {
  if (f32) {
    const float* q = static_cast<const float*>(p) + at;
    if (vec && left >= 8) {
      const float4 a = reinterpret_cast<const float4*>(q)[0], b = reinterpret_cast<const float4*>(q)[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < left ? q[j] : 0.f;
    }
    return;
  }
  const uint16_t* q = static_cast<const uint16_t*>(p) + at;
  union {
    uint4 u;
    uint16_t h[8];
  } w;
  if (vec && left >= 8) {
    w.u = *reinterpret_cast<const uint4*>(q);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) w.h[j] = j < left ? q[j] : uint16_t(0);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = E::up(w.h[j]);
}

template <typename E>
__device__ __forceinline__ void st8(void* p, int64_t at, bool f32, bool vec, int left, const float v[8]) {
  if (f32) {
    float* q = static_cast<float*>(p) + at;
    if (vec && left >= 8) {
      reinterpret_cast<float4*>(q)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(q)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) q[j] = v[j];
    }
    return;
  }
  uint16_t* q = static_cast<uint16_t*>(p) + at;
  union {
    uint4 u;
    uint16_t h[8];
  } w;
#pragma unroll
  for (int j = 0; j < 8; ++j) w.h[j] = E::down(v[j]);
  if (vec && left >= 8) {
    *reinterpret_cast<uint4*>(q) = w.u;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) q[j] = w.h[j];
  }
}

// ---- the epilogue -------------------------------------------------------------
struct Epi {
  const uint16_t* bias;  // or NULL
  const void* res;       // or NULL
  void* y;
  uint16_t* z;           // or NULL: z for the backward, its rows padded to 8 with zeros
  int64_t ldr, ldy, ldz;
  int act;
  bool bias_vec, res_f32, res_vec, y_f32, y_vec;
};

// 8 values of a row: bias b and residual r were loaded before (zeros where there is none)
template <typename E>
__device__ __forceinline__ void epilogue8(const Epi& e, int64_t m, int n, int N, const float b[8], const float r[8],
                                          float v[8]) {
  const int left = N - n < 8 ? N - n : 8;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] += b[j];
  if (e.z) {
    float z[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = j < left ? v[j] : 0.f;
    st8<E>(e.z, m * e.ldz + n, false, true, 8, z);
  }
  activate8(v, e.act);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] += r[j];
  st8<E>(e.y, m * e.ldy + n, e.y_f32, e.y_vec, left, v);
}

// ---- the product ----------------------------------------------------------------
struct Gemm {
  const uint16_t *a, *b;  // 16-byte aligned, row pitches multiples of 8
  int64_t lda, ldb;
  int M, N;      // the output
  int ra, rb;    // extents of r in memory; the shorter operand counts as zero beyond (rows: multiples of 8)
  int ca, cb;    // columns in memory of a "columns" operand, multiples of 8
  int splits, r_per_split;  // r_per_split: a multiple of kR
  int tiles_m, tiles_n, group;  // group: see tile_of
  float* part;   // splits > 1: [splits][M][N]
  Epi epi;
};

constexpr int kR = 64;  // values of r per staged chunk

// A workgroup's tile.  Each XCD gets a contiguous range of the parts' tiles (its L2 is its own), in bands of `group`
// rows of tiles, down the band first: the tiles that run at one time on an XCD then cover a block of the output
// that is about square, and need the fewest rows of A and B from beyond its L2.
struct Tile {
  int m, n, split;
};
__device__ __forceinline__ Tile tile_of(const Gemm& p) {
  const int L = xcd_remap(int(blockIdx.x), int(gridDim.x));
  const int tiles = p.tiles_m * p.tiles_n;
  Tile t;
  t.split = L / tiles;
  const int i = L - t.split * tiles, band = i / (p.group * p.tiles_n), first = band * p.group;
  const int high = p.tiles_m - first < p.group ? p.tiles_m - first : p.group, j = i - first * p.tiles_n;
  t.m = first + j % high;
  t.n = j / high;
  return t;
}

// Offset of 16-byte chunk ch of row r in an LDS image.  Rows image [x][64 r]: 128-byte rows; 16 lanes read the same
// chunk of 16 consecutive rows, so the chunk index is xored with row / 2: with the row's parity that is every one of
// the 16 positions of 256 bytes, all 64 banks.
__device__ __forceinline__ int row_swz(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ int row_at(int row, int ch) { return row * kR + ((ch ^ row_swz(row)) << 3); }
// Columns image [64 r][X]: the transposing read (ds_read_b64_tr_b16) of half a wave touches rows q and 8 + q, q < 4, 32
// bytes each, which have to lie 32 bytes apart modulo 256.
template <int X>
__device__ __forceinline__ int col_swz(int r) {
  return X == 64 ? 2 * ((r >> 1) & 1) + 4 * ((r >> 3) & 1) : 2 * (r & 3) + 8 * ((r >> 3) & 1);
}
template <int X>
__device__ __forceinline__ int col_at(int r, int ch) { return r * X + ((ch ^ col_swz<X>(r)) << 3); }

__device__ __forceinline__ gd_i16x4 lds_tr(const uint16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) gd_i16x4*)(p));
}

// the operand of one 16 x 16 x 32 product: lane (c, g) holds r = 8 g .. 8 g + 7 of row x0 + c, chunk s of 32
template <int X, bool COL>
__device__ __forceinline__ gd_i16x8 fragment(const uint16_t* img, int x0, int s, int lane) {
  if constexpr (!COL) {
    return *reinterpret_cast<const gd_i16x8*>(img + row_at(x0 + (lane & 15), 4 * s + (lane >> 4)));
  } else {
    const int g = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
    const int ch = (x0 >> 3) + (p >> 1), sub = 4 * (p & 1);
    const gd_i16x4 lo = lds_tr(img + col_at<X>(32 * s + 8 * g + q, ch) + sub);
    const gd_i16x4 hi = lds_tr(img + col_at<X>(32 * s + 8 * g + 4 + q, ch) + sub);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// One operand's way into its LDS image of X rows (or columns) by 64 values of r.  A wave instruction moves 64 pieces
// of 16 bytes to consecutive LDS positions, so the swizzle is applied to the source: position pos of a row holds
// its chunk pos ^ swz.  Rows (columns) past the operand's end read its last one instead: their products land in
// outputs that are not stored.
template <int X, bool COL, int WAVES>
struct Loader {
  static constexpr int kInstr = X * 8 / 64 / WAVES;  // per wave and chunk
  static_assert(kInstr * 64 * WAVES == X * 8, "the waves share an image evenly");
  const uint16_t* base;      // of the tile and chunk, the same for every lane
  int64_t step;              // from chunk to chunk
  uint32_t offset[kInstr];   // bytes (the host keeps row pitches below kMaxPitch)
  __device__ __forceinline__ Loader(const uint16_t* p, int64_t ld, int x0, int end, int cols, int r0, int wave, int lane) {
    step = COL ? kR * ld : kR;
    base = p + (COL ? int64_t(r0) * ld + x0 : int64_t(x0) * ld + r0);
#pragma unroll
    for (int h = 0; h < kInstr; ++h) {
      const int piece = (wave + WAVES * h) * 64 + lane;
      if (COL) {
        const int r = piece / (X / 8), x = 8 * ((piece % (X / 8)) ^ col_swz<X>(r));
        offset[h] = uint32_t(r * uint32_t(ld) + (x0 + x < cols ? x : cols - 8 - x0)) * 2;
      } else {
        const int row = piece >> 3, x = x0 + row < end ? row : end - 1 - x0;
        offset[h] = (uint32_t(x) * uint32_t(ld) + 8 * ((piece & 7) ^ row_swz(row))) * 2;
      }
    }
  }
  // piece h of the chunk to the image at byte `at` of the LDS array
  __device__ __forceinline__ void issue(uint16_t* lds, uint32_t at, int wave, int h) const {
    GD_LDS_DMA16_AT(base, offset[h], lds, at + uint32_t(wave + WAVES * h) * 1024);
  }
  __device__ __forceinline__ void issue(uint16_t* lds, uint32_t at, int wave) {
#pragma unroll
    for (int h = 0; h < kInstr; ++h) issue(lds, at, wave, h);
    base += step;
  }
};

// the chunk of r that ends inside: through registers, zeros past the operand's end
template <int X, bool COL, int WAVES>
__device__ __forceinline__ void load_tail(uint16_t* img, const uint16_t* p, int64_t ld, int x0, int end, int cols, int r0,
                                          int r_end) {
#pragma unroll
  for (int v = threadIdx.x; v < X * 8; v += 64 * WAVES) {
    const int xi = COL ? 8 * (v % (X / 8)) : v >> 3, ri = COL ? v / (X / 8) : 8 * (v & 7);
    const int x = x0 + xi, r = r0 + ri;
    const bool ok = r < r_end && x < (COL ? cols : end);
    const uint4 u = ok ? *reinterpret_cast<const uint4*>(p + (COL ? int64_t(r) * ld + x : int64_t(x) * ld + r))
                       : make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(img + (COL ? col_at<X>(ri, v % (X / 8)) : row_at(xi, v & 7))) = u;
  }
}

// A wave's TM x TN blocks to memory: 16 rows at a time through its own LDS (own), so that a row leaves in 16-byte
// pieces of neighbouring lanes; pitch 16 TN + 4: 16 rows' float4s, and the reads of 8 neighbouring columns, touch
// all banks once.  A lane keeps its columns, so the bias is loaded once; the residual of its next row is under way
// meanwhile.  m0, n0: the wave's corner.
template <typename E, int TM, int TN>
__device__ __forceinline__ void store_tile(const Gemm& p, const gd_f32x4 (&acc)[TM][TN], float* own, int m0, int n0,
                                           int split, int lane) {
  constexpr int kPitch = 16 * TN + 4;
  constexpr int kLanes = 2 * TN, kRows = 64 / kLanes, kPasses = 16 / kRows;  // lanes per row, rows per pass
  const int col = 8 * (lane % kLanes), n = n0 + col, left = p.N - n < 8 ? p.N - n : 8;
  const bool whole = p.splits == 1;
  float bias[8], res[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) bias[j] = res[j] = 0.f;
  if (whole && p.epi.bias && left > 0) ld8<E>(p.epi.bias, n, false, p.epi.bias_vec, left, bias);
  const bool has_res = whole && p.epi.res != nullptr;
  auto load_res = [&](int m) {
    if (has_res && m < p.M && left > 0) ld8<E>(p.epi.res, m * p.epi.ldr + n, p.epi.res_f32, p.epi.res_vec, left, res);
  };
  m0 += lane / kLanes;  // this lane's first row; it takes every kRows-th
  load_res(m0);
  __syncthreads();  // the images have been read
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
      *reinterpret_cast<gd_f32x4*>(own + (lane & 15) * kPitch + 16 * j + 4 * (lane >> 4)) = acc[i][j];
    gd_wave_sync();
#pragma unroll 1
    for (int h = 0; h < kPasses; ++h) {
      const int row = h * kRows + lane / kLanes, m = m0 + 16 * i + h * kRows;
      float now[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) now[j] = res[j];
      load_res(m + kRows);  // of the next pass
      const float4 u = *reinterpret_cast<const float4*>(own + row * kPitch + col);
      const float4 w = *reinterpret_cast<const float4*>(own + row * kPitch + col + 4);
      float v[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
      if (m < p.M && left > 0) {
        if (whole)
          epilogue8<E>(p.epi, m, n, p.N, bias, now, v);
        else
          st8<E>(p.part, (int64_t(split) * p.M + m) * p.N + n, true, (p.N & 3) == 0, left, v);
      }
    }
    gd_wave_sync();
  }
}

// WM x WN waves, each of TM x TN blocks of 16 x 16; a ring of ST images, ST - 1 chunks of r in flight
template <typename E, int WM, int WN, int TM, int TN, int ST, bool AC, bool BC>
__global__ void __launch_bounds__(64 * WM * WN) linear_gemm(const Gemm p) {
  constexpr int kWaves = WM * WN, BM = 16 * WM * TM, BN = 16 * WN * TN;
  constexpr int kStage = (BM + BN) * kR;
  constexpr int kPitch = 16 * TN + 4;  // floats: the epilogue's rows
  static_assert(kWaves * 16 * kPitch * 2 <= ST * kStage, "the epilogue's staging fits");
  __shared__ __attribute__((aligned(16))) uint16_t lds[ST * kStage];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / WN, wn = wave % WN;
  const Tile t = tile_of(p);
  const int m0 = t.m * BM, n0 = t.n * BN, split = t.split;
  const int r_end = p.ra > p.rb ? p.ra : p.rb, r_both = p.ra < p.rb ? p.ra : p.rb;
  const int rb0 = split * p.r_per_split;
  const int re = rb0 + p.r_per_split < r_end ? rb0 + p.r_per_split : r_end;
  const int rf = re < r_both ? re : r_both;
  const int nfull = rf > rb0 ? (rf - rb0) / kR : 0;

  using LA = Loader<BM, AC, kWaves>;
  using LB = Loader<BN, BC, kWaves>;
  constexpr int kInstr = LA::kInstr + LB::kInstr;
  LA la(p.a, p.lda, m0, p.M, p.ca, rb0, wave, lane);
  LB lb(p.b, p.ldb, n0, p.N, p.cb, rb0, wave, lane);
  auto issue = [&](int k) {
    const uint32_t at = uint32_t(k % ST) * (2 * kStage);
    la.issue(lds, at, wave);
    lb.issue(lds, at + 2 * BM * kR, wave);
  };

  gd_f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = gd_f32x4{0.f, 0.f, 0.f, 0.f};
  auto compute = [&](const uint16_t* img) {
#pragma unroll
    for (int s = 0; s < kR / 32; ++s) {
      gd_i16x8 fa[TM], fb[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) fb[j] = fragment<BN, BC>(img + BM * kR, 16 * (wn * TN + j), s, lane);
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[i] = fragment<BM, AC>(img, 16 * (wm * TM + i), s, lane);
      // transposed: lane (c, g) receives C[16 i + c][16 j + 4 g .. + 3], four values of a row
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = E::mma(fb[j], fa[i], acc[i][j]);
    }
  };

#pragma unroll
  for (int k = 0; k < ST - 1; ++k)
    if (k < nfull) issue(k);
  for (int k = 0; k < nfull; ++k) {
    if (ST > 2 && nfull - 1 - k >= ST - 2)
      gd_wait_vmcnt((ST - 2) * kInstr);
    else if (ST > 3 && nfull - 1 - k == ST - 3)
      gd_wait_vmcnt((ST > 3 ? ST - 3 : 0) * kInstr);
    else
      gd_wait_vmcnt(0);
    gd_lds_barrier();  // chunk k has landed for every wave, and every wave has read chunk k - 1
    if (k + ST - 1 < nfull) issue(k + ST - 1);
    compute(lds + k % ST * kStage);
  }
  for (int r0 = rb0 + nfull * kR; r0 < re; r0 += kR) {  // (none of the ring is in flight)
    __syncthreads();
    load_tail<BM, AC, kWaves>(lds, p.a, p.lda, m0, p.M, p.ca, r0, p.ra < re ? p.ra : re);
    load_tail<BN, BC, kWaves>(lds + BM * kR, p.b, p.ldb, n0, p.N, p.cb, r0, p.rb < re ? p.rb : re);
    __syncthreads();
    compute(lds);
  }

  store_tile<E, TM, TN>(p, acc, reinterpret_cast<float*>(lds) + wave * 16 * kPitch, m0 + 16 * wm * TM, n0 + 16 * wn * TN,
                        split, lane);
}

// 256 x 256 tiles of 4 waves, 128 x 128 each, one per SIMD: the largest wave tile its 512 registers allow, since LDS is
// what the matrix cores compete for (128 KB are read and 64 KB written per chunk of 64 values of r; 8 waves of 128 x
// 64 read 192 KB and wait for each other: 444 us at 16384 x 4096 x 4096, the products and reads alone 286, the
// loads alone 299).  A phase multiplies half a chunk whose fragments are in registers; between its products the next
// half's fragments are read and the loads issued, so nothing waits but for the barrier in the middle of a chunk.
// LDS holds a ring of 5 images of one operand each, in the order A0 B0 A1 B1 A2 ...: when chunk k has been read, its two
// images take B of chunk k + 2, needed first, and A of chunk k + 3.
template <typename E, bool AC, bool BC>
__global__ void __launch_bounds__(256, 1) linear_gemm256(const Gemm p) {
  constexpr int T = 8, kWaves = 4, BX = 256, kImg = BX * kR, kRing = 5;
  constexpr int kPitch = 16 * T + 4;
  __shared__ __attribute__((aligned(16))) uint16_t lds[kRing * kImg];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave >> 1, wn = wave & 1;
  const Tile t = tile_of(p);
  const int m0 = t.m * BX, n0 = t.n * BX, split = t.split;
  const int r_end = p.ra > p.rb ? p.ra : p.rb, r_both = p.ra < p.rb ? p.ra : p.rb;
  const int rb0 = split * p.r_per_split;
  const int re = rb0 + p.r_per_split < r_end ? rb0 + p.r_per_split : r_end;
  const int rf = re < r_both ? re : r_both;
  const int nfull = rf > rb0 ? (rf - rb0) / kR : 0;

  using Load = Loader<BX, AC, kWaves>;  // 8 instructions a wave and image
  Load la(p.a, p.lda, m0, p.M, p.ca, rb0, wave, lane);
  Loader<BX, BC, kWaves> lb(p.b, p.ldb, n0, p.N, p.cb, rb0, wave, lane);
  static_assert(Load::kInstr == T, "one instruction per row of blocks");

  gd_f32x4 acc[T][T];
#pragma unroll
  for (int i = 0; i < T; ++i)
#pragma unroll
    for (int j = 0; j < T; ++j) acc[i][j] = gd_f32x4{0.f, 0.f, 0.f, 0.f};
  struct Frags {
    gd_i16x8 a[T], b[T];
  };
  // image q of the ring, as its byte in LDS; its operand's fragment i, half s
  auto wrap = [](int q) { return q >= kRing ? q - kRing : q; };
  auto read1 = [&](Frags& f, int qa, int s, int i) {
    f.a[i] = fragment<BX, AC>(lds + qa * kImg, 16 * (wm * T + i), s, lane);
    f.b[i] = fragment<BX, BC>(lds + wrap(qa + 1) * kImg, 16 * (wn * T + i), s, lane);
  };
  auto multiply1 = [&](const Frags& f, int i) {
#pragma unroll
    for (int j = 0; j < T; ++j) E::mma_in(acc[i][j], f.b[j], f.a[i]);
  };

  Frags f0, f1;
  if (nfull > 0) {
    la.issue(lds, 0, wave);
    lb.issue(lds, 2 * kImg, wave);
    if (nfull > 1) {
      la.issue(lds, 4 * kImg, wave);
      lb.issue(lds, 6 * kImg, wave);
    }
    if (nfull > 2) {
      la.issue(lds, 8 * kImg, wave);
      gd_wait_vmcnt(3 * T);
    } else {
      gd_wait_vmcnt(0);
    }
    gd_raw_barrier();
#pragma unroll
    for (int i = 0; i < T; ++i) read1(f0, 0, 0, i);
    // one chunk; q: its A's image.  MORE: chunks k + 2 and k + 3 exist
    auto chunk = [&](int k, int q, auto MORE) {
      constexpr bool kMore = decltype(MORE)::value;
#pragma unroll
      for (int i = 0; i < T; ++i) {
        read1(f1, q, 1, i);
        multiply1(f0, i);
        __builtin_amdgcn_sched_barrier(0);
      }
      // chunk k + 1 has landed, all but A of chunk k + 2; and chunk k has been read
      if (kMore || k + 2 < nfull)
        gd_wait_vmcnt(T);
      else
        gd_wait_vmcnt(0);
      gd_lds_barrier();
      const int qn = k + 1 < nfull ? wrap(q + 2) : q;  // (the last chunk's is read again, for nothing)
      const uint32_t to_b = uint32_t(q) * (2 * kImg), to_a = uint32_t(wrap(q + 1)) * (2 * kImg);
#pragma unroll
      for (int i = 0; i < T; ++i) {
        read1(f0, qn, 0, i);
        if (i < T / 2) {
          if (kMore || k + 2 < nfull) {
            lb.issue(lds, to_b, wave, 2 * i);
            lb.issue(lds, to_b, wave, 2 * i + 1);
          }
        } else if (kMore) {
          la.issue(lds, to_a, wave, 2 * i - T);
          la.issue(lds, to_a, wave, 2 * i - T + 1);
        }
        multiply1(f1, i);
        __builtin_amdgcn_sched_barrier(0);
      }
      la.base += la.step;
      lb.base += lb.step;
    };
    int k = 0, q = 0;
    for (; k + 3 < nfull; ++k, q = wrap(q + 2)) chunk(k, q, std::true_type());
    for (; k < nfull; ++k, q = wrap(q + 2)) chunk(k, q, std::false_type());
  }
  for (int r0 = rb0 + nfull * kR; r0 < re; r0 += kR) {
    __syncthreads();
    load_tail<BX, AC, kWaves>(lds, p.a, p.lda, m0, p.M, p.ca, r0, p.ra < re ? p.ra : re);
    load_tail<BX, BC, kWaves>(lds + kImg, p.b, p.ldb, n0, p.N, p.cb, r0, p.rb < re ? p.rb : re);
    __syncthreads();
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < T; ++i) read1(f0, 0, s, i);
#pragma unroll
      for (int i = 0; i < T; ++i) multiply1(f0, i);
    }
  }
  GD_MMA_WAIT8("s_nop 15\n\ts_nop 7", acc[0]);
#pragma unroll
  for (int i = 1; i < T; ++i) GD_MMA_WAIT8("", acc[i]);
  store_tile<E, T, T>(p, acc, reinterpret_cast<float*>(lds) + wave * 16 * kPitch, m0 + 16 * wm * T, n0 + 16 * wn * T,
                      split, lane);
}

// the parts added in order, then the epilogue; a thread per 8 columns
template <typename E>
__global__ void __launch_bounds__(256) linear_finish(const float* __restrict__ part, int splits, int M, int N, Epi epi) {
  const int per_row = (N + 7) / 8;
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= int64_t(M) * per_row) return;
  const int64_t m = i / per_row;
  const int n = int(i - m * per_row) * 8;
  const bool vec = (N & 3) == 0;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    float u[8];
    ld8<E>(part, (int64_t(s) * M + m) * N + n, true, vec, N - n, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += u[j];
  }
  float b[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, r[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int left = N - n < 8 ? N - n : 8;
  if (epi.bias) ld8<E>(epi.bias, n, false, epi.bias_vec, left, b);
  if (epi.res) ld8<E>(epi.res, m * epi.ldr + n, epi.res_f32, epi.res_vec, left, r);
  epilogue8<E>(epi, m, n, N, b, r, v);
}

// ---- dz = dy * act'(z), and parts of its column sums -------------------------------
struct Dact {
  const void* dy;
  const uint16_t* z;  // NULL: no activation
  uint16_t* dz;       // or NULL; rows padded to 8 with zeros
  float* sums;        // or NULL: [workgroups][N]
  int64_t lddy, ldz, lddz, rows;  // rows: of one workgroup
  int M, N, act, lanes;           // lanes: of a row, a power of two up to 64
  bool dy_f32, dy_vec, z_vec;
};

template <typename E>
__global__ void __launch_bounds__(256) linear_dact(const Dact p) {
  __shared__ float lds[256 * 9];
  const int slab = 8 * p.lanes, at = threadIdx.x / p.lanes, rows = 256 / p.lanes;
  const int n = int(blockIdx.y) * slab + 8 * (threadIdx.x % p.lanes);
  const int64_t begin = int64_t(blockIdx.x) * p.rows;
  const int64_t end = begin + p.rows < p.M ? begin + p.rows : p.M;
  const int left = p.N - n < 8 ? p.N - n : 8;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (left > 0) {
#pragma unroll 2
    for (int64_t m = begin + at; m < end; m += rows) {
      float d[8];
      ld8<E>(p.dy, m * p.lddy + n, p.dy_f32, p.dy_vec, left, d);
      if (p.z) {
        float z[8];
        ld8<E>(p.z, m * p.ldz + n, false, p.z_vec, left, z);
        slope8(d, z, p.act);  // (beyond `left` both are zero)
      }
      if (p.dz) st8<E>(p.dz, m * p.lddz + n, false, true, 8, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += d[j];
    }
  }
  if (!p.sums) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) lds[threadIdx.x * 9 + j] = sum[j];
  __syncthreads();
  for (int i = threadIdx.x; i < slab; i += 256) {
    const int col = int(blockIdx.y) * slab + i;
    if (col >= p.N) break;
    float s = 0.f;
    for (int k = 0; k < rows; ++k) s += lds[(k * p.lanes + (i >> 3)) * 9 + (i & 7)];
    p.sums[int64_t(blockIdx.x) * p.N + col] = s;
  }
}

// db[n] = sum of `parts` rows; 32 columns and 8 groups of rows per workgroup, the groups' sums added in order
template <typename E>
__global__ void __launch_bounds__(256) linear_colsum(const float* __restrict__ sums, int parts, int N,
                                                     void* __restrict__ db, int f32) {
  __shared__ float lds[8][32];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int n = int(blockIdx.x) * 32 + c;
  float s = 0.f;
  if (n < N) {
#pragma unroll 8
    for (int k = g; k < parts; k += 8) s += sums[int64_t(k) * N + n];
  }
  lds[g][c] = s;
  __syncthreads();
  if (g == 0 && n < N) {
    for (int k = 1; k < 8; ++k) s += lds[k][c];
    if (f32)
      static_cast<float*>(db)[n] = s;
    else
      static_cast<uint16_t*>(db)[n] = E::down(s);
  }
}

// ---- rows that are not 16-byte aligned, copied with their ends filled with zeros ------
__global__ void __launch_bounds__(256) linear_pack(const uint16_t* __restrict__ src, int64_t ld, int rows, int cols,
                                                   uint16_t* __restrict__ dst, int per_row) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= int64_t(rows) * per_row) return;
  const int64_t r = i / per_row;
  const int c = int(i - r * per_row) * 8;
  union {
    uint4 u;
    uint16_t h[8];
  } w;
#pragma unroll
  for (int j = 0; j < 8; ++j) w.h[j] = c + j < cols ? src[r * ld + c + j] : uint16_t(0);
  *reinterpret_cast<uint4*>(dst + i * 8) = w.u;
}

// ---------------------------------------------------------------------------- host
int pad8(int n) { return (n + 7) / 8 * 8; }
size_t align256(size_t n) { return (n + 255) / 256 * 256; }
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
constexpr int64_t kMaxPitch = int64_t(1) << 22;  // 256 rows' offsets fit 32 bits
bool packed(const void* p, int64_t ld, int cols) {
  return !(aligned(p, 16) && ld % 8 == 0 && cols % 8 == 0 && ld <= kMaxPitch);
}
int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tiles and parts of one product.  128 x 128 where that alone makes three quarters of a workgroup per CU, or where
// r is long enough to be split to it; else 64 x 64, which has four times the workgroups.  r is split while two
// workgroups per CU are not reached and each part keeps 256 values of r.
struct Plan {
  int tile, splits, r_per_split;
  size_t bytes;
};
Plan plan_of(int M, int N, int r) {
  Plan p;
  const int64_t big = div_up(M, 128) * div_up(N, 128), small = div_up(M, 64) * div_up(N, 64);
  p.tile = big >= 192 || (M > 64 && N > 64 && big * (r / 512) >= 192) ? 128 : 64;
  const int forced = env_int("GD_LINEAR_TILE", 0);  // (A/B: 64, 128 or 256)
  if (forced == 64 || forced == 128 || forced >= 255) p.tile = forced;
  const int64_t tiles = p.tile >= 255 ? div_up(M, 256) * div_up(N, 256) : p.tile == 128 ? big : small;
  int64_t s = tiles >= 192 ? 1 : 512 / tiles;
  const int64_t most = r / 256;
  s = s > most ? most : s;
  s = s < 1 ? 1 : s;
  p.r_per_split = int(div_up(div_up(r, s), kR) * kR);
  p.splits = int(div_up(r, p.r_per_split));
  p.bytes = p.splits > 1 ? align256(size_t(p.splits) * M * N * sizeof(float)) : 0;
  return p;
}

template <typename E, bool AC, bool BC>
gd_status product(const Plan& plan, Gemm g, void* part, hipStream_t s) {
  g.splits = plan.splits;
  g.r_per_split = plan.r_per_split;
  g.part = static_cast<float*>(part);
  const int tile = plan.tile == 255 ? 256 : plan.tile;
  g.tiles_m = int(div_up(g.M, tile));
  g.tiles_n = int(div_up(g.N, tile));
  g.group = env_int("GD_LINEAR_GROUP", tile >= 256 ? 4 : 8);
  const int64_t grid = int64_t(g.tiles_m) * g.tiles_n * plan.splits;
  GD_REQUIRE(grid < (int64_t(1) << 31), "linear: grid too large");
  if (plan.tile == 256)
    hipLaunchKernelGGL((linear_gemm256<E, AC, BC>), dim3(unsigned(grid)), dim3(256), 0, s, g);
  else if (plan.tile == 255)
    hipLaunchKernelGGL((linear_gemm<E, 2, 4, 8, 4, 2, AC, BC>), dim3(unsigned(grid)), dim3(512), 0, s, g);
  else if (plan.tile == 128)
    hipLaunchKernelGGL((linear_gemm<E, 2, 2, 4, 4, 2, AC, BC>), dim3(unsigned(grid)), dim3(256), 0, s, g);
  else
    hipLaunchKernelGGL((linear_gemm<E, 2, 2, 2, 2, 3, AC, BC>), dim3(unsigned(grid)), dim3(256), 0, s, g);
  GD_LAUNCH_CHECK("linear_gemm");
  if (plan.splits > 1) {
    const int64_t blocks = div_up(int64_t(g.M) * ((g.N + 7) / 8), 256);
    GD_REQUIRE(blocks < (int64_t(1) << 31), "linear: grid too large");
    hipLaunchKernelGGL(linear_finish<E>, dim3(unsigned(blocks)), dim3(256), 0, s, g.part, plan.splits, g.M, g.N, g.epi);
    GD_LAUNCH_CHECK("linear_finish");
  }
  return GD_OK;
}

// an operand's rows: as they are, or packed into the workspace
struct Rows {
  const uint16_t* p;
  int64_t ld;
  int cols;  // readable, a multiple of 8
};
gd_status rows_of(const void* p, int64_t ld, int rows, int cols, char** ws, Rows* out, hipStream_t s) {
  if (!packed(p, ld, cols)) {
    *out = {static_cast<const uint16_t*>(p), ld, cols};
    return GD_OK;
  }
  const int per_row = pad8(cols) / 8;
  const int64_t blocks = div_up(int64_t(rows) * per_row, 256);
  GD_REQUIRE(blocks < (int64_t(1) << 31), "linear: grid too large");
  uint16_t* dst = reinterpret_cast<uint16_t*>(*ws);
  *ws += align256(size_t(rows) * per_row * 16);
  if (rows > 0) {
    hipLaunchKernelGGL(linear_pack, dim3(unsigned(blocks)), dim3(256), 0, s, static_cast<const uint16_t*>(p), ld, rows,
                       cols, dst, per_row);
    GD_LAUNCH_CHECK("linear_pack");
  }
  *out = {dst, pad8(cols), pad8(cols)};
  return GD_OK;
}
size_t rows_bytes(bool pack, int rows, int cols) { return pack ? align256(size_t(rows) * pad8(cols) * 2) : 0; }

Epi plain_epi(void* y, bool f32, int64_t ldy) {
  Epi e = {};
  e.y = y;
  e.y_f32 = f32;
  e.ldy = ldy;
  e.y_vec = aligned(y, 16) && ldy % (f32 ? 4 : 8) == 0;
  return e;
}

// workgroups along the rows of linear_dact: about 1024 in all, each of at least 32 rows per lane group
struct DactPlan {
  int lanes, slabs, blocks;
  int64_t rows;
};
DactPlan dact_plan(int M, int N) {
  DactPlan d;
  d.lanes = 64;
  while (d.lanes > 1 && d.lanes / 2 * 8 >= N) d.lanes /= 2;
  d.slabs = int(div_up(N, 8 * d.lanes));
  const int64_t group = 256 / d.lanes;
  int64_t rows = div_up(M, div_up(1024, d.slabs));
  rows = div_up(rows < 4 * group ? 4 * group : rows, group) * group;
  d.rows = rows;
  d.blocks = int(div_up(M, rows));
  return d;
}

#define GD_TRY(expr)                     \
  do {                                   \
    const gd_status _s = (expr);         \
    if (_s != GD_OK) return _s;          \
  } while (0)

gd_status check_shape(int dtype, int act, int M, int K, int N) {
  GD_REQUIRE(dtype == GD_BF16 || dtype == GD_F16, "linear: bf16 or fp16 operands");
  GD_REQUIRE(act >= kNone && act <= kSilu, "linear: activation %d", act);
  GD_REQUIRE(M >= 0 && K > 0 && N > 0, "linear: M=%d K=%d N=%d", M, K, N);
  // (tile origins and chunk ends stay in int; features are a row's pitch)
  GD_REQUIRE(M <= (1 << 30) && K <= kMaxPitch && N <= kMaxPitch, "linear: M=%d K=%d N=%d (K, N up to 2^22)", M, K, N);
  return GD_OK;
}

template <typename E>
gd_status forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int act, const void* res,
                  int res_dtype, int64_t ldr, int M, int K, int N, void* y, int y_dtype, int64_t ldy, void* z,
                  int64_t ldz, char* ws, hipStream_t s) {
  Rows rx, rw;
  GD_TRY(rows_of(x, ldx, M, K, &ws, &rx, s));
  GD_TRY(rows_of(w, ldw, N, K, &ws, &rw, s));
  Gemm g = {};
  g.a = rx.p;
  g.lda = rx.ld;
  g.b = rw.p;
  g.ldb = rw.ld;
  g.M = M;
  g.N = N;
  g.ra = rx.cols;
  g.rb = rw.cols;
  g.epi = plain_epi(y, y_dtype == GD_F32, ldy);
  g.epi.bias = static_cast<const uint16_t*>(bias);
  g.epi.bias_vec = aligned(bias, 16);
  g.epi.act = act;
  g.epi.res = res;
  g.epi.res_f32 = res_dtype == GD_F32;
  g.epi.ldr = ldr;
  g.epi.res_vec = aligned(res, 16) && ldr % (g.epi.res_f32 ? 4 : 8) == 0;
  g.epi.z = static_cast<uint16_t*>(z);
  g.epi.ldz = ldz;
  return product<E, false, false>(plan_of(M, N, rx.cols), g, ws, s);
}

template <typename E>
gd_status backward(int act, const void* dy, int dy_dtype, int64_t lddy, const void* z, int64_t ldz, const void* x,
                   int64_t ldx, const void* w, int64_t ldw, int M, int K, int N, void* dx, int dx_dtype,
                   int64_t lddx, void* dw, void* db, int param_dtype, char* ws, hipStream_t s) {
  const int n8 = pad8(N);
  Rows rz = {static_cast<const uint16_t*>(dy), lddy, N};
  const bool make = act != kNone || dy_dtype == GD_F32 || packed(dy, lddy, N);
  if (make && (dx || dw)) {
    rz = {reinterpret_cast<uint16_t*>(ws), n8, n8};
    ws += align256(size_t(M) * n8 * 2);
  }
  if (db || (make && (dx || dw))) {
    const DactPlan d = dact_plan(M, N);
    Dact a = {};
    a.dy = dy;
    a.lddy = lddy;
    a.dy_f32 = dy_dtype == GD_F32;
    a.dy_vec = aligned(dy, 16) && lddy % (a.dy_f32 ? 4 : 8) == 0;
    a.z = act == kNone ? nullptr : static_cast<const uint16_t*>(z);
    a.ldz = ldz;
    a.z_vec = aligned(z, 16) && ldz % 8 == 0;
    a.act = act;
    a.dz = make && (dx || dw) ? const_cast<uint16_t*>(rz.p) : nullptr;
    a.lddz = n8;
    a.M = M;
    a.N = N;
    a.rows = d.rows;
    a.lanes = d.lanes;
    if (db) {
      a.sums = reinterpret_cast<float*>(ws);
      ws += align256(size_t(d.blocks) * N * sizeof(float));
    }
    hipLaunchKernelGGL(linear_dact<E>, dim3(d.blocks, d.slabs), dim3(256), 0, s, a);
    GD_LAUNCH_CHECK("linear_dact");
    if (db) {
      hipLaunchKernelGGL(linear_colsum<E>, dim3(unsigned(div_up(N, 32))), dim3(256), 0, s, a.sums, d.blocks, N,
                         db, int(param_dtype == GD_F32));
      GD_LAUNCH_CHECK("linear_colsum");
    }
  }
  if (dx) {
    Rows rw;
    GD_TRY(rows_of(w, ldw, N, K, &ws, &rw, s));
    Gemm g = {};
    g.a = rz.p;
    g.lda = rz.ld;
    g.ra = rz.cols;
    g.b = rw.p;
    g.ldb = rw.ld;
    g.rb = N;
    g.cb = rw.cols;
    g.M = M;
    g.N = K;
    g.epi = plain_epi(dx, dx_dtype == GD_F32, lddx);
    const Plan p = plan_of(M, K, n8);
    GD_TRY((product<E, false, true>(p, g, ws, s)));
    ws += p.bytes;
  }
  if (dw) {
    Rows rx;
    GD_TRY(rows_of(x, ldx, M, K, &ws, &rx, s));
    Gemm g = {};
    g.a = rz.p;
    g.lda = rz.ld;
    g.ca = rz.cols;
    g.b = rx.p;
    g.ldb = rx.ld;
    g.cb = rx.cols;
    g.ra = g.rb = M;
    g.M = N;
    g.N = K;
    g.epi = plain_epi(dw, param_dtype == GD_F32, K);
    GD_TRY((product<E, true, true>(plan_of(N, K, M), g, ws, s)));
  }
  return GD_OK;
}

size_t forward_bytes(bool pack_x, bool pack_w, int M, int K, int N) {
  return rows_bytes(pack_x, M, K) + rows_bytes(pack_w, N, K) + plan_of(M, N, pad8(K)).bytes;
}

size_t backward_bytes(int M, int K, int N, bool dx, bool dw, bool db, bool pack_x, bool pack_w) {
  const int n8 = pad8(N);
  size_t b = dx || dw ? align256(size_t(M) * n8 * 2) : 0;
  if (db) b += align256(size_t(dact_plan(M, N).blocks) * N * sizeof(float));
  if (dx) b += rows_bytes(pack_w, N, K) + plan_of(M, K, n8).bytes;
  if (dw) b += rows_bytes(pack_x, M, K) + plan_of(N, K, M).bytes;
  return b;
}

}  // namespace
}  // namespace gd

using namespace gd;

extern "C" size_t gd_linear_forward_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int M,
                                                    int K, int N) {
  if (M <= 0 || K <= 0 || N <= 0) return 0;
  return forward_bytes(packed(x, ldx, K), packed(w, ldw, K), M, K, N);
}

extern "C" gd_status gd_linear_forward(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw,
                                       const void* bias, int act, const void* residual, int residual_dtype,
                                       int64_t ldr, int M, int K, int N, void* y, int y_dtype, int64_t ldy, void* z,
                                       int64_t ldz, void* workspace, size_t workspace_bytes, gd_stream_t stream) {
  GD_TRY(check_shape(dtype, act, M, K, N));
  if (M == 0) return GD_OK;
  GD_REQUIRE(x && w && y && ldx >= K && ldw >= K && ldy >= N, "linear: null pointer or short rows");
  GD_REQUIRE(aligned(x, 2) && aligned(w, 2) && aligned(bias, 2), "linear: misaligned operands");
  GD_REQUIRE(!residual || (ldr >= N && (residual_dtype == dtype || residual_dtype == GD_F32)),
             "linear: the residual is fp32 or of the operands' type");
  GD_REQUIRE(y_dtype == (residual ? residual_dtype : dtype), "linear: y has the residual's type, without one x's");
  GD_REQUIRE(aligned(y, y_dtype == GD_F32 ? 4 : 2) && aligned(residual, residual_dtype == GD_F32 ? 4 : 2),
             "linear: misaligned y or residual");
  GD_REQUIRE(!z || (aligned(z, 16) && ldz % 8 == 0 && ldz >= pad8(N)), "linear: z has rows padded to 8 values");
  const size_t want = forward_bytes(packed(x, ldx, K), packed(w, ldw, K), M, K, N);
  GD_REQUIRE(workspace_bytes >= want && (want == 0 || (workspace && aligned(workspace, 16))),
             "linear: workspace of %zu bytes, %zu wanted", workspace_bytes, want);
  char* ws = static_cast<char*>(workspace);
  hipStream_t s = as_hip(stream);
  return dtype == GD_BF16 ? forward<Bf16>(x, ldx, w, ldw, bias, act, residual, residual_dtype, ldr, M, K, N, y, y_dtype,
                                          ldy, z, ldz, ws, s)
                          : forward<Fp16>(x, ldx, w, ldw, bias, act, residual, residual_dtype, ldr, M, K, N, y, y_dtype,
                                          ldy, z, ldz, ws, s);
}

extern "C" size_t gd_linear_backward_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int M,
                                                     int K, int N, int dx, int dw, int db) {
  if (M <= 0 || K <= 0 || N <= 0) return 0;
  return backward_bytes(M, K, N, dx, dw, db, packed(x, ldx, K), packed(w, ldw, K));
}

extern "C" gd_status gd_linear_backward(int dtype, int act, const void* dy, int dy_dtype, int64_t lddy, const void* z,
                                        int64_t ldz, const void* x, int64_t ldx, const void* w, int64_t ldw, int M,
                                        int K, int N, void* dx, int dx_dtype, int64_t lddx, void* dw, void* db,
                                        int param_dtype, void* workspace, size_t workspace_bytes,
                                        gd_stream_t stream) {
  GD_TRY(check_shape(dtype, act, M, K, N));
  GD_REQUIRE(M > 0, "linear: gradients of no rows");
  GD_REQUIRE(dy && x && w && lddy >= N && ldx >= K && ldw >= K && (!dx || lddx >= K), "linear: null pointer or short rows");
  GD_REQUIRE(dy_dtype == dtype || dy_dtype == GD_F32, "linear: dy is fp32 or of the operands' type");
  GD_REQUIRE((dx_dtype == dtype || dx_dtype == GD_F32) && (param_dtype == dtype || param_dtype == GD_F32),
             "linear: gradients are fp32 or of the operands' type");
  GD_REQUIRE(act == kNone || (z && ldz >= N), "linear: the activation's slope needs z");
  GD_REQUIRE(aligned(dy, dy_dtype == GD_F32 ? 4 : 2) && aligned(z, 2) && aligned(x, 2) && aligned(w, 2) &&
                 aligned(dx, dx_dtype == GD_F32 ? 4 : 2) && aligned(dw, param_dtype == GD_F32 ? 4 : 2) &&
                 aligned(db, param_dtype == GD_F32 ? 4 : 2),
             "linear: misaligned operands");
  const size_t want = backward_bytes(M, K, N, dx, dw, db, packed(x, ldx, K), packed(w, ldw, K));
  GD_REQUIRE(workspace_bytes >= want && (want == 0 || (workspace && aligned(workspace, 16))),
             "linear: workspace of %zu bytes, %zu wanted", workspace_bytes, want);
  GD_REQUIRE(dact_plan(M, N).slabs < 65536, "linear: N=%d", N);
  char* ws = static_cast<char*>(workspace);
  hipStream_t s = as_hip(stream);
  return dtype == GD_BF16 ? backward<Bf16>(act, dy, dy_dtype, lddy, z, ldz, x, ldx, w, ldw, M, K, N, dx, dx_dtype, lddx,
                                           dw, db, param_dtype, ws, s)
                          : backward<Fp16>(act, dy, dy_dtype, lddy, z, ldz, x, ldx, w, ldw, M, K, N, dx, dx_dtype, lddx,
                                           dw, db, param_dtype, ws, s);
}
