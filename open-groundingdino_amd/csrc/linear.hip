// A linear layer with its epilogue, and its gradients, for gfx950:
//
//   z = x W^T + b     y = act(z) + r          x [M, K], W [N, K], bf16 / fp16
//   dz = dy * act'(z)     dx = dz W     dW = dz^T x     db = sum_m dz     (dr = dy)
//
// All three products are C[m][n] = sum_r A(m, r) B(n, r), whose operands lie in
// memory either with r contiguous ("rows": x, W, dz in the forward and dx) or with
// m / n contiguous ("columns": W in dx, dz and x in dW).  `plan_of` chooses the tile:
//   linear_gemm      64 x 64 and 128 x 128, any layout and edge; dW, small and ragged layers
//   linear_stream    128 x 128, workgroups that go from tile to tile; layers and dx of whole pieces
//   linear_gemm256   256 x 256; large products, bound by the LDS that feeds the matrix cores
//   linear_dz_dx     the activation's slope and dx in one, where memory is what costs
// Products of 16-bit values are exact in fp32 and the accumulators are fp32
// matrix-core registers; bias, activation and residual are applied to them in
// fp32 and the result is rounded once.  The backward rounds dz to 16 bits, as the
// matrix instructions take it, and needs act'(z): the forward writes z rounded to
// 16 bits beside y (for ReLU without a residual y itself tells where z <= 0).
//
// Where the output has too few tiles to fill 256 CUs the sum over r is split: the
// parts go to a workspace in fp32 and a finishing kernel adds them in a fixed
// order and applies the epilogue.  There are no atomics: results repeat bit
// by bit.
#include "gd_common.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace gd {
namespace {

enum Act : int { kNone = 0, kRelu = 1, kGelu = 2, kGeluTanh = 3, kSilu = 4 };

typedef short gd_i16x8 __attribute__((ext_vector_type(8)));
typedef short gd_i16x4 __attribute__((ext_vector_type(4)));
typedef float gd_f32x2 __attribute__((ext_vector_type(2)));
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

#ifndef GD_STORE_NT
#define GD_STORE_NT(value, to) __builtin_nontemporal_store(value, to)
#define GD_LOAD_NT(from) __builtin_nontemporal_load(from)
#endif

// the two 16-bit types
struct Bf16 {
  static __device__ __forceinline__ float up(uint16_t h) { return bf16_to_f32(h); }
  static __device__ __forceinline__ uint16_t down(float f) { return f32_to_bf16(f); }
  static __device__ __forceinline__ uint32_t down2(float a, float b) {  // (one instruction)
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(gd_f32x2{a, b}, bf16x2));
  }
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
  static __device__ __forceinline__ uint32_t down2(float a, float b) { return down(a) | uint32_t(down(b)) << 16; }
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
// sigmoid(2 c (z + a z^3)), which is (1 + tanh(c (z + a z^3))) / 2, as 1 / (1 + 2^(z (p + q z^2)))
__device__ __forceinline__ float tanh_gate(float z) {
  constexpr float p = -2.f * kTanhC * 1.4426950408889634f, q = p * kTanhA;
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * (p + q * (z * z))));
}

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
    case kGeluTanh:
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= tanh_gate(v[j]);
      break;
    case kSilu:
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= sigmoid(v[j]);
      break;
    default: break;
  }
}

// z as a factor of a term that vanishes far from zero: an infinite one (in fp16 any beyond 65504, whose layer may well be
// finite with an fp32 residual) would make it inf * 0.  From 128 on the smooth slopes are 0 and 1 in fp32; NaN stays, by
// the other factors.
__device__ __forceinline__ float slope_arg(float z) { return fminf(fmaxf(z, -128.f), 128.f); }

// d[j] *= act'(z[j])
__device__ __forceinline__ void slope8(float d[8], const float z[8], int act) {
  switch (act) {
    case kRelu:
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = z[j] <= 0.f ? 0.f : d[j];  // (at NaN, as the forward keeps it, dy goes on)
      break;
    case kGelu:
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float bell;
        const float c = normal_cdf(z[j], &bell);
        d[j] *= c + slope_arg(z[j]) * bell * 0.39894228040143268f;
      }
      break;
    case kGeluTanh:
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = slope_arg(z[j]), q = tanh_gate(z[j]);
        d[j] *= q + 2.f * x * q * (1.f - q) * kTanhC * (1.f + 3.f * kTanhA * x * x);
      }
      break;
    case kSilu:
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = slope_arg(z[j]), q = sigmoid(z[j]);
        d[j] *= q * (1.f + x * (1.f - q));
      }
      break;
    default: break;
  }
}

// 16 bytes of an input that is read once: it leaves the memory-side cache to what is read again (the layer 44446 x 256 ->
// 2048 with its gradients 287 us with plain loads of dy and z, 264 with these, since dz is there when dW reads it;
// with the slope as a kernel of its own 344 and 282)
__device__ __forceinline__ uint4 ld_once(const void* p) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 u = GD_LOAD_NT(static_cast<const u32x4*>(p));
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// ---- 8 consecutive 16-bit or fp32 values, the first `left` of them valid ------
// ONCE: see ld_once
template <typename E, bool ONCE = false>
__device__ __forceinline__ void ld8(const void* p, int64_t at, bool f32, bool vec, int left, float v[8]) {
  if (f32) {
    const float* q = static_cast<const float*>(p) + at;
    if (vec && left >= 8) {
      const uint4* const u = reinterpret_cast<const uint4*>(q);
      const uint4 a = ONCE ? ld_once(u) : u[0], b = ONCE ? ld_once(u + 1) : u[1];
      v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
      v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
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
    w.u = ONCE ? ld_once(q) : *reinterpret_cast<const uint4*>(q);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) w.h[j] = j < left ? q[j] : uint16_t(0);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = E::up(w.h[j]);
}

// 16 bytes of an output: past the caches' ways of lines that are kept (16384 x 512 -> 4096: 112 us with plain stores, 102
// with these; 44446 x 256 -> 2048: 108 and 98).  Measured as a call by itself: what a next layer that reads the output at
// once pays for it is not in these figures.
__device__ __forceinline__ void st_out(void* p, uint4 u) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  GD_STORE_NT((u32x4{u.x, u.y, u.z, u.w}), static_cast<u32x4*>(p));
}

template <typename E>
__device__ __forceinline__ uint4 pack8(const float v[8]) {
  return make_uint4(E::down2(v[0], v[1]), E::down2(v[2], v[3]), E::down2(v[4], v[5]), E::down2(v[6], v[7]));
}

template <typename E, bool NT = true>
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
  if (vec && left >= 8) {
    if (NT)
      st_out(q, pack8<E>(v));
    else
      *reinterpret_cast<uint4*>(q) = pack8<E>(v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) q[j] = E::down(v[j]);
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
__device__ __forceinline__ void epilogue8(const Epi& e, int act, int64_t m, int n, int left, const float b[8],
                                          const float r[8], float v[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] += b[j];
  if (e.z) {
    float z[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = j < left ? v[j] : 0.f;
    st8<E>(e.z, m * e.ldz + n, false, true, 8, z);
  }
  activate8(v, act);
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
__device__ __forceinline__ Tile tile_of(const Gemm& p, int block, int blocks) {
  const int L = xcd_remap(block, blocks);
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
// PAIRS: as Loader's, here for columns: of the two blocks of 32 columns, the one of x0 takes 4 of every 8
template <int X, bool COL, bool PAIRS = false>
__device__ __forceinline__ gd_i16x8 fragment(const uint16_t* img, int x0, int s, int lane) {
  if constexpr (!COL) {
    return *reinterpret_cast<const gd_i16x8*>(img + row_at(x0 + (lane & 15), 4 * s + (lane >> 4)));
  } else {
    const int g = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
    const int ch = PAIRS ? ((x0 >> 3) & ~3) + p : (x0 >> 3) + (p >> 1);
    const int sub = 4 * (PAIRS ? (x0 >> 4) & 1 : p & 1);
    const gd_i16x4 lo = lds_tr(img + col_at<X>(32 * s + 8 * g + q, ch) + sub);
    const gd_i16x4 hi = lds_tr(img + col_at<X>(32 * s + 8 * g + 4 + q, ch) + sub);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// One operand's way into its LDS image of X rows (or columns) by 64 values of r.  A wave instruction moves 64 pieces
// of 16 bytes to consecutive LDS positions, so the swizzle is applied to the source: position pos of a row holds
// its chunk pos ^ swz.  Rows (columns) past the operand's end read its last one instead: their products land in
// outputs that are not stored.
// PAIRS: of 32 rows, those whose products one lane of two blocks holds (4 each) follow each other.
template <int X, bool COL, int WAVES, bool PAIRS = false>
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
        const int row = piece >> 3;
        const int from = PAIRS ? (row & ~31) + 8 * ((row >> 2) & 3) + 4 * ((row >> 4) & 1) + (row & 3) : row;
        const int x = x0 + from < end ? from : end - 1 - x0;
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

// A wave's TM x TN blocks to memory, through its own LDS in TM / GI parts, so that a row leaves in 16-byte pieces of
// neighbouring lanes and the loop over the rows is short code with several rows under way (the accumulators can
// only be addressed by unrolled code).  Pitch 16 TN + 4 floats: 16 rows' float4s, and the reads of 8 neighbouring
// columns, touch all banks once.
template <int TN>
constexpr int store_pitch() { return 16 * TN + 4; }
template <int TN>
constexpr int store_floats(int gi) { return 16 * gi * store_pitch<TN>(); }  // of one wave

// The residual of B rows, asked for before the previous ones are used: it comes from far, and y may be anywhere,
// so the compiler would not move a load before a store.  Without a branch in between: the second half of an fp32
// row is of a 16-bit one the same piece again, and rows past the end are the last one.
template <int B>
struct Residual {
  uint4 a[B], b[B];
  __device__ __forceinline__ void load(const Gemm& p, int m, int step, int n) {
    const char* const from = static_cast<const char*>(p.epi.res);
    const int64_t size = p.epi.res_f32 ? 4 : 2;
#pragma unroll
    for (int h = 0; h < B; ++h) {
      const int row = m + h * step < p.M ? m + h * step : p.M - 1;
      const uint4* q = reinterpret_cast<const uint4*>(from + (row * p.epi.ldr + n) * size);
      a[h] = q[0];
      b[h] = q[p.epi.res_f32 ? 1 : 0];
    }
  }
  template <typename E>
  __device__ __forceinline__ void get(const Gemm& p, int h, float r[8]) const {
    union {
      uint4 u[2];
      uint16_t h16[8];
      float f[8];
    } raw;
    raw.u[0] = a[h];
    raw.u[1] = b[h];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = p.epi.res_f32 ? raw.f[j] : E::up(raw.h16[j]);
  }
};

template <int TN>
constexpr int rows_per_pass() { return 64 / (2 * TN); }  // 2 TN lanes per row
template <int TN, int GI>
constexpr int batch() { return 16 * GI / rows_per_pass<TN>() < 4 ? 16 * GI / rows_per_pass<TN>() : 4; }

// 16 GI rows in LDS, whose corner in the output is m0, n0; a lane keeps its 8 columns.  next: the residual's rows from m0
// on, where `ahead` says that it is loaded this way.
template <typename E, int TN, int GI, int ACT>
__device__ __forceinline__ void store_rows(const Gemm& p, const float* own, Residual<batch<TN, GI>()>& next,
                                           bool ahead, int m0, int n0,
                                           int lane) {
  constexpr int kLanes = 2 * TN, kRows = rows_per_pass<TN>(), kBatch = batch<TN, GI>();
  constexpr int kBatches = 16 * GI / (kRows * kBatch);
  const int col = 8 * (lane % kLanes), n = n0 + col, left = p.N - n < 8 ? p.N - n : 8;
  if (left <= 0) return;
  float bias[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) bias[j] = 0.f;
  if (p.epi.bias) ld8<E>(p.epi.bias, n, false, p.epi.bias_vec, left, bias);
#pragma unroll 1
  for (int b = 0; b < kBatches; ++b) {
    const int row0 = b * kBatch * kRows + lane / kLanes;
    Residual<kBatch> now;
    if (ahead) {
      now = next;
      if (m0 + row0 + kBatch * kRows < p.M) next.load(p, m0 + row0 + kBatch * kRows, kRows, n);
    }
#pragma unroll
    for (int h = 0; h < kBatch; ++h) {
      const int row = row0 + h * kRows, m = m0 + row;
      if (m < p.M) {
        float res[8];
        if (ahead) {
          now.template get<E>(p, h, res);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) res[j] = 0.f;
          if (p.epi.res) ld8<E>(p.epi.res, m * p.epi.ldr + n, p.epi.res_f32, p.epi.res_vec, left, res);
        }
        const float4 u = *reinterpret_cast<const float4*>(own + row * store_pitch<TN>() + col);
        const float4 w = *reinterpret_cast<const float4*>(own + row * store_pitch<TN>() + col + 4);
        float v[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
        epilogue8<E>(p.epi, ACT, m, n, left, bias, res, v);
      }
    }
  }
}

// the same without an epilogue: a gradient, or a part of a split sum
template <typename E, int TN>
__device__ __forceinline__ void store_plain(const Gemm& p, const float* own, int rows, int m0, int n0, int split, int lane) {
  constexpr int kLanes = 2 * TN, kRows = 64 / kLanes;
  const int col = 8 * (lane % kLanes), n = n0 + col, left = p.N - n < 8 ? p.N - n : 8;
  if (left <= 0) return;
  const bool whole = p.splits == 1;
  void* const to = whole ? p.epi.y : static_cast<void*>(p.part + int64_t(split) * p.M * p.N);
  const int64_t ld = whole ? p.epi.ldy : p.N;
  const bool f32 = !whole || p.epi.y_f32, vec = whole ? p.epi.y_vec : (p.N & 3) == 0;
  const int end = p.M - m0 < rows ? p.M - m0 : rows;
#pragma unroll 4
  for (int row = lane / kLanes; row < end; row += kRows) {
    const float4 u = *reinterpret_cast<const float4*>(own + row * store_pitch<TN>() + col);
    const float4 w = *reinterpret_cast<const float4*>(own + row * store_pitch<TN>() + col + 4);
    const float v[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
    st8<E>(to, (m0 + row) * ld + n, f32, vec, left, v);
  }
}

// own: the wave's LDS, its part of the images, which every wave has read
template <typename E, int TM, int TN, int GI, bool LAYER>
__device__ __forceinline__ void store_tile(const Gemm& p, const gd_f32x4 (&acc)[TM][TN], float* own, int m0, int n0,
                                           int split, int lane) {
  static_assert(TM % GI == 0, "whole parts");
  Residual<batch<TN, GI>()> next;
  // (uniform: whole pieces of 8 columns, so that no lane needs another path)
  const bool ahead = LAYER && p.splits == 1 && p.epi.res && p.epi.res_vec && (p.N & 7) == 0;
  if (ahead) {
    const int n = n0 + 8 * (lane % (2 * TN));
    if (n < p.N && m0 < p.M) next.load(p, m0 + lane / (2 * TN), rows_per_pass<TN>(), n);
  }
  __syncthreads();
  // (one copy of the rows' code, which is long; the accumulators are picked by comparison)
#pragma unroll 1
  for (int part = 0; part < TM / GI; ++part) {
#pragma unroll
    for (int q = 0; q < TM / GI; ++q)
      if (q == part) {
#pragma unroll
        for (int i = 0; i < GI; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j)
            *reinterpret_cast<gd_f32x4*>(own + (16 * i + (lane & 15)) * store_pitch<TN>() + 16 * j + 4 * (lane >> 4)) =
                acc[q * GI + i][j];
      }
    gd_wave_sync();
    const int m = m0 + 16 * GI * part;
    if (LAYER && p.splits == 1) {
      switch (p.epi.act) {
        case kRelu: store_rows<E, TN, GI, kRelu>(p, own, next, ahead, m, n0, lane); break;
        case kGelu: store_rows<E, TN, GI, kGelu>(p, own, next, ahead, m, n0, lane); break;
        case kGeluTanh: store_rows<E, TN, GI, kGeluTanh>(p, own, next, ahead, m, n0, lane); break;
        case kSilu: store_rows<E, TN, GI, kSilu>(p, own, next, ahead, m, n0, lane); break;
        default: store_rows<E, TN, GI, kNone>(p, own, next, ahead, m, n0, lane); break;
      }
    } else {
      store_plain<E, TN>(p, own, 16 * GI, m, n0, split, lane);
    }
    gd_wave_sync();
  }
}

// WM x WN waves, each of TM x TN blocks of 16 x 16; a ring of ST images, ST - 1 chunks of r in flight.  64 x 64 tiles with 3
// images (48 KB, three workgroups per CU): 900 x 256 x 256 4.6 us, latency; 128 x 128 with 2 (64 KB, two): dW of 44446 x
// 256 x 2048 54 us (870 TFLOP/s), 16384 x 4096 x 4096 485 us (1.13 PFLOP/s), both by LDS, 96 KB in and out per chunk and
// 512 products' worth of cycles.  Chunks of 32 values double the requests to L2 and were slower.
template <typename E, int WM, int WN, int TM, int TN, int ST, bool AC, bool BC>
__global__ void __launch_bounds__(64 * WM * WN) linear_gemm(const Gemm p) {
  constexpr int kWaves = WM * WN, BM = 16 * WM * TM, BN = 16 * WN * TN;
  constexpr int kStage = (BM + BN) * kR;
  constexpr int kOwn = store_floats<TN>(2);
  static_assert(kWaves * kOwn * 2 <= ST * kStage, "the output's way through LDS fits");
  __shared__ __attribute__((aligned(16))) uint16_t lds[ST * kStage];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / WN, wn = wave % WN;
  const Tile t = tile_of(p, int(blockIdx.x), int(gridDim.x));
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

  store_tile<E, TM, TN, 2, !AC && !BC>(p, acc, reinterpret_cast<float*>(lds) + wave * kOwn, m0 + 16 * wm * TM,
                                       n0 + 16 * wn * TN, split, lane);
}

// 16 rows from m on: lane (c, g) has two 16-byte pieces of row c, at bytes 16 g and 64 + 16 g of 128 (16-bit output, 64
// columns; pitch `apart` 64) or at 32 g and 32 g + 16 (fp32 output, 32 columns; 16).  Lanes c and c ^ 1 trade one, so that
// an instruction writes whole rows of 128 bytes (64 bytes of twice the rows take twice the time: 199 us against 82
// for 44446 x 256 -> 2048).
__device__ __forceinline__ void write_rows(char* row0, int64_t pitch, int at, int apart, int m, int M, int bytes, int lane,
                                           uint4 first, uint4 second) {
  const bool odd = (lane & 1) != 0;
  const uint4 give = odd ? first : second;
  uint4 take;
  take.x = __float_as_uint(dpp<DPP_XOR1>(__uint_as_float(give.x)));
  take.y = __float_as_uint(dpp<DPP_XOR1>(__uint_as_float(give.y)));
  take.z = __float_as_uint(dpp<DPP_XOR1>(__uint_as_float(give.z)));
  take.w = __float_as_uint(dpp<DPP_XOR1>(__uint_as_float(give.w)));
  m += lane & 14;
  at += odd ? apart : 0;
  char* const to = row0 + m * pitch + at;
  if (m < M && at < bytes) st_out(to, odd ? take : first);
  if (m + 1 < M && at < bytes) st_out(to + pitch, odd ? second : take);
}
// 64 columns from n on, of 16 bits: the pieces of columns 8 g and 32 + 8 g
__device__ __forceinline__ void write16(uint16_t* to, int64_t ld, int m, int n, int M, int N, int lane, uint4 first,
                                        uint4 second) {
  write_rows(reinterpret_cast<char*>(to), 2 * ld, 2 * n + 16 * (lane >> 4), 64, m, M, 2 * N, lane, first, second);
}
// 32 columns from n on, fp32: the pieces of columns 8 g and 8 g + 4
__device__ __forceinline__ void write32(float* to, int64_t ld, int m, int n, int M, int N, int lane, const float v[8]) {
  const uint4 first = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  const uint4 second = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
  write_rows(reinterpret_cast<char*>(to), 4 * ld, 4 * n + 32 * (lane >> 4), 16, m, M, 4 * N, lane, first, second);
}

// A wave's T x 8 blocks (of operands read as PAIRS) with their epilogue, straight from the registers, one row of blocks after
// the other (the accumulators are picked by comparison); the residual is asked for a row of blocks ahead.
template <typename E, int T>
__device__ __forceinline__ void store_direct(const Gemm& p, const gd_f32x4 (&acc)[T][8], int m0, int n0, int lane) {
  const int c = lane & 15, g = lane >> 4;
  uint4 bias[4], res[4][2];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const int n = n0 + 32 * h + 8 * g;
    bias[h] = p.epi.bias ? *reinterpret_cast<const uint4*>(p.epi.bias + (n < p.N ? n : p.N - 8)) : make_uint4(0, 0, 0, 0);
  }
  const char* const from = static_cast<const char*>(p.epi.res);
  const int64_t size = p.epi.res_f32 ? 4 : 2;
  auto ask = [&](int i) {
    const int m = m0 + 16 * i + c;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int n = n0 + 32 * h + 8 * g;
      const uint4* const r =
          reinterpret_cast<const uint4*>(from + ((m < p.M ? m : p.M - 1) * p.epi.ldr + (n < p.N ? n : p.N - 8)) * size);
      res[h][0] = r[0];
      res[h][1] = r[p.epi.res_f32 ? 1 : 0];
    }
  };
  if (from) ask(0);
#pragma unroll 1
  for (int i = 0; i < T; ++i) {
    float x[4][8];
#pragma unroll
    for (int q = 0; q < T; ++q)
      if (q == i) {
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
          for (int j = 0; j < 8; ++j) x[h][j] = acc[q][2 * h + (j >> 2)][j & 3];
      }
    uint4 z[4], y[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      union {
        uint4 u[2];
        uint16_t h16[16];
        float f[8];
      } b, r;
      b.u[0] = bias[h];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[h][j] += E::up(b.h16[j]);
      if (p.epi.z) z[h] = pack8<E>(x[h]);
      activate8(x[h], p.epi.act);
      if (from) {
        r.u[0] = res[h][0];
        r.u[1] = res[h][1];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[h][j] += p.epi.res_f32 ? r.f[j] : E::up(r.h16[j]);
      }
    }
    if (from) ask(i + 1 < T ? i + 1 : i);
    const int m = m0 + 16 * i;
    if (p.epi.z) {
      write16(p.epi.z, p.epi.ldz, m, n0, p.M, p.N, lane, z[0], z[1]);
      write16(p.epi.z, p.epi.ldz, m, n0 + 64, p.M, p.N, lane, z[2], z[3]);
    }
    if (p.epi.y_f32) {
#pragma unroll
      for (int h = 0; h < 4; ++h)
        write32(static_cast<float*>(p.epi.y), p.epi.ldy, m, n0 + 32 * h, p.M, p.N, lane, x[h]);
    } else {
#pragma unroll
      for (int h = 0; h < 4; ++h) y[h] = pack8<E>(x[h]);
      write16(static_cast<uint16_t*>(p.epi.y), p.epi.ldy, m, n0, p.M, p.N, lane, y[0], y[1]);
      write16(static_cast<uint16_t*>(p.epi.y), p.epi.ldy, m, n0 + 64, p.M, p.N, lane, y[2], y[3]);
    }
  }
}

// 256 x 256 tiles of 4 waves, 128 x 128 each, one per SIMD: the largest wave tile its 512 registers allow, since LDS is
// what the matrix cores compete for (128 KB are read and 64 KB written per chunk of 64 values of r; 8 waves of 128 x
// 64 read 192 KB and wait for each other: 444 us at 16384 x 4096 x 4096, the products and reads alone 286, the
// loads alone 299).  A phase multiplies half a chunk whose fragments are in registers; between its products the next
// half's fragments are read and the loads issued, so nothing waits but for the barrier in the middle of a chunk.
// LDS holds a ring of 5 images of one operand each, in the order A0 B0 A1 B1 A2 ...: A of chunk k + 2 is loaded in the
// first phase of chunk k, to the image that B of chunk k - 1 left, B of chunk k + 2 in the second, to that of A of
// chunk k: one load per 8 products, all the time.
// DIRECT, a layer with whole pieces (`streams`): the output leaves straight from the registers (16384 x 4096 x 4096 with
// tanh-GELU and residual: 449 us, through LDS 476; a gradient, without an epilogue, is as fast through LDS, and going on
// to a next tile whose chunks are asked for before the output brought nothing, 450).
template <typename E, bool AC, bool BC, bool DIRECT>
__global__ void __launch_bounds__(256, 1) linear_gemm256(const Gemm p) {
  constexpr int T = 8, kWaves = 4, BX = 256, kImg = BX * kR, kRing = 5;
  constexpr int kOwn = store_floats<T>(4);
  static_assert(kWaves * kOwn * 2 <= kRing * kImg, "the output's way through LDS fits");
  __shared__ __attribute__((aligned(16))) uint16_t lds[kRing * kImg];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave >> 1, wn = wave & 1;
  const Tile t = tile_of(p, int(blockIdx.x), int(gridDim.x));
  const int m0 = t.m * BX, n0 = t.n * BX, split = t.split;
  const int r_end = p.ra > p.rb ? p.ra : p.rb, r_both = p.ra < p.rb ? p.ra : p.rb;
  const int rb0 = split * p.r_per_split;
  const int re = rb0 + p.r_per_split < r_end ? rb0 + p.r_per_split : r_end;
  const int rf = re < r_both ? re : r_both;
  const int nfull = rf > rb0 ? (rf - rb0) / kR : 0;

  using Load = Loader<BX, AC, kWaves>;  // 8 instructions a wave and image
  Load la(p.a, p.lda, m0, p.M, p.ca, rb0, wave, lane);
  Loader<BX, BC, kWaves, DIRECT> lb(p.b, p.ldb, n0, p.N, p.cb, rb0, wave, lane);
  static_assert(!DIRECT || (!AC && !BC), "a layer");
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
    if (nfull > 1)
      gd_wait_vmcnt(2 * T);
    else
      gd_wait_vmcnt(0);
    gd_raw_barrier();
#pragma unroll
    for (int i = 0; i < T; ++i) read1(f0, 0, 0, i);
    // one chunk; q: its A's image.  MORE: chunk k + 2 exists
    auto chunk = [&](int k, int q, auto MORE) {
      constexpr bool kMore = decltype(MORE)::value;
      const uint32_t to_a = uint32_t(wrap(q + 4)) * (2 * kImg), to_b = uint32_t(q) * (2 * kImg);
#pragma unroll
      for (int i = 0; i < T; ++i) {
        read1(f1, q, 1, i);
        if (kMore) la.issue(lds, to_a, wave, i);
        multiply1(f0, i);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (kMore)
        gd_wait_vmcnt(T);  // chunk k + 1 has landed, A of chunk k + 2 may be under way
      else
        gd_wait_vmcnt(0);
      gd_lds_barrier();  // and chunk k has been read
      const int qn = k + 1 < nfull ? wrap(q + 2) : q;  // (the last chunk's is read again, for nothing)
#pragma unroll
      for (int i = 0; i < T; ++i) {
        read1(f0, qn, 0, i);
        if (kMore) lb.issue(lds, to_b, wave, i);
        multiply1(f1, i);
        __builtin_amdgcn_sched_barrier(0);
      }
      la.base += la.step;
      lb.base += lb.step;
    };
    int k = 0, q = 0;
    for (; k + 2 < nfull; ++k, q = wrap(q + 2)) chunk(k, q, std::true_type());
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
  if constexpr (DIRECT)
    store_direct<E, T>(p, acc, m0 + 16 * wm * T, n0 + 16 * wn * T, lane);
  else
    store_tile<E, T, T, 4, !AC && !BC>(p, acc, reinterpret_cast<float*>(lds) + wave * kOwn, m0 + 16 * wm * T,
                                       n0 + 16 * wn * T, split, lane);
}

// 128 x 128 tiles by workgroups that go from tile to tile: the next tile's first two chunks are asked for before the output
// is stored, straight from the registers (a lane holds 8 consecutive columns of a row), so loads, products and stores
// of the two workgroups of a CU run side by side.  It matters for layers with few features in, whose tiles are short:
// 44446 x 256 -> 2048 with ReLU 82 us (one tile per workgroup and outputs through LDS 98), 33400 x 192 -> 768 21 (30),
// 16384 x 512 -> 4096 84 (99); with many features it is no slower.  For whole pieces only (see `streams`).
template <typename E, bool BC>
__global__ void __launch_bounds__(256, 2) linear_stream(const Gemm p) {
  constexpr int T = 4, kWaves = 4, BX = 128, kStage = 2 * BX * kR;
  __shared__ __attribute__((aligned(16))) uint16_t lds[2 * kStage];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave >> 1, wn = wave & 1, c = lane & 15, g = lane >> 4;
  const int chunks = p.ra / kR, tiles = p.tiles_m * p.tiles_n;
  using LA = Loader<BX, false, kWaves>;
  using LB = Loader<BX, BC, kWaves, !BC>;
  constexpr int kInstr = LA::kInstr + LB::kInstr, kStores = 2 * T;  // of a wave: per chunk; per tile at least
  Tile t = tile_of(p, int(blockIdx.x), tiles);
  LA la(p.a, p.lda, t.m * BX, p.M, p.ca, 0, wave, lane);
  LB lb(p.b, p.ldb, t.n * BX, p.N, p.cb, 0, wave, lane);
  uint32_t now = 0;  // the image of the chunk at hand
  auto issue = [&](uint32_t image) {
    la.issue(lds, image * (2 * kStage), wave);
    lb.issue(lds, image * (2 * kStage) + 2 * BX * kR, wave);
  };
  // the bias of a lane's 2 x 8 columns
  auto bias_of = [&](int n0, uint4 (&b)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = n0 + 64 * wn + 32 * h + 8 * g;
      b[h] = p.epi.bias ? *reinterpret_cast<const uint4*>(p.epi.bias + (n < p.N ? n : p.N - 8)) : make_uint4(0, 0, 0, 0);
    }
  };
  uint4 braw[2];
  issue(0);
  bias_of(t.n * BX, braw);
  issue(1);
  bool stored = false;  // at least kStores stores of this wave follow the chunks under way
  for (int v = int(blockIdx.x); v < tiles; v += int(gridDim.x)) {
    const int m0 = t.m * BX + 64 * wm, n0 = t.n * BX + 64 * wn;
    const bool whole = t.m * BX + BX <= p.M && t.n * BX + BX <= p.N;
    const bool more = v + int(gridDim.x) < tiles;
    gd_f32x4 acc[T][T];
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
      for (int j = 0; j < T; ++j) acc[i][j] = gd_f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < chunks; ++k) {
      if (k == 0) {
        if (stored)
          gd_wait_vmcnt(kInstr + kStores);
        else
          gd_wait_vmcnt(kInstr);
      } else if (k == 1 && stored) {
        gd_wait_vmcnt(kStores);
      } else {
        gd_wait_vmcnt(0);
      }
      gd_lds_barrier();
      if (k + 1 == chunks) {
        if (more) {
          t = tile_of(p, v + int(gridDim.x), tiles);
          la = LA(p.a, p.lda, t.m * BX, p.M, p.ca, 0, wave, lane);
          lb = LB(p.b, p.ldb, t.n * BX, p.N, p.cb, 0, wave, lane);
          issue(now ^ 1);
        }
      } else if (k > 0) {
        issue(now ^ 1);
      }
      const uint16_t* const img = lds + now * kStage;
#pragma unroll
      for (int s = 0; s < kR / 32; ++s) {
        gd_i16x8 fa[T], fb[T];
#pragma unroll
        for (int j = 0; j < T; ++j) fb[j] = fragment<BX, BC, BC>(img + BX * kR, 16 * (wn * T + j), s, lane);
#pragma unroll
        for (int i = 0; i < T; ++i) fa[i] = fragment<BX, false>(img, 16 * (wm * T + i), s, lane);
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
          for (int j = 0; j < T; ++j) acc[i][j] = E::mma(fb[j], fa[i], acc[i][j]);
      }
      now ^= 1;
    }
    union {
      uint4 u[2];
      uint16_t h[16];
    } bias;
    bias.u[0] = braw[0];
    bias.u[1] = braw[1];
    uint4 res[2 * T][2];
    if (p.epi.res) {
      const char* const from = static_cast<const char*>(p.epi.res);
      const int64_t size = p.epi.res_f32 ? 4 : 2;
#pragma unroll
      for (int q = 0; q < 2 * T; ++q) {
        const int m = m0 + 16 * (q >> 1) + c, n = n0 + 32 * (q & 1) + 8 * g;
        const uint4* const r = reinterpret_cast<const uint4*>(
            from + ((m < p.M ? m : p.M - 1) * p.epi.ldr + (n < p.N ? n : p.N - 8)) * size);
        res[q][0] = r[0];
        res[q][1] = r[p.epi.res_f32 ? 1 : 0];
      }
    }
    gd_lds_barrier();  // the last chunk has been read
    if (more) {
      bias_of(t.n * BX, braw);
      issue(now ^ 1);
    }
    auto store = [&](auto ACT) {
#pragma unroll
      for (int i = 0; i < T; ++i) {
        uint4 y[2], z[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = acc[i][2 * h + (j >> 2)][j & 3] + E::up(bias.h[8 * h + j]);
          if (p.epi.z) z[h] = pack8<E>(x);
          activate8(x, decltype(ACT)::value);
          if (p.epi.res) {
            union {
              uint4 u[2];
              uint16_t h16[8];
              float f[8];
            } raw;
            raw.u[0] = res[2 * i + h][0];
            raw.u[1] = res[2 * i + h][1];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] += p.epi.res_f32 ? raw.f[j] : E::up(raw.h16[j]);
          }
          if (p.epi.y_f32)
            write32(static_cast<float*>(p.epi.y), p.epi.ldy, m0 + 16 * i, n0 + 32 * h, p.M, p.N, lane, x);
          else
            y[h] = pack8<E>(x);
        }
        if (p.epi.z) write16(p.epi.z, p.epi.ldz, m0 + 16 * i, n0, p.M, p.N, lane, z[0], z[1]);
        if (!p.epi.y_f32) write16(static_cast<uint16_t*>(p.epi.y), p.epi.ldy, m0 + 16 * i, n0, p.M, p.N, lane, y[0], y[1]);
      }
    };
    switch (p.epi.act) {
      case kRelu: store(std::integral_constant<int, kRelu>()); break;
      case kGelu: store(std::integral_constant<int, kGelu>()); break;
      case kGeluTanh: store(std::integral_constant<int, kGeluTanh>()); break;
      case kSilu: store(std::integral_constant<int, kSilu>()); break;
      default: store(std::integral_constant<int, kNone>()); break;
    }
    stored = whole;
  }
}

// db[n] = sum of `parts` rows of column sums; 8 columns and 32 groups of rows per workgroup, the groups' sums added in order
struct Join {
  const float* sums;  // [parts][N]
  void* db;
  int parts, N, f32;
  int first;          // the first workgroup that does this (of linear_finish)
};
constexpr int kJoinColumns = 8;
template <typename E>
__device__ __forceinline__ void join_sums(const Join& j, int block) {
  constexpr int kGroups = 256 / kJoinColumns;
  __shared__ float lds[kGroups][kJoinColumns];
  const int c = threadIdx.x % kJoinColumns, g = threadIdx.x / kJoinColumns;
  const int n = block * kJoinColumns + c;
  float s = 0.f;
  if (n < j.N) {
#pragma unroll 8
    for (int k = g; k < j.parts; k += kGroups) s += j.sums[int64_t(k) * j.N + n];
  }
  lds[g][c] = s;
  __syncthreads();
  if (g == 0 && n < j.N) {
    for (int k = 1; k < kGroups; ++k) s += lds[k][c];
    if (j.f32)
      static_cast<float*>(j.db)[n] = s;
    else
      static_cast<uint16_t*>(j.db)[n] = E::down(s);
  }
}
template <typename E>
__global__ void __launch_bounds__(256) linear_colsum(const Join j) {
  join_sums<E>(j, int(blockIdx.x));
}

// the parts added in order, then the epilogue; a thread per 8 columns.  Further workgroups join column sums (a launch less)
template <typename E>
__global__ void __launch_bounds__(256) linear_finish(const float* __restrict__ part, int splits, int M, int N, Epi epi, Join join) {
  if (int(blockIdx.x) >= join.first) {
    join_sums<E>(join, int(blockIdx.x) - join.first);
    return;
  }
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
  epilogue8<E>(epi, epi.act, m, n, left, b, r, v);
}

// ---- dz = dy * act'(z), and parts of its column sums -------------------------------
// A stream: 44446 x 2048 with ReLU, 546 MB, 108 us (5.1 TB/s).  dz is stored plainly: past the caches it costs the products
// that read it next more than it saves here (the layer with its gradients 352 us instead of 342).
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
    // (4 rows are loaded before the first is stored, which the compiler could not do by itself: dz may be anywhere)
    constexpr int kRowsAhead = 4;
    for (int64_t m = begin + at; m < end; m += kRowsAhead * rows) {
      float d[kRowsAhead][8], z[kRowsAhead][8];
#pragma unroll
      for (int h = 0; h < kRowsAhead; ++h) {
        const int64_t row = m + h * rows < end ? m + h * rows : end - 1;
        ld8<E, true>(p.dy, row * p.lddy + n, p.dy_f32, p.dy_vec, left, d[h]);
        if (p.z) ld8<E, true>(p.z, row * p.ldz + n, false, p.z_vec, left, z[h]);
      }
#pragma unroll
      for (int h = 0; h < kRowsAhead; ++h) {
        const int64_t row = m + h * rows;
        if (row < end) {
          if (p.z) slope8(d[h], z[h], p.act);  // (beyond `left` both are zero)
          if (p.dz) st8<E, false>(p.dz, row * p.lddz + n, false, true, 8, d[h]);
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[j] += d[h][j];
        }
      }
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

// dz = dy * act'(z) and dx = dz W together, for layers with up to 256 features in: a workgroup's tile of dx has all of
// its columns, so dy and z are read once, and dz is not read back for dx (it is written where dW needs it).  A
// chunk's dy and z are asked for a chunk ahead, into registers; their dz goes to LDS as the product's operand A, while
// W's chunk comes by LDS-DMA.  64 rows by 64 WN columns: small, so that three workgroups of a CU wait for memory in turn
// (128 rows need more registers than two workgroups of a CU have: 349 us against 125 for 44446 x 256 <- 2048, which
// moves 570 MB; apart the two take 190, since dz's way out goes on while it is read back).
struct DzDx {
  const uint16_t *dy, *z, *w;
  uint16_t *dz, *dx;  // dz: or NULL
  float* sums;        // or NULL: [workgroups][N]
  int64_t lddy, ldz, lddz, ldw, lddx;
  int M, K, N, act, w_cols;
};

constexpr int kTogetherRows = 64;
template <typename E, int WN>
__global__ void __launch_bounds__(256, 3) linear_dz_dx(const DzDx p) {
  constexpr int kWaves = 4, BM = kTogetherRows, BN = 64 * WN, TM = BM / 16 * WN / kWaves, TN = 4;
  constexpr int kA = BM * kR, kB = BN * kR, kPieces = BM * kR / 8 / 256;
  __shared__ __attribute__((aligned(16))) uint16_t lds[kA + kB];
  __shared__ float4 lds_sums[kWaves][kR / 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / WN, wn = wave % WN;
  const int m0 = int(blockIdx.x) * BM, chunks = p.N / kR;
  const int row = int(threadIdx.x >> 3), ch = int(threadIdx.x & 7);  // of a thread's first piece, 32 rows to the next
  Loader<BN, true, kWaves> lw(p.w, p.ldw, 0, p.K, p.w_cols, 0, wave, lane);
  // (rows past the end are the last one again, and count as zero)
  const char* dy = reinterpret_cast<const char*>(p.dy + int64_t(m0) * p.lddy);
  const char* z = reinterpret_cast<const char*>(p.z + int64_t(m0) * p.ldz);
  uint32_t dy_at[kPieces], z_at[kPieces];  // bytes (the host keeps row pitches below kMaxPitch)
#pragma unroll
  for (int h = 0; h < kPieces; ++h) {
    const int r = m0 + row + 32 * h < p.M ? row + 32 * h : p.M - 1 - m0;
    dy_at[h] = (uint32_t(r) * uint32_t(p.lddy) + 8 * ch) * 2;
    z_at[h] = (uint32_t(r) * uint32_t(p.ldz) + 8 * ch) * 2;
  }
  uint16_t* dz = p.dz + int64_t(m0) * p.lddz;
  const uint32_t dz_at = uint32_t(row) * uint32_t(p.lddz) + 8 * ch;
  uint4 dy_of[kPieces], z_of[kPieces];
  auto ask = [&]() {
#pragma unroll
    for (int h = 0; h < kPieces; ++h) {
      dy_of[h] = ld_once(dy + dy_at[h]);
      z_of[h] = ld_once(z + z_at[h]);
    }
    dy += 2 * kR;
    z += 2 * kR;
  };
  gd_f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = gd_f32x4{0.f, 0.f, 0.f, 0.f};
  ask();
  for (int k = 0; k < chunks; ++k) {
    if (k > 0) gd_lds_barrier();  // the last chunk's operands have been read
    lw.issue(lds, 2 * kA, wave);
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    auto slopes = [&](auto ACT) {
#pragma unroll
      for (int h = 0; h < kPieces; ++h) {
        union {
          uint4 u;
          uint16_t h16[8];
        } a, b;
        a.u = dy_of[h];
        b.u = z_of[h];
        const bool in = m0 + row + 32 * h < p.M;
        float d[8], zz[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          d[j] = E::up(a.h16[j]);
          zz[j] = E::up(b.h16[j]);
        }
        slope8(d, zz, decltype(ACT)::value);
        const uint4 u = pack8<E>(d);
        *reinterpret_cast<uint4*>(lds + row_at(row + 32 * h, ch)) = u;
        if (in) {
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[j] += d[j];
          if (p.dz) *reinterpret_cast<uint4*>(dz + 32 * h * p.lddz + dz_at) = u;
        }
      }
    };
    switch (p.act) {
      case kRelu: slopes(std::integral_constant<int, kRelu>()); break;
      case kGelu: slopes(std::integral_constant<int, kGelu>()); break;
      case kGeluTanh: slopes(std::integral_constant<int, kGeluTanh>()); break;
      default: slopes(std::integral_constant<int, kSilu>()); break;
    }
    dz += kR;
    if (p.sums) {  // over the wave's 8 rows of lanes
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum[j] += dpp<DPP_ROR8>(sum[j]);
        sum[j] += __shfl_xor(sum[j], 16, 64);
        sum[j] += __shfl_xor(sum[j], 32, 64);
      }
      if (lane < 8) {
        lds_sums[wave][2 * ch] = make_float4(sum[0], sum[1], sum[2], sum[3]);
        lds_sums[wave][2 * ch + 1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
      }
    }
    // W's chunk has landed: it is older than dz's stores (in a tile with all its rows every wave has them) and the next
    // chunk of dy and z
    if (k + 1 < chunks) {
      ask();
      if (p.dz && m0 + BM <= p.M)
        gd_wait_vmcnt(3 * kPieces);
      else
        gd_wait_vmcnt(2 * kPieces);
    } else {
      gd_wait_vmcnt(0);
    }
    gd_lds_barrier();
    if (p.sums && threadIdx.x < kR) {
      const float* const s = reinterpret_cast<const float*>(lds_sums) + threadIdx.x;
      p.sums[int64_t(blockIdx.x) * p.N + k * kR + threadIdx.x] = (s[0] + s[kR]) + (s[2 * kR] + s[3 * kR]);
    }
    const uint16_t* const img = lds + kA;
#pragma unroll
    for (int s = 0; s < kR / 32; ++s) {
      gd_i16x8 fa[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[i] = fragment<BM, false>(lds, 16 * (wm * TM + i), s, lane);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const gd_i16x8 fb = fragment<BN, true, true>(img, 16 * (wn * TN + j), s, lane);
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[i][j] = E::mma(fb, fa[i], acc[i][j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    uint4 x[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = acc[i][2 * h + (j >> 2)][j & 3];
      x[h] = pack8<E>(v);
    }
    write16(p.dx, p.lddx, m0 + 16 * (wm * TM + i), 64 * wn, p.M, p.K, lane, x[0], x[1]);
  }
}

// ---- rows that are not 16-byte aligned, copied with their ends filled with zeros; two matrices in one launch ------
struct Pack {
  const uint16_t* src[2];
  uint16_t* dst[2];
  int64_t ld[2], pieces[2];  // pieces: of 8 values, of the whole matrix (0: none)
  int cols, per_row;
};
__global__ void __launch_bounds__(256) linear_pack(const Pack p) {
  int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const int which = i >= p.pieces[0];
  if (which) i -= p.pieces[0];
  if (i >= p.pieces[which]) return;
  const int64_t r = i / p.per_row;
  const int c = int(i - r * p.per_row) * 8;
  const uint16_t* src = p.src[which] + r * p.ld[which] + c;
  union {
    uint4 u;
    uint16_t h[8];
  } w;
#pragma unroll
  for (int j = 0; j < 8; ++j) w.h[j] = c + j < p.cols ? src[j] : uint16_t(0);
  *reinterpret_cast<uint4*>(p.dst[which] + i * 8) = w.u;
}

// ---------------------------------------------------------------------------- host
int pad8(int n) { return (n + 7) / 8 * 8; }
size_t align256(size_t n) { return (n + 255) / 256 * 256; }
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
constexpr int64_t kMaxPitch = int64_t(1) << 22;  // 256 rows' offsets fit 32 bits
// whether a product can read these rows as they are
bool readable(const void* p, int64_t ld, int cols, bool padded) {
  return aligned(p, 16) && ld % 8 == 0 && (cols % 8 == 0 || (padded && ld >= pad8(cols))) && ld <= kMaxPitch;
}
int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tile and parts of one product: the cheapest by a model of what was measured (us, 16-bit, 64 values of r at a time).
// A round is as many tiles as run at once (1, 2 or 3 workgroups per CU, by their LDS); it costs `base` (the first loads
// and the output) and `chunk` per 64 values of r, `alone` where a CU has one workgroup only:
//   256 x 256  16384 x 4096 x 4096 in 4 rounds of 64 chunks: 425 us.  Only where 4 tiles or more share each operand's
//              chunk: it waits for one chunk at a time, which has to come from L2 (44446 x 2048 x 256: 100 us, by 128s 56)
//   128 x 128  the same 485 us in 8 rounds; 8400 x 1536 x 384 in one, 198 workgroups: 20 us
//   64 x 64    900 x 256 x 256 in one round of 60: 4.6 us (by 128s 7.1)
// Parts of a split sum are written and read once more, in fp32 at about 6 TB/s (they stay near), by a further launch.
// Over 72 products of this detector's sizes and wider ones the choice is 0.7 % off the best of the three on average, 14 % at most.
struct Plan {
  int tile, splits, r_per_split;
  size_t bytes;
};
Plan plan_of(int M, int N, int r) {
  struct Kind {
    int tile, slots;
    double chunk, alone, base;
  };
  constexpr Kind kinds[] = {{256, 256, 1.5, 1.5, 11.5}, {128, 512, 0.80, 0.67, 5.0}, {64, 768, 0.55, 0.40, 2.9}};
  const int asked = env_int("GD_LINEAR_TILE", 0);  // (A/B: 64, 128 or 256; another value is none)
  const int forced = asked == 64 || asked == 128 || asked == 256 ? asked : 0;
  const int64_t chunks = div_up(r, kR);
  Plan p = {};
  double best = 1e30;
  for (const Kind& k : kinds) {
    const int64_t tm = div_up(M, k.tile), tn = div_up(N, k.tile);
    if (forced ? forced != k.tile : (k.tile == 256 && (tm < 4 || tn < 4))) continue;
    for (int64_t s = 1; s == 1 || (s <= 64 && chunks / s >= 4); s *= 2) {
      const int64_t part = div_up(chunks, s), parts = div_up(chunks, part), blocks = tm * tn * parts;
      double cost = double(div_up(blocks, k.slots)) * (double(part) * (blocks <= 256 ? k.alone : k.chunk) + k.base);
      if (parts > 1) cost += 3.4 + double(parts) * M * N * 8.0 / 6e6;
      if (cost < best) {
        best = cost;
        p.tile = k.tile;
        p.splits = int(parts);
        p.r_per_split = int(part * kR);
      }
    }
  }
  p.bytes = p.splits > 1 ? align256(size_t(p.splits) * M * N * sizeof(float)) : 0;
  return p;
}

// whether linear_stream takes a layer: whole chunks, at least two, and whole aligned pieces in every row
bool streams(const Gemm& g) {
  return g.ra == g.rb && g.ra % kR == 0 && g.ra >= 2 * kR && g.N % 8 == 0 && g.epi.y_vec &&
         (!g.epi.bias || g.epi.bias_vec) && (!g.epi.res || g.epi.res_vec);
}

template <typename E, bool AC, bool BC>
gd_status product(const Plan& plan, Gemm g, void* part, hipStream_t s, Join join = Join()) {
  g.splits = plan.splits;
  g.r_per_split = plan.r_per_split;
  g.part = static_cast<float*>(part);
  g.tiles_m = int(div_up(g.M, plan.tile));
  g.tiles_n = int(div_up(g.N, plan.tile));
  g.group = plan.tile == 256 ? 4 : 8;  // (32 or 64 workgroups per XCD at a time)
  const int64_t grid = int64_t(g.tiles_m) * g.tiles_n * plan.splits;
  GD_REQUIRE(grid < (int64_t(1) << 31), "linear: grid too large");
  if (!AC && plan.tile == 128 && plan.splits == 1 && env_int("GD_LINEAR_STREAM", 1) && streams(g)) {
    const int64_t at_once = std::max(1, env_int("GD_LINEAR_GROUPS", 512));  // (A/B) two of a CU
    hipLaunchKernelGGL((linear_stream<E, BC>), dim3(unsigned(grid < at_once ? grid : at_once)), dim3(256), 0, s, g);
  } else if (plan.tile == 256) {
    if (!AC && !BC && plan.splits == 1 && env_int("GD_LINEAR_STREAM", 1) && streams(g))
      hipLaunchKernelGGL((linear_gemm256<E, false, false, true>), dim3(unsigned(grid)), dim3(256), 0, s, g);
    else
      hipLaunchKernelGGL((linear_gemm256<E, AC, BC, false>), dim3(unsigned(grid)), dim3(256), 0, s, g);
  } else if (plan.tile == 128)
    hipLaunchKernelGGL((linear_gemm<E, 2, 2, 4, 4, 2, AC, BC>), dim3(unsigned(grid)), dim3(256), 0, s, g);
  else
    hipLaunchKernelGGL((linear_gemm<E, 2, 2, 2, 2, 3, AC, BC>), dim3(unsigned(grid)), dim3(256), 0, s, g);
  GD_LAUNCH_CHECK("linear_gemm");
  if (plan.splits > 1) {
    const int64_t blocks = div_up(int64_t(g.M) * ((g.N + 7) / 8), 256);
    GD_REQUIRE(blocks < (int64_t(1) << 30), "linear: grid too large");
    join.first = int(blocks);
    const int64_t more = join.db ? div_up(join.N, kJoinColumns) : 0;
    hipLaunchKernelGGL(linear_finish<E>, dim3(unsigned(blocks + more)), dim3(256), 0, s, g.part, plan.splits, g.M, g.N, g.epi,
                       join);
    GD_LAUNCH_CHECK("linear_finish");
  }
  return GD_OK;
}

// an operand's rows; `padded`: their ends are filled with zeros up to a multiple of 8
struct Rows {
  const uint16_t* p;
  int64_t ld;
  int cols;  // readable, a multiple of 8
};
Rows rows_of(const void* p, int64_t ld, int cols) { return {static_cast<const uint16_t*>(p), ld, pad8(cols)}; }

Epi plain_epi(void* y, bool f32, int64_t ldy) {
  Epi e = {};
  e.y = y;
  e.y_f32 = f32;
  e.ldy = ldy;
  e.y_vec = aligned(y, 16) && ldy % (f32 ? 4 : 8) == 0;
  return e;
}

// workgroups along the rows of linear_dact: about 1024 in all, each of at least 4 rows per lane group
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

// Whether the backward of an activation and dx are one kernel (the rest of the conditions is about the pieces).  Its
// workgroups take some 1.8 us per chunk whatever their number, so it pays for many rows, and where dz on its way
// through memory costs more than its place in the caches: 44446 x 256 <- 2048 193 us and 217 apart (the whole
// backward), 33400 x 192 <- 768 84 and 94; 16384 x 256 <- 1024 66 and 65, 8192 x 256 <- 2048 79 and 62.
bool dz_dx_fits(int M, int K, int N) {
  const int from = env_int("GD_LINEAR_TOGETHER", 0);  // (A/B: rows)
  return K <= 256 && (from > 0 ? M >= from : M >= 24576 && int64_t(M) * N >= 20000000);
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
  const Rows rx = rows_of(x, ldx, K), rw = rows_of(w, ldw, K);
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
  const bool make = act != kNone || dy_dtype == GD_F32 || !readable(dy, lddy, N, false);
  if (make && (dx || dw)) {
    rz = {reinterpret_cast<uint16_t*>(ws), n8, n8};
    ws += align256(size_t(M) * n8 * 2);
  }
  Join join = {};
  const Rows rw = dx ? rows_of(w, ldw, K) : Rows();
  const Epi to_dx = dx ? plain_epi(dx, dx_dtype == GD_F32, lddx) : Epi();
  const bool together = dx && act != kNone && dy_dtype != GD_F32 && aligned(dy, 16) && lddy % 8 == 0 && aligned(z, 16) &&
                        ldz % 8 == 0 && lddy <= kMaxPitch && ldz <= kMaxPitch && N % kR == 0 && K % 8 == 0 && dz_dx_fits(M, K, N) && !to_dx.y_f32 && to_dx.y_vec;
  if (together) {
    DzDx a = {};
    a.dy = static_cast<const uint16_t*>(dy);
    a.lddy = lddy;
    a.z = static_cast<const uint16_t*>(z);
    a.ldz = ldz;
    a.w = rw.p;
    a.ldw = rw.ld;
    a.w_cols = rw.cols;
    a.dz = dw ? const_cast<uint16_t*>(rz.p) : nullptr;
    a.lddz = n8;
    a.dx = static_cast<uint16_t*>(dx);
    a.lddx = lddx;
    a.M = M;
    a.K = K;
    a.N = N;
    a.act = act;
    const int blocks = int(div_up(M, kTogetherRows));
    if (db) {
      a.sums = reinterpret_cast<float*>(ws);
      ws += align256(size_t(blocks) * N * sizeof(float));
    }
    if (K <= 128)
      hipLaunchKernelGGL((linear_dz_dx<E, 2>), dim3(blocks), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((linear_dz_dx<E, 4>), dim3(blocks), dim3(256), 0, s, a);
    GD_LAUNCH_CHECK("linear_dz_dx");
    if (db) join = {a.sums, db, blocks, N, int(param_dtype == GD_F32), 0};
  } else if (db || (make && (dx || dw))) {
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
    if (db) join = {a.sums, db, d.blocks, N, int(param_dtype == GD_F32), 0};
  }
  if (dx && !together) {
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
    g.epi = to_dx;
    const Plan p = plan_of(M, K, n8);
    GD_TRY((product<E, false, true>(p, g, ws, s)));
    ws += p.bytes;
  }
  if (dw) {
    const Rows rx = rows_of(x, ldx, K);
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
    const Plan p = plan_of(N, K, M);
    GD_TRY((product<E, true, true>(p, g, ws, s, join)));
    if (p.splits > 1) return GD_OK;  // (with the column sums)
  }
  if (join.db) {
    hipLaunchKernelGGL(linear_colsum<E>, dim3(unsigned(div_up(N, kJoinColumns))), dim3(256), 0, s, join);
    GD_LAUNCH_CHECK("linear_colsum");
  }
  return GD_OK;
}

size_t backward_bytes(int M, int K, int N, bool dx, bool dw, bool db) {
  const int n8 = pad8(N);
  size_t b = dx || dw ? align256(size_t(M) * n8 * 2) : 0;
  if (db) {
    const int64_t alone = dact_plan(M, N).blocks, together = dx && dz_dx_fits(M, K, N) ? div_up(M, kTogetherRows) : 0;
    b += align256(size_t(alone > together ? alone : together) * N * sizeof(float));
  }
  if (dx) b += plan_of(M, K, n8).bytes;
  if (dw) b += plan_of(N, K, M).bytes;
  return b;
}

}  // namespace
}  // namespace gd

using namespace gd;

extern "C" int gd_linear_readable(const void* p, int64_t ld, int cols, int padded) {
  return readable(p, ld, cols, padded != 0);
}

extern "C" gd_status gd_linear_pack(const void* a, int64_t lda, int rows_a, const void* b, int64_t ldb, int rows_b,
                                    int cols, void* a_out, void* b_out, gd_stream_t stream) {
  GD_REQUIRE(cols > 0 && cols <= kMaxPitch && rows_a >= 0 && rows_b >= 0 && rows_a <= (1 << 30) && rows_b <= (1 << 30),
             "linear_pack: %d and %d rows of %d", rows_a, rows_b, cols);
  GD_REQUIRE(rows_a == 0 || (a && a_out && aligned(a, 2) && aligned(a_out, 16) && lda >= cols), "linear_pack: first matrix");
  GD_REQUIRE(rows_b == 0 || (b && b_out && aligned(b, 2) && aligned(b_out, 16) && ldb >= cols), "linear_pack: second matrix");
  Pack p;
  p.src[0] = static_cast<const uint16_t*>(a);
  p.src[1] = static_cast<const uint16_t*>(b);
  p.dst[0] = static_cast<uint16_t*>(a_out);
  p.dst[1] = static_cast<uint16_t*>(b_out);
  p.ld[0] = lda;
  p.ld[1] = ldb;
  p.cols = cols;
  p.per_row = pad8(cols) / 8;
  p.pieces[0] = int64_t(rows_a) * p.per_row;
  p.pieces[1] = int64_t(rows_b) * p.per_row;
  const int64_t blocks = div_up(p.pieces[0] + p.pieces[1], 256);
  if (blocks == 0) return GD_OK;
  GD_REQUIRE(blocks < (int64_t(1) << 31), "linear_pack: grid too large");
  hipLaunchKernelGGL(linear_pack, dim3(unsigned(blocks)), dim3(256), 0, as_hip(stream), p);
  GD_LAUNCH_CHECK("linear_pack");
  return GD_OK;
}

extern "C" size_t gd_linear_forward_workspace_bytes(int M, int K, int N) {
  return M > 0 && K > 0 && N > 0 ? plan_of(M, N, pad8(K)).bytes : 0;
}

extern "C" gd_status gd_linear_forward(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw,
                                       const void* bias, int act, const void* residual, int residual_dtype,
                                       int64_t ldr, int M, int K, int N, void* y, int y_dtype, int64_t ldy, void* z,
                                       int64_t ldz, int padded, void* workspace, size_t workspace_bytes, gd_stream_t stream) {
  GD_TRY(check_shape(dtype, act, M, K, N));
  if (M == 0) return GD_OK;
  GD_REQUIRE(x && w && y && ldx >= K && ldw >= K && ldy >= N, "linear: null pointer or short rows");
  GD_REQUIRE(readable(x, ldx, K, padded) && readable(w, ldw, K, padded) && aligned(bias, 2),
             "linear: x and W need rows of 16-byte pieces (gd_linear_pack)");
  GD_REQUIRE(!residual || (ldr >= N && (residual_dtype == dtype || residual_dtype == GD_F32)),
             "linear: the residual is fp32 or of the operands' type");
  GD_REQUIRE(y_dtype == (residual ? residual_dtype : dtype), "linear: y has the residual's type, without one x's");
  GD_REQUIRE(aligned(y, y_dtype == GD_F32 ? 4 : 2) && aligned(residual, residual_dtype == GD_F32 ? 4 : 2),
             "linear: misaligned y or residual");
  GD_REQUIRE(!z || (aligned(z, 16) && ldz % 8 == 0 && ldz >= pad8(N)), "linear: z has rows padded to 8 values");
  const size_t want = plan_of(M, N, pad8(K)).bytes;
  GD_REQUIRE(workspace_bytes >= want && (want == 0 || (workspace && aligned(workspace, 16))),
             "linear: workspace of %zu bytes, %zu wanted", workspace_bytes, want);
  char* ws = static_cast<char*>(workspace);
  hipStream_t s = as_hip(stream);
  return dtype == GD_BF16 ? forward<Bf16>(x, ldx, w, ldw, bias, act, residual, residual_dtype, ldr, M, K, N, y, y_dtype,
                                          ldy, z, ldz, ws, s)
                          : forward<Fp16>(x, ldx, w, ldw, bias, act, residual, residual_dtype, ldr, M, K, N, y, y_dtype,
                                          ldy, z, ldz, ws, s);
}

extern "C" size_t gd_linear_backward_workspace_bytes(int M, int K, int N, int dx, int dw, int db) {
  return M > 0 && K > 0 && N > 0 ? backward_bytes(M, K, N, dx, dw, db) : 0;
}

extern "C" gd_status gd_linear_backward(int dtype, int act, const void* dy, int dy_dtype, int64_t lddy, const void* z,
                                        int64_t ldz, const void* x, int64_t ldx, const void* w, int64_t ldw, int M,
                                        int K, int N, void* dx, int dx_dtype, int64_t lddx, void* dw, void* db,
                                        int param_dtype, int padded, void* workspace, size_t workspace_bytes,
                                        gd_stream_t stream) {
  GD_TRY(check_shape(dtype, act, M, K, N));
  GD_REQUIRE(M > 0, "linear: gradients of no rows");
  GD_REQUIRE(dy && lddy >= N && (!dw || (x && ldx >= K)) && (!dx || (w && ldw >= K && lddx >= K)),
             "linear: null pointer or short rows");
  GD_REQUIRE(dy_dtype == dtype || dy_dtype == GD_F32, "linear: dy is fp32 or of the operands' type");
  GD_REQUIRE((dx_dtype == dtype || dx_dtype == GD_F32) && (param_dtype == dtype || param_dtype == GD_F32),
             "linear: gradients are fp32 or of the operands' type");
  GD_REQUIRE(act == kNone || (z && ldz >= N), "linear: the activation's slope needs z");
  GD_REQUIRE(aligned(dy, dy_dtype == GD_F32 ? 4 : 2) && aligned(z, 2) && aligned(dx, dx_dtype == GD_F32 ? 4 : 2) && aligned(dw, param_dtype == GD_F32 ? 4 : 2) &&
                 aligned(db, param_dtype == GD_F32 ? 4 : 2),
             "linear: misaligned operands");
  GD_REQUIRE((!dw || readable(x, ldx, K, padded)) && (!dx || readable(w, ldw, K, padded)),
             "linear: x and W need rows of 16-byte pieces (gd_linear_pack)");
  const size_t want = backward_bytes(M, K, N, dx, dw, db);
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
