// Optimizer kernels for gfx950 over many tensors per launch: AdamW with the
// gradient clip folded in, and the 2-norm over all gradients.
//
//   g  = grad * min(1, max_norm / (norm + 1e-6))
//   m' = b1 m + (1 - b1) g          v' = b2 v + (1 - b2) g^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Both are bound by HBM: every value is read and written once (28 B per
// element with fp32 moments, 16.1 B with 8-bit ones, 4 or 2 B for the norm),
// so the work is a plain stream and the design is about launches.  A model
// has hundreds of tensors, most of them small; the tensors of a launch travel
// as a table in the kernel arguments (below 4 KB, so a captured graph holds it and
// no copy to the device precedes the launch), and each workgroup finds its
// tensor and chunk there from its index.
//
// Moments in 8 bits: per 32 consecutive elements one power of two (a biased
// exponent byte) and e4m3 values, for the first moment and for the ROOT of the
// second (its square spans twice the exponents: 2^17 of root are 2^34 of
// second moment).  The rounding is stochastic: with 1 - b2 = 1e-3 an
// average moves by a thousandth per step, half of e4m3's step is a
// sixteenth, so rounding to nearest would never let it decay; rounding up with
// the probability of the distance keeps its expectation.  A positive root
// never becomes zero (the update would divide by eps).  The update itself
// uses the fp32 moments before they are rounded.
#include "gd_common.h"

#include <cmath>

namespace gd {
namespace {

constexpr int kOpThreads = 256;
constexpr int kOpVec = 4;                         // consecutive elements per lane
// elements per workgroup: one group of four per thread, and the many waves hide its loads (two or four groups in a
// loop, all loaded ahead: 405 and 418 us against 401 for the detector's clipped step, 220 and 245 against 212 in 8 bits)
constexpr int kOpChunk = kOpThreads * kOpVec;
constexpr uint32_t kOpPiece = 1u << 30;           // elements of one table entry at most
constexpr uint32_t kOpAligned = 1u << 31;         // flag on an entry's count: vector accesses are aligned
constexpr uint32_t kOpFirst = kOpPiece - 1;       // an entry's first workgroup; the bits above: its first element within
                                                  // its tensor, a multiple of kOpPiece, modulo 2^32
constexpr uint32_t kOpBlocks = 1u << 23;          // workgroups after which a launch is closed (its threads fit 32 bits)
constexpr int kOpArgBytes = 3840;                 // the table's share of the 4 KB of kernel arguments

// The table entry whose chunks hold workgroup b: `first` ascends from 0, so it is the number of entries
// that start at or before b, less one.  One load per lane instead of a search's chain of loads.
__device__ __forceinline__ int find_entry(const uint32_t* first, int n, uint32_t b) {
  const int lane = threadIdx.x & 63;
  int at = -1;
  for (int i = 0; i < n; i += 64) {
    const bool here = i + lane < n && (first[i + lane] & kOpFirst) <= b;
    at += __popcll(__ballot(here));
  }
  return at;
}

// ---- 4 consecutive elements from / to memory, the first `left` of them valid ----
// Weights and moments pass by the caches (ONCE, and the stores): they are next touched a step later, and the gradients
// that the norm has just read stay in the 256 MB memory-side cache for the update (62 M weights, clipped: 397 us with
// plain accesses, 393 with these loads, 313 with loads and stores; moments in 8 bits 209 and 185; 400 M masters 1378 and
// 1268, 1250 with the bf16 copies as well).
#ifndef GD_STORE_NT
#define GD_STORE_NT(value, to) __builtin_nontemporal_store(value, to)
#define GD_LOAD_NT(from) __builtin_nontemporal_load(from)
#endif
typedef float op_f32x4 __attribute__((ext_vector_type(4)));

template <bool ONCE = false>
__device__ __forceinline__ void ld4(const float* p, int left, bool vec, float v[4]) {
  if (vec && left >= 4) {
    const op_f32x4* const q = reinterpret_cast<const op_f32x4*>(p);
    const op_f32x4 a = ONCE ? GD_LOAD_NT(q) : *q;
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < left ? p[j] : 0.f;
  }
}
__device__ __forceinline__ void ld4(const uint16_t* p, int left, bool vec, float v[4]) {
  if (vec && left >= 4) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    v[0] = bf16_lo(a.x); v[1] = bf16_hi(a.x); v[2] = bf16_lo(a.y); v[3] = bf16_hi(a.y);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < left ? bf16_to_f32(p[j]) : 0.f;
  }
}
__device__ __forceinline__ uint32_t ld4b(const uint8_t* p, int left, bool vec) {
  if (vec && left >= 4) return GD_LOAD_NT(reinterpret_cast<const uint32_t*>(p));
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) w |= j < left ? uint32_t(p[j]) << (8 * j) : 0u;
  return w;
}
__device__ __forceinline__ void st4(float* p, int left, bool vec, const float v[4]) {
  if (vec && left >= 4) {
    GD_STORE_NT((op_f32x4{v[0], v[1], v[2], v[3]}), reinterpret_cast<op_f32x4*>(p));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = v[j];
  }
}
__device__ __forceinline__ void st4(uint16_t* p, int left, bool vec, const float v[4]) {
  if (vec && left >= 4) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    GD_STORE_NT((u32x2{uint32_t(f32_to_bf16(v[0])) | (uint32_t(f32_to_bf16(v[1])) << 16),
                       uint32_t(f32_to_bf16(v[2])) | (uint32_t(f32_to_bf16(v[3])) << 16)}),
                reinterpret_cast<u32x2*>(p));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = f32_to_bf16(v[j]);
  }
}
__device__ __forceinline__ void st4b(uint8_t* p, int left, bool vec, uint32_t w) {
  if (vec && left >= 4) {
    GD_STORE_NT(w, reinterpret_cast<uint32_t*>(p));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = uint8_t(w >> (8 * j));
  }
}

// ---- the 8-bit moments --------------------------------------------------------
__device__ __forceinline__ uint32_t op_hash(uint32_t i, uint32_t key) {
  uint32_t h = (i * 0x9E3779B1u) ^ key;
  h ^= h >> 16;
  h *= 0x7FEB352Du;
  h ^= h >> 15;
  h *= 0x846CA68Bu;
  return h ^ (h >> 16);
}

typedef float gd_f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ void unpack_e4m3(uint32_t w, float scale, float v[4]) {
  const gd_f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false);
  const gd_f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
  v[0] = a[0] * scale; v[1] = a[1] * scale; v[2] = b[0] * scale; v[3] = b[1] * scale;
}

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// 32 elements (8 lanes of 4) -> e4m3 and their scale's exponent byte.  r: 16 random bits per element.
// The largest finite magnitude lands in (224, 448], e4m3's largest value, so rounding up cannot leave the
// range; values that are not finite become NaN and do not touch the others of their block.
template <bool KEEP>
__device__ __forceinline__ uint32_t pack_e4m3(const float x[4], const uint32_t r[4], uint32_t* byte) {
  float a[4];
  uint32_t top = 0;  // magnitudes ordered as their bits
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    a[j] = __uint_as_float(__float_as_uint(x[j]) & 0x7fffffffu);
    const uint32_t b = __float_as_uint(a[j]);
    top = b < 0x7f800000u && b > top ? b : top;
  }
#pragma unroll
  for (int s = 0; s < 3; ++s) {
    const float t = __uint_as_float(top);
    const float o = s == 0 ? dpp<DPP_XOR1>(t) : s == 1 ? dpp<DPP_XOR2>(t) : dpp<DPP_HALF_MIRROR>(t);
    const uint32_t ob = __float_as_uint(o);
    top = ob > top ? ob : top;
  }
  int e = int(top >> 23) - 127 - ((top & 0x7fffffu) > 0x600000u ? 7 : 8);
  e = e < -126 ? -126 : e;  // (at most 127 - 7)
  *byte = uint32_t(e + 127);
  const float inv = __uint_as_float(uint32_t(127 - e) << 23);
  float q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float y = a[j] * inv;
    // below 2^-6 e4m3's steps stay 2^-9: shifted by 2^-6 such a value has them as its last mantissa bits
    const float shift = y < 0.015625f ? 0.015625f : 0.f;
    const float t = __uint_as_float((__float_as_uint(y + shift) + (r[j] << 4)) & 0xfff00000u) - shift;
    q[j] = KEEP && t == 0.f && a[j] > 0.f ? 0.001953125f : t;
    q[j] = __uint_as_float(__float_as_uint(q[j]) | (__float_as_uint(x[j]) & 0x80000000u));
    if (!(a[j] <= 3.402823466e38f)) q[j] = __uint_as_float(0x7fc00000u);
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true));
}

// ---- AdamW ---------------------------------------------------------------------
struct AdamConst {
  float beta1, beta2, one_minus_beta1, one_minus_beta2, eps, weight_decay, lr;
  float inv_bc1, inv_sqrt_bc2;  // 1 / (1 - b1^t), 1 / sqrt(1 - b2^t): with the step on the host
  float max_norm;
  double log2_beta1, log2_beta2;
  const float* lr_dev;      // or NULL
  const float* total_norm;  // or NULL
  uint32_t seed, key;       // key: seed + t * 0x85EBCA77, with the step on the host
};

// E8: 8-bit moments, CP: a bf16 copy of the weights, ST: the step counts are on the device
template <bool E8, bool CP, bool ST>
struct AdamTable {
  static constexpr int kEntry = 32 + (E8 ? 16 : 0) + (CP ? 8 : 0) + (ST ? 8 : 0) + 8;
  static constexpr int kCap = kOpArgBytes / kEntry;
  float* p[kCap];
  const void* g[kCap];
  void* m[kCap];
  void* v[kCap];
  uint8_t* ms[E8 ? kCap : 1];
  uint8_t* vs[E8 ? kCap : 1];
  uint16_t* copy[CP ? kCap : 1];
  const float* step[ST ? kCap : 1];
  uint32_t n[kCap];      // elements | kOpAligned
  uint32_t first[kCap];  // see kOpFirst
  int entries;
};

// The hardware's root and reciprocal, an ulp each: exact ones are some 20 instructions per weight (8-bit moments:
// 245 us -> 212 for the detector).  The root takes denormal values for 0: scaled around it.
__device__ __forceinline__ float op_sqrt(float x) {
  const bool tiny = x < 0x1p-96f;
  const float r = __builtin_amdgcn_sqrtf(tiny ? x * 0x1p96f : x);
  return tiny ? r * 0x1p-48f : r;
}

// what a launch's thread knows of its step
struct AdamStep {
  float step_size, decay, clip, inv_sqrt_bc2;
  uint32_t key;
};

// A thread's 4 elements, the first of them `i`.  FULL: the whole chunk exists and its accesses are aligned.
template <typename TG, bool E8, bool CP, bool ST, bool FULL>
__device__ __forceinline__ void adamw_four(const AdamTable<E8, CP, ST>& t, const AdamConst& c, const AdamStep& s, int e,
                                           uint32_t i, uint32_t n, bool vec) {
  const int k = FULL ? 4 : (i < n ? int(n - i < 4u ? n - i : 4u) : 0);
  float w[4], gr[4], m[4], v[4], root[4];
  ld4<true>(t.p[e] + i, k, FULL || vec, w);
  ld4(static_cast<const TG*>(t.g[e]) + i, k, FULL || vec, gr);
  if constexpr (E8) {
    const uint32_t mw = ld4b(static_cast<const uint8_t*>(t.m[e]) + i, k, FULL || vec);
    const uint32_t vw = ld4b(static_cast<const uint8_t*>(t.v[e]) + i, k, FULL || vec);
    unpack_e4m3(mw, scale_of(k > 0 ? t.ms[e][i >> 5] : 1), m);
    unpack_e4m3(vw, scale_of(k > 0 ? t.vs[e][i >> 5] : 1), v);
  } else {
    ld4<true>(static_cast<const float*>(t.m[e]) + i, k, FULL || vec, m);
    ld4<true>(static_cast<const float*>(t.v[e]) + i, k, FULL || vec, v);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float gj = gr[j] * s.clip;
    if (E8) v[j] *= v[j];
    m[j] = c.beta1 * m[j] + c.one_minus_beta1 * gj;
    v[j] = c.beta2 * v[j] + c.one_minus_beta2 * gj * gj;
    root[j] = op_sqrt(v[j]);
    const float inv = __builtin_amdgcn_rcpf(root[j] * s.inv_sqrt_bc2 + c.eps);
    w[j] = (w[j] - s.decay * w[j]) - s.step_size * (m[j] * inv);
  }
  st4(t.p[e] + i, k, FULL || vec, w);
  if constexpr (CP) st4(t.copy[e] + i, k, FULL || vec, w);
  if constexpr (E8) {
    // (the 8 lanes of a block of 32 exchange its maximum: lanes past the end take part, with zeros)
    uint32_t rm[4], rv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t h = op_hash((t.first[e] & ~kOpFirst) + i + j, s.key);
      rm[j] = h & 0xffffu;
      rv[j] = h >> 16;
      if (j >= k) m[j] = root[j] = 0.f;
    }
    uint32_t mb, vb;
    const uint32_t mw = pack_e4m3<false>(m, rm, &mb);
    const uint32_t vw = pack_e4m3<true>(root, rv, &vb);
    st4b(static_cast<uint8_t*>(t.m[e]) + i, k, FULL || vec, mw);
    st4b(static_cast<uint8_t*>(t.v[e]) + i, k, FULL || vec, vw);
    if (k > 0 && (i & 31u) == 0) {
      t.ms[e][i >> 5] = uint8_t(mb);
      t.vs[e][i >> 5] = uint8_t(vb);
    }
  } else {
    st4(static_cast<float*>(t.m[e]) + i, k, FULL || vec, m);
    st4(static_cast<float*>(t.v[e]) + i, k, FULL || vec, v);
  }
}

// Measured: 62 M weights in 385 tensors with moments in 8 bits 185 us (5.4 TB/s); with fp32 moments and the norm 313 us, 400 M
// fp32 masters with bf16 gradients and copies, 8 bits and the norm 1250 us (5.8 TB/s).  A copy of 1 GiB runs at 5.2 TB/s.
// With the counts on the device (ST) 62 M weights take 285 us for 280 (no norm), in 8 bits 212 for 194: doubles in every
// wave, and a table of 60 tensors for 68.
template <typename TG, bool E8, bool CP, bool ST>
__global__ void __launch_bounds__(kOpThreads)
adamw_kernel(const AdamTable<E8, CP, ST> t, const AdamConst c) {
  const int e = find_entry(t.first, t.entries, blockIdx.x);
  const bool vec = (t.n[e] & kOpAligned) != 0;
  const uint32_t n = t.n[e] & ~kOpAligned;
  const uint32_t begin = (blockIdx.x - (t.first[e] & kOpFirst)) * uint32_t(kOpChunk);

  AdamStep s;
  float inv_bc1 = c.inv_bc1;
  s.inv_sqrt_bc2 = c.inv_sqrt_bc2;
  s.key = c.key;
  if constexpr (ST) {
    const float step = *t.step[e];
    // in double: 1 - b^t cancels for small t
    inv_bc1 = float(1.0 / (1.0 - exp2(double(step) * c.log2_beta1)));
    s.inv_sqrt_bc2 = float(1.0 / sqrt(1.0 - exp2(double(step) * c.log2_beta2)));
    s.key = c.seed + uint32_t(step) * 0x85EBCA77u;
  }
  const float lr = c.lr_dev ? *c.lr_dev : c.lr;
  s.step_size = lr * inv_bc1;
  s.decay = lr * c.weight_decay;
  s.clip = 1.f;
  if (c.total_norm) {
    s.clip = c.max_norm / (*c.total_norm + 1e-6f);
    s.clip = s.clip > 1.f ? 1.f : s.clip;  // (NaN stays)
  }
  const uint32_t i = begin + threadIdx.x * kOpVec;
  if (vec && n - begin >= uint32_t(kOpChunk))
    adamw_four<TG, E8, CP, ST, true>(t, c, s, e, i, n, vec);
  else
    adamw_four<TG, E8, CP, ST, false>(t, c, s, e, i, n, vec);
}

bool op_aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

struct AdamLists {
  const uint64_t *p, *g, *m, *v, *ms, *vs, *copy, *step;
  const int64_t* n;
  int grad_bf16;
};

template <typename T>
T* at(const uint64_t* list, int i) { return reinterpret_cast<T*>(uintptr_t(list[i])); }

template <typename TG, bool E8, bool CP, bool ST>
gd_status adamw_launch(int tensors, const AdamLists& l, const AdamConst& c, hipStream_t s) {
  AdamTable<E8, CP, ST> t;
  static_assert(sizeof(t) + sizeof(c) <= 4000, "kernel arguments stay below 4 KB");
  uint32_t blocks = 0;
  t.entries = 0;
  auto flush = [&]() -> gd_status {
    if (t.entries == 0) return GD_OK;
    hipLaunchKernelGGL((adamw_kernel<TG, E8, CP, ST>), dim3(blocks), dim3(kOpThreads), 0, s, t, c);
    GD_LAUNCH_CHECK("adamw_step");
    t.entries = 0;
    blocks = 0;
    return GD_OK;
  };
  // from the last tensor on: the norm, which goes from the first, has left the last gradients in the memory-side cache (400 M
  // masters with clipping 1248 us in the lists' order, 1225 in this one)
  for (int i = tensors - 1; i >= 0; --i) {
    for (int64_t off = 0; off < l.n[i]; off += kOpPiece) {
      const uint32_t n = uint32_t(l.n[i] - off < int64_t(kOpPiece) ? l.n[i] - off : int64_t(kOpPiece));
      const int e = t.entries++;
      t.p[e] = at<float>(l.p, i) + off;
      t.g[e] = at<const TG>(l.g, i) + off;
      bool al = op_aligned(t.p[e], 16) && op_aligned(t.g[e], 4 * sizeof(TG));
      if constexpr (E8) {
        t.m[e] = at<uint8_t>(l.m, i) + off;
        t.v[e] = at<uint8_t>(l.v, i) + off;
        t.ms[e] = at<uint8_t>(l.ms, i) + off / 32;
        t.vs[e] = at<uint8_t>(l.vs, i) + off / 32;
        al = al && op_aligned(t.m[e], 4) && op_aligned(t.v[e], 4);
      } else {
        t.m[e] = at<float>(l.m, i) + off;
        t.v[e] = at<float>(l.v, i) + off;
        al = al && op_aligned(t.m[e], 16) && op_aligned(t.v[e], 16);
      }
      if constexpr (CP) {
        t.copy[e] = at<uint16_t>(l.copy, i) + off;
        al = al && op_aligned(t.copy[e], 8);
      }
      if constexpr (ST) t.step[e] = at<const float>(l.step, i);
      t.n[e] = n | (al ? kOpAligned : 0u);
      t.first[e] = blocks | uint32_t(off);
      blocks += (n + kOpChunk - 1) / kOpChunk;
      if (t.entries == AdamTable<E8, CP, ST>::kCap || blocks >= kOpBlocks) {
        const gd_status st = flush();
        if (st != GD_OK) return st;
      }
    }
  }
  return flush();
}

template <typename TG, bool E8, bool CP>
gd_status adamw_pick3(int tensors, const AdamLists& l, const AdamConst& c, hipStream_t s) {
  return l.step ? adamw_launch<TG, E8, CP, true>(tensors, l, c, s) : adamw_launch<TG, E8, CP, false>(tensors, l, c, s);
}
template <typename TG, bool E8>
gd_status adamw_pick2(int tensors, const AdamLists& l, const AdamConst& c, hipStream_t s) {
  return l.copy ? adamw_pick3<TG, E8, true>(tensors, l, c, s) : adamw_pick3<TG, E8, false>(tensors, l, c, s);
}
template <typename TG>
gd_status adamw_pick(int tensors, const AdamLists& l, const AdamConst& c, hipStream_t s) {
  return l.ms ? adamw_pick2<TG, true>(tensors, l, c, s) : adamw_pick2<TG, false>(tensors, l, c, s);
}

// ---- the 2-norm over many tensors -------------------------------------------------
// Squares and sums in double: their cost hides behind the loads, gradients above 1.8e19 do not overflow, and
// the order (a chunk per workgroup, then one workgroup over the chunks) is fixed, so the result repeats.
struct NormTable {
  static constexpr int kCap = kOpArgBytes / 16;
  const void* g[kCap];
  uint32_t n[kCap];
  uint32_t first[kCap];
  int entries;
  uint32_t chunk;     // elements per workgroup, a multiple of 1024
  double* partial;    // of this launch's workgroups
};

__device__ __forceinline__ double block_sum(double x, double* lds) {
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  double r = 0.0;
  for (int i = 0; i < int(blockDim.x >> 6); ++i) r += lds[i];
  return r;
}

// Measured: 400 M fp32 values in 290 tensors 276 us when repeated (the last 256 MB stay in the
// memory-side cache), 326 on gradients not read before (4.9 TB/s); eight loads under way, coarser or finer pieces: no faster.
template <typename TG>
__global__ void __launch_bounds__(kOpThreads) norm_chunk_kernel(const NormTable t) {
  __shared__ double lds[kOpThreads / 64];
  const int e = find_entry(t.first, t.entries, blockIdx.x);
  const bool vec = (t.n[e] & kOpAligned) != 0;
  const uint32_t n = t.n[e] & ~kOpAligned;
  const uint32_t begin = (blockIdx.x - t.first[e]) * t.chunk;
  const uint32_t end = n - begin < t.chunk ? n : begin + t.chunk;
  const TG* const g = static_cast<const TG*>(t.g[e]);
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  constexpr uint32_t kStep = kOpThreads * kOpVec;
  uint32_t i = begin + threadIdx.x * kOpVec;
  if (vec) {
    for (; i + 3 * kStep + 4 <= end; i += 4 * kStep) {  // four loads under way
      float v[4][4];
#pragma unroll
      for (int h = 0; h < 4; ++h) ld4(g + i + h * kStep, 4, true, v[h]);
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += double(v[h][j]) * double(v[h][j]);
    }
  }
  for (; i < end; i += kStep) {
    float v[4];
    ld4(g + i, int(end - i < 4u ? end - i : 4u), vec, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] += double(v[j]) * double(v[j]);
  }
  const double r = block_sum((sum[0] + sum[1]) + (sum[2] + sum[3]), lds);
  if (threadIdx.x == 0) t.partial[blockIdx.x] = r;
}

constexpr int kNormJoin = 1024;

__global__ void __launch_bounds__(kNormJoin) norm_join_kernel(const double* __restrict__ partial, int n,
                                                             float* __restrict__ out) {
  __shared__ double lds[kNormJoin / 64];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kNormJoin) s += partial[i];
  s = block_sum(s, lds);
  if (threadIdx.x == 0) *out = float(sqrt(s));
}

// Elements per workgroup: 4096 (latency: a few vector loads per lane) up to 2^25 elements in all, beyond that
// an 8192nd of them, 2^22 at most, so that the joining workgroup reads some ten values per thread.
int64_t norm_chunk(int64_t total) {
  const int64_t c = (total / 8192 + 1023) / 1024 * 1024;
  return c < 4096 ? 4096 : (c > (1 << 22) ? (1 << 22) : c);
}

int64_t norm_blocks(int tensors, const int64_t* n, int64_t chunk) {
  int64_t b = 0;
  for (int i = 0; i < tensors; ++i)
    for (int64_t off = 0; off < n[i]; off += kOpPiece) {
      const int64_t k = n[i] - off < int64_t(kOpPiece) ? n[i] - off : int64_t(kOpPiece);
      b += (k + chunk - 1) / chunk;
    }
  return b;
}

gd_status check_sizes(const char* what, int tensors, const int64_t* n, int64_t* total) {
  GD_REQUIRE(tensors >= 0 && (tensors == 0 || n), "%s: %d tensors without their sizes", what, tensors);
  *total = 0;
  for (int i = 0; i < tensors; ++i) {
    GD_REQUIRE(n[i] >= 0 && n[i] <= (int64_t(1) << 40), "%s: tensor %d has %lld elements", what, i, (long long)n[i]);
    *total += n[i];
  }
  return GD_OK;
}

gd_status check_list(const char* what, const char* name, int tensors, const int64_t* n, const uint64_t* list,
                     uintptr_t align) {
  GD_REQUIRE(tensors == 0 || list, "%s: no %s", what, name);
  for (int i = 0; i < tensors; ++i)
    GD_REQUIRE(n[i] == 0 || (list[i] != 0 && list[i] % align == 0), "%s: %s %d is null or misaligned", what, name, i);
  return GD_OK;
}

#define GD_TRY(expr)                     \
  do {                                   \
    const gd_status _s = (expr);         \
    if (_s != GD_OK) return _s;          \
  } while (0)

}  // namespace
}  // namespace gd

using namespace gd;

extern "C" gd_status gd_adamw_step(int tensors, const int64_t* numel, const uint64_t* params, int grad_dtype,
                                   const uint64_t* grads, int state_bits, const uint64_t* exp_avgs,
                                   const uint64_t* exp_avg_sqs, const uint64_t* exp_avg_scales,
                                   const uint64_t* exp_avg_sq_scales, const uint64_t* copies,
                                   const uint64_t* steps_dev, double step, double lr, const float* lr_dev,
                                   double beta1, double beta2, double eps, double weight_decay,
                                   const float* total_norm, double max_norm, uint32_t seed, gd_stream_t stream) {
  const char* what = "adamw_step";
  int64_t total;
  GD_TRY(check_sizes(what, tensors, numel, &total));
  GD_REQUIRE(grad_dtype == GD_F32 || grad_dtype == GD_BF16, "%s: gradients in fp32 or bf16", what);
  GD_REQUIRE(state_bits == 32 || state_bits == 8, "%s: moments in 32 or 8 bits, not %d", what, state_bits);
  GD_REQUIRE(lr_dev || lr >= 0.0, "%s: lr=%g", what, lr);
  GD_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "%s: betas (%g, %g)", what, beta1, beta2);
  GD_REQUIRE(eps >= 0.0 && weight_decay >= 0.0, "%s: eps=%g weight_decay=%g", what, eps, weight_decay);
  GD_REQUIRE(steps_dev || step >= 1.0, "%s: step=%g (counted from 1)", what, step);
  GD_REQUIRE(!total_norm || max_norm > 0.0, "%s: max_norm=%g", what, max_norm);
  GD_TRY(check_list(what, "param", tensors, numel, params, 4));
  GD_TRY(check_list(what, "grad", tensors, numel, grads, grad_dtype == GD_F32 ? 4 : 2));
  GD_TRY(check_list(what, "exp_avg", tensors, numel, exp_avgs, state_bits == 8 ? 1 : 4));
  GD_TRY(check_list(what, "exp_avg_sq", tensors, numel, exp_avg_sqs, state_bits == 8 ? 1 : 4));
  if (state_bits == 8) {
    GD_TRY(check_list(what, "exp_avg_scale", tensors, numel, exp_avg_scales, 1));
    GD_TRY(check_list(what, "exp_avg_sq_scale", tensors, numel, exp_avg_sq_scales, 1));
  } else {
    GD_REQUIRE(!exp_avg_scales && !exp_avg_sq_scales, "%s: scales belong to moments in 8 bits", what);
  }
  if (copies) GD_TRY(check_list(what, "copy", tensors, numel, copies, 2));
  if (steps_dev) GD_TRY(check_list(what, "step", tensors, numel, steps_dev, 4));
  AdamConst c;
  c.beta1 = float(beta1);
  c.beta2 = float(beta2);
  c.one_minus_beta1 = float(1.0 - beta1);
  c.one_minus_beta2 = float(1.0 - beta2);
  c.eps = float(eps);
  c.weight_decay = float(weight_decay);
  c.lr = float(lr);
  c.log2_beta1 = std::log2(beta1);  // (-inf at 0: exp2 gives 0)
  c.log2_beta2 = std::log2(beta2);
  c.inv_bc1 = steps_dev ? 0.f : float(1.0 / (1.0 - std::pow(beta1, step)));
  c.inv_sqrt_bc2 = steps_dev ? 0.f : float(1.0 / std::sqrt(1.0 - std::pow(beta2, step)));
  c.max_norm = float(max_norm);
  c.lr_dev = lr_dev;
  c.total_norm = total_norm;
  c.seed = seed;
  c.key = steps_dev ? 0u : seed + uint32_t(int64_t(step)) * 0x85EBCA77u;
  const AdamLists l = {params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, copies, steps_dev,
                       numel, grad_dtype == GD_BF16};
  return l.grad_bf16 ? adamw_pick<uint16_t>(tensors, l, c, as_hip(stream))
                     : adamw_pick<float>(tensors, l, c, as_hip(stream));
}

extern "C" size_t gd_grad_norm_workspace_bytes(int tensors, const int64_t* numel) {
  int64_t total;
  if (check_sizes("grad_norm", tensors, numel, &total) != GD_OK) return 0;
  return size_t(norm_blocks(tensors, numel, norm_chunk(total))) * sizeof(double);
}

extern "C" gd_status gd_grad_norm(int tensors, const int64_t* numel, int dtype, const uint64_t* grads, void* workspace,
                                  size_t workspace_bytes, float* out, gd_stream_t stream) {
  const char* what = "grad_norm";
  int64_t total;
  GD_TRY(check_sizes(what, tensors, numel, &total));
  GD_REQUIRE(dtype == GD_F32 || dtype == GD_BF16, "%s: gradients in fp32 or bf16", what);
  GD_TRY(check_list(what, "grad", tensors, numel, grads, dtype == GD_F32 ? 4 : 2));
  GD_REQUIRE(out, "%s: null output", what);
  const int64_t chunk = norm_chunk(total), blocks = norm_blocks(tensors, numel, chunk);
  GD_REQUIRE(blocks < (int64_t(1) << 30), "%s: too many chunks", what);
  GD_REQUIRE(blocks == 0 || (workspace && op_aligned(workspace, 8) && workspace_bytes >= size_t(blocks) * sizeof(double)),
             "%s: workspace of %zu bytes, %lld wanted", what, workspace_bytes, (long long)(blocks * 8));
  hipStream_t s = as_hip(stream);
  NormTable t;
  static_assert(sizeof(t) <= 4000, "kernel arguments stay below 4 KB");
  t.chunk = uint32_t(chunk);
  t.entries = 0;
  t.partial = static_cast<double*>(workspace);
  uint32_t launched = 0;
  auto flush = [&]() -> gd_status {
    if (t.entries == 0) return GD_OK;
    if (dtype == GD_F32)
      hipLaunchKernelGGL(norm_chunk_kernel<float>, dim3(launched), dim3(kOpThreads), 0, s, t);
    else
      hipLaunchKernelGGL(norm_chunk_kernel<uint16_t>, dim3(launched), dim3(kOpThreads), 0, s, t);
    GD_LAUNCH_CHECK("grad_norm");
    t.partial += launched;
    t.entries = 0;
    launched = 0;
    return GD_OK;
  };
  const int elem = dtype == GD_F32 ? 4 : 2;
  for (int i = 0; i < tensors; ++i) {
    for (int64_t off = 0; off < numel[i]; off += kOpPiece) {
      const uint32_t n = uint32_t(numel[i] - off < int64_t(kOpPiece) ? numel[i] - off : int64_t(kOpPiece));
      const int e = t.entries++;
      t.g[e] = at<const char>(grads, i) + off * elem;
      t.n[e] = n | (op_aligned(t.g[e], 4 * elem) ? kOpAligned : 0u);
      t.first[e] = launched;
      launched += uint32_t((n + chunk - 1) / chunk);
      if (t.entries == NormTable::kCap) GD_TRY(flush());
    }
  }
  GD_TRY(flush());
  hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(kNormJoin), 0, s, static_cast<const double*>(workspace),
                     int(blocks), out);
  GD_LAUNCH_CHECK("grad_norm_join");
  return GD_OK;
}
