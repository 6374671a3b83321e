// ah_fp8_rows.cu — rows of activations to e4m3 with one f32 scale per 128
// columns: a plain quantiser, SwiGLU and quantise (inference/ffn.rs:155-174's
// activation), residual add, RMS norm (inference/math.rs:53-63) and quantise.
//
//   quantise:  g = max(max |z|, 2^-100) over the group, q = e4m3(z * (448 / g)), scale = g / 448
//   SwiGLU:    z = gate / (1 + exp(-gate)) * up
//   norm:      h = x + residual rounded to the residual's type, r = 1 / sqrt(mean h^2 + eps),
//              z = h * w, scale = g * r / 448
//
// The row's r scales every z of the row alike, so it leaves q unchanged and
// enters the scales alone: a norm row is quantised and stored in one pass over
// its data, without waiting for the row's sum.  All arithmetic is f32; each z
// is rounded once, to e4m3.
//
// Bound by HBM once there are rows enough: 16384 x 8192 bf16 with a residual 144 us
// (6.5 TB/s, a copy's rate), 2048 x 28672 bf16 SwiGLU 45 us (6.5 TB/s).  A group is 16 or
// 32 neighbouring lanes' 16-byte pieces, so its maximum is a few shuffles and nothing
// waits for another warp but a norm row's sum.  One row of 4096 takes 2.4 us, a launch's
// latency.  Without a residual the norm's arithmetic, the same for half the bytes, is the
// bound: 16384 x 8192 bf16 89 us (4.5 TB/s), 77 % of issue slots busy.
//
// Rows that do not start at multiples of 16 bytes are read by elements, at two thirds of
// the rate, or, 16-bit norm rows, cut out of aligned 16-byte words: 16384 x 8190 bf16 with a
// residual 276 us (by elements 400), without 149 (190).  f32 rows and the other two
// operators are faster by elements (16384 x 8190 SwiGLU 172 us against 181, 8192 x 8191 f32
// with a residual 164 against 234).
//
// A group's maximum keeps a NaN, and an infinite one has a NaN inverse: a group
// with a NaN or an infinity comes out as NaN.
#include <algorithm>

#include "ah_common.cuh"
#include "ah_fp8.cuh"
#include "ah_sm100.cuh"

namespace ah {
namespace {

enum RowMode { kRowQuantize, kRowSwiglu };

// kV columns = 16 bytes of T; 128 / kV neighbouring lanes hold one group.
template <typename T>
struct Vec {
  static constexpr int kV = 16 / (int)sizeof(T);
  static constexpr int kLanes = kFp8Group / kV;
};

// A 16-byte piece as f32 values, and back with one rounding.
__device__ __forceinline__ void unpack(const uint4& p, float (&v)[4], const float*) {
  v[0] = __uint_as_float(p.x); v[1] = __uint_as_float(p.y);
  v[2] = __uint_as_float(p.z); v[3] = __uint_as_float(p.w);
}
__device__ __forceinline__ void unpack(const uint4& p, float (&v)[8], const __half*) {
  const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack(const uint4& p, float (&v)[8], const __nv_bfloat16*) {
  const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <typename T>
__device__ __forceinline__ void unpack(const uint4& p, float (&v)[Vec<T>::kV]) {
  unpack(p, v, static_cast<const T*>(nullptr));
}
__device__ __forceinline__ uint4 pack(const float (&v)[4], const float*) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ uint4 pack(const float (&v)[8], const __half*) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&v)[8], const __nv_bfloat16*) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Bytes [off, off + 16) of the 32 bytes lo, hi (off < 16, a multiple of T's size).
__device__ __forceinline__ uint4 bytes_from(const uint4& lo, const uint4& hi, uint32_t off) {
  uint32_t v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) v[i] = off & 8 ? v[i + 2] : v[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) v[i] = off & 4 ? v[i + 1] : v[i];
  const uint32_t bits = (off & 3) * 8;
  return make_uint4(__funnelshift_r(v[0], v[1], bits), __funnelshift_r(v[1], v[2], bits),
                    __funnelshift_r(v[2], v[3], bits), __funnelshift_r(v[3], v[4], bits));
}

// Columns [c, c + kV) of a row of k columns as its 16 bytes (zero past the row).
// kVec: rows start at multiples of 16 bytes and k is a multiple of kV.  Otherwise it is
// read by elements or, kCut, cut out of the two aligned 16-byte words that hold it,
// except a row's first and last pieces, whose words reach past the row.  A word's other
// bytes, which a neighbour may be storing where the row is the residual, are dropped.
template <bool kVec, bool kCut, typename T>
__device__ __forceinline__ uint4 load_piece(const T* row, int c, int k) {
  constexpr int kV = Vec<T>::kV;
  uint4 p = make_uint4(0, 0, 0, 0);
  if constexpr (kVec) {
    if (c < k) p = *reinterpret_cast<const uint4*>(row + c);
    return p;
  }
  if constexpr (kCut) {
    const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15;  // the same for every piece of the row
    const int before = (int)(off / sizeof(T)), after = off ? kV - before : 0;
    if (c >= before && c + kV + after <= k) {
      const uint4* words = reinterpret_cast<const uint4*>(row + c - before);
      p = words[0];
      if (off) p = bytes_from(p, words[1], off);
      return p;
    }
  }
  T* e = reinterpret_cast<T*>(&p);
#pragma unroll
  for (int i = 0; i < kV; ++i)
    if (c + i < k) e[i] = row[c + i];
  return p;
}

// Stores a piece to columns [c, c + kV) of a row (c < k): the widest stores that the
// row's alignment has, elements at the end of a ragged row.
template <bool kVec, typename T>
__device__ __forceinline__ void store_piece(T* row, int c, int k, const uint4& p) {
  constexpr int kV = Vec<T>::kV;
  if constexpr (kVec) {
    *reinterpret_cast<uint4*>(row + c) = p;
    return;
  }
  const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15;
  T* e = row + c;
  const uint32_t w[4] = {p.x, p.y, p.z, p.w};
  if (c + kV > k) {
    const T* v = reinterpret_cast<const T*>(&p);
#pragma unroll
    for (int i = 0; i < kV; ++i)
      if (c + i < k) e[i] = v[i];
  } else if (off == 0) {
    *reinterpret_cast<uint4*>(e) = p;
  } else if (off % 8 == 0) {
    reinterpret_cast<uint2*>(e)[0] = make_uint2(w[0], w[1]);
    reinterpret_cast<uint2*>(e)[1] = make_uint2(w[2], w[3]);
  } else if (off % 4 == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(e)[i] = w[i];
  } else if constexpr (sizeof(T) == 2) {
    unsigned short* h = reinterpret_cast<unsigned short*>(e);
    h[0] = (unsigned short)w[0];
#pragma unroll
    for (int i = 0; i < 3; ++i) reinterpret_cast<uint32_t*>(h + 1)[i] = __funnelshift_r(w[i], w[i + 1], 16);
    h[7] = (unsigned short)(w[3] >> 16);
  }
}

// The group maximum of |z| (at least 2^-100) over the group's lanes.
template <typename T>
__device__ __forceinline__ float group_max(const float (&z)[Vec<T>::kV]) {
  float f = kFp8Tiny;
#pragma unroll
  for (int i = 0; i < Vec<T>::kV; i += 2) f = max_abs3(f, z[i], z[i + 1]);
  uint32_t a = __float_as_uint(f);  // a NaN's bits are above every number's
  if constexpr (Vec<T>::kLanes == 32) {
    a = __reduce_max_sync(0xFFFFFFFFu, a);
  } else {
#pragma unroll
    for (int o = Vec<T>::kLanes / 2; o; o >>= 1) a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, o));
  }
  return __uint_as_float(a);
}

// q bytes of columns [c, c + kV): one 4- or 8-byte store (ldq and q are
// multiples of 16 bytes), bytes at the end of a ragged row.
template <bool kVec, int kV>
__device__ __forceinline__ void store_q(uint8_t* qrow, int c, int k, const float (&z)[kV], float inv) {
  uint32_t w[kV / 4];
#pragma unroll
  for (int i = 0; i < kV / 4; ++i)
    w[i] = cvt_e4m3x4(z[4 * i] * inv, z[4 * i + 1] * inv, z[4 * i + 2] * inv, z[4 * i + 3] * inv);
  if (kVec || c + kV <= k) {
    if constexpr (kV == 4)
      *reinterpret_cast<uint32_t*>(qrow + c) = w[0];
    else
      *reinterpret_cast<uint2*>(qrow + c) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i)
      if (c + i < k) qrow[c + i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
  }
}

struct RowArgs {
  const void* a;  // x, or gate
  const void* b;  // up
  int64_t lda, ldb;
  int64_t m;
  int k;
  uint8_t* q;
  int64_t ldq;
  float* scales;
  int64_t lds;
};

constexpr int kRowThreads = 256;

// One row and 256 * kN * kV columns per CTA, or kNarrow: kN * blockDim.y rows of one piece
// per thread (blockDim.x is a multiple of 32).  A thread requests its kN pieces of
// every input before it uses the first.  SwiGLU is held to the registers of a full SM
// (kN == 1) or of six CTAs: 16384 x 2048 bf16 30.0 us, 33.8 with those it would take.
template <int kMode, typename T, bool kVec, bool kNarrow, int kN>
__global__ void __launch_bounds__(kRowThreads, kMode != kRowSwiglu ? 0 : kN == 1 ? 8 : 6) k_fp8_rows(const RowArgs g) {
  constexpr int kV = Vec<T>::kV;
  pdl_launch_dependents();
  pdl_wait();
  const int ty = kNarrow ? (int)blockDim.y : 1, rows = kNarrow ? kN * ty : 1;
  const int c0 = (kNarrow ? (int)threadIdx.x : (int)(blockIdx.x * kN * kRowThreads + threadIdx.x)) * kV;
  for (int64_t r0 = (int64_t)blockIdx.y * rows + (kNarrow ? threadIdx.y : 0); r0 < g.m; r0 += (int64_t)gridDim.y * rows) {
    uint4 pa[kN], pb[kMode == kRowSwiglu ? kN : 1];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int64_t row = kNarrow ? min(r0 + i * ty, g.m - 1) : r0;  // past the last row: read, not stored
      const int c = kNarrow ? c0 : c0 + i * kRowThreads * kV;
      pa[i] = load_piece<kVec, false>(static_cast<const T*>(g.a) + row * g.lda, c, g.k);
      if constexpr (kMode == kRowSwiglu)
        pb[i] = load_piece<kVec, false>(static_cast<const T*>(g.b) + row * g.ldb, c, g.k);
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int64_t row = kNarrow ? r0 + i * ty : r0;
      const int c = kNarrow ? c0 : c0 + i * kRowThreads * kV;
      float z[kV];
      unpack<T>(pa[i], z);
      if constexpr (kMode == kRowSwiglu) {
        float u[kV];
        unpack<T>(pb[i], u);
        fp8_silu_mul(z, u, z);
      }
      const float gm = group_max<T>(z);
      if (c < g.k && row < g.m) {
        store_q<kVec>(g.q + row * g.ldq, c, g.k, z, fp8_inverse(gm));
        if (c % kFp8Group == 0) g.scales[row * g.lds + c / kFp8Group] = gm * (1.0f / kFp8Max);
      }
    }
  }
}

struct NormArgs {
  const void* x;
  void* residual;
  const void* w;
  int64_t ldx, ldr;
  int64_t m;
  int k;
  uint8_t* q;
  int64_t ldq;
  float* scales;
  int64_t lds;
  uint32_t w_dtype;
  bool w_aligned;
  float eps;
};

// Norm weights of columns [c, c + kV), zero past the row; by elements at the end of a
// ragged row and where w is not 16-byte aligned (kVec: neither occurs).
template <bool kVec, int kV>
__device__ __forceinline__ void norm_weights(const NormArgs& g, int c, float (&w)[kV]) {
  if (kVec ? c < g.k : g.w_aligned && c + kV <= g.k) {
    if (g.w_dtype == AH_DTYPE_F32) {
#pragma unroll
      for (int i = 0; i < kV; i += 4) {
        const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(g.w) + c + i);
        w[i] = f.x; w[i + 1] = f.y; w[i + 2] = f.z; w[i + 3] = f.w;
      }
    } else {
      uint32_t b[kV / 2];
      const unsigned short* p = static_cast<const unsigned short*>(g.w) + c;
      if constexpr (kV == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        b[0] = v.x; b[1] = v.y;
      } else {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        b[0] = v.x; b[1] = v.y; b[2] = v.z; b[3] = v.w;
      }
#pragma unroll
      for (int i = 0; i < kV / 2; ++i) {
        const float2 f = g.w_dtype == AH_DTYPE_F16
                             ? __half22float2(*reinterpret_cast<const __half2*>(&b[i]))
                             : make_float2(__uint_as_float(b[i] << 16), __uint_as_float(b[i] & 0xFFFF0000u));
        w[2 * i] = f.x;
        w[2 * i + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      if (kVec || c + i >= g.k) {
        w[i] = 0.0f;
      } else if (g.w_dtype == AH_DTYPE_F32) {
        w[i] = static_cast<const float*>(g.w)[c + i];
      } else {
        const unsigned short b = static_cast<const unsigned short*>(g.w)[c + i];
        w[i] = g.w_dtype == AH_DTYPE_F16 ? __half2float(__ushort_as_half(b)) : __uint_as_float((uint32_t)b << 16);
      }
    }
  }
}

// One row per threadIdx.y: blockDim.x threads take kN pieces each per sweep (one
// sweep for most widths).  Several rows share a CTA only where a warp takes a row.
template <typename T, bool kVec, bool kRes, int kN>
__global__ void __launch_bounds__(kN == 1 ? 1024 : 512, kN == 1 ? 1 : 2) k_fp8_norm(const NormArgs g) {
  constexpr int kV = Vec<T>::kV;
  constexpr bool kCut = sizeof(T) == 2;  // both sides measured: at the top of this file
  __shared__ float red[32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= g.m) return;  // a whole warp: CTAs of one row have no such row
  const T* xrow = static_cast<const T*>(g.x) + row * g.ldx;
  T* rrow = static_cast<T*>(g.residual) + row * g.ldr;
  float* scales = g.scales + row * g.lds;
  const int sweep = (int)blockDim.x * kN * kV;
  float ss = 0.0f, gm[kN];
  for (int s = 0; s < g.k; s += sweep) {
    uint4 px[kN], pr[kRes ? kN : 1];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int c = s + (int)(i * blockDim.x + threadIdx.x) * kV;
      px[i] = load_piece<kVec, kCut>(xrow, c, g.k);
      if constexpr (kRes) pr[i] = load_piece<kVec, kCut, T>(rrow, c, g.k);
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int c = s + (int)(i * blockDim.x + threadIdx.x) * kV;
      float h[kV], w[kV];
      unpack<T>(px[i], h);
      if constexpr (kRes) {
        float r[kV];
        unpack<T>(pr[i], r);
#pragma unroll
        for (int j = 0; j < kV; ++j) h[j] += r[j];
        const uint4 p = pack(h, static_cast<const T*>(nullptr));
        unpack<T>(p, h);
        if (c < g.k) store_piece<kVec>(rrow, c, g.k, p);
      }
      norm_weights<kVec>(g, c, w);
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        ss = fmaf(h[j], h[j], ss);
        h[j] *= w[j];
      }
      gm[i] = group_max<T>(h);
      if (c < g.k) {
        store_q<kVec>(g.q + row * g.ldq, c, g.k, h, fp8_inverse(gm[i]));
        // more than one sweep: the maximum waits for r in the scales themselves
        if (sweep < g.k && c % kFp8Group == 0) scales[c / kFp8Group] = gm[i];
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
  if (blockDim.x > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
    __syncthreads();
    // every warp adds the partial sums in the same order
    ss = threadIdx.x % 32 < blockDim.x / 32 ? red[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
  }
  const float r = __fdiv_rn(1.0f, sqrtf(__fdiv_rn(ss, (float)g.k) + g.eps)) * (1.0f / kFp8Max);
  if (sweep >= g.k) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int c = (int)(i * blockDim.x + threadIdx.x) * kV;
      if (c < g.k && c % kFp8Group == 0) scales[c / kFp8Group] = gm[i] * r;
    }
  } else {
    for (int c = (int)threadIdx.x * kV; c < g.k; c += (int)blockDim.x * kV)
      if (c % kFp8Group == 0) scales[c / kFp8Group] *= r;  // this thread's own store
  }
}

int check_rows(const char* who, int64_t m, int64_t k, const void* q, int64_t ldq, const void* scales, int64_t lds,
               uint32_t dtype) {
  AH_REQUIRE(m >= 0 && k >= 1, "%s: needs m >= 0 rows of k >= 1 columns", who);
  AH_REQUIRE(m <= 0x7FFFFFFF && k < (1 << 30), "%s: m must be below 2^31 and k below 2^30", who);
  AH_REQUIRE(dtype == AH_DTYPE_F32 || dtype == AH_DTYPE_F16 || dtype == AH_DTYPE_BF16,
             "%s: dtype %u is not f32, f16 or bf16", who, dtype);
  AH_REQUIRE(m == 0 || (q && scales), "%s: null pointer", who);
  AH_REQUIRE(aligned16(q) && ldq % 16 == 0 && ldq >= k, "%s: q rows must start at multiples of 16 bytes, ldq >= k",
             who);
  AH_REQUIRE(lds >= fp8_groups(k), "%s: lds must be at least ceil(k / 128)", who);
  AH_REQUIRE(element_aligned(scales, AH_DTYPE_F32), "%s: scales are not aligned to their elements", who);
  return AH_OK;
}

bool vec_rows(const void* p, int64_t ld, uint32_t dtype) {
  return aligned16(p) && ld * (dtype == AH_DTYPE_F32 ? 4 : 2) % 16 == 0;
}

template <int kMode, typename T>
int launch_rows(const RowArgs& g, bool vec, cudaStream_t st) {
  const int64_t pieces = (g.k + Vec<T>::kV - 1) / Vec<T>::kV;
  vec = vec && g.k % Vec<T>::kV == 0;
  if (pieces <= kRowThreads) {
    // Narrow rows share a CTA, and a thread takes a piece of kRows rows once that leaves every
    // SM four CTAs.  16384 x 2048 bf16 quantise: 18.8 us with four, 20.8 with two, 24.6 with
    // one; 16384 x 1024 f32 SwiGLU 29.8, 23.3, 24.3; bf16 SwiGLU 16384 x 2048 39.7, 29.2, 30.0,
    // 16384 x 512 14.6, 9.2, 9.0.
    constexpr int kRows = kMode == kRowQuantize ? 4 : sizeof(T) == 4 ? 2 : 1;
    const unsigned tx = (unsigned)((pieces + 31) / 32 * 32), ty = kRowThreads / tx;
    const bool many = vec && g.m >= (int64_t)kRows * ty * 4 * sm_count();
    const int64_t rows = (many ? kRows : 1) * ty;
    const dim3 grid(1, (unsigned)std::min<int64_t>((g.m + rows - 1) / rows, 65535));
    return launch_pdl(many ? k_fp8_rows<kMode, T, true, true, kRows>
                      : vec ? k_fp8_rows<kMode, T, true, true, 1> : k_fp8_rows<kMode, T, false, true, 1>,
                      grid, dim3(tx, ty), 0, st, g);
  }
  // Wide ones take two pieces per thread once that still leaves every SM four CTAs
  // (16384 x 8192 bf16 SwiGLU: 100 us with two, 117 with one).
  const bool many = vec && g.m * ((pieces + 2 * kRowThreads - 1) / (2 * kRowThreads)) >= 4 * (int64_t)sm_count();
  const int64_t cols = (int64_t)kRowThreads * (many ? 2 : 1);
  const dim3 grid((unsigned)((pieces + cols - 1) / cols), (unsigned)std::min<int64_t>(g.m, 65535));
  return launch_pdl(many ? k_fp8_rows<kMode, T, true, false, 2>
                    : vec ? k_fp8_rows<kMode, T, true, false, 1> : k_fp8_rows<kMode, T, false, false, 1>,
                    grid, dim3(kRowThreads), 0, st, g);
}

template <int kMode>
int dispatch_rows(const RowArgs& g, uint32_t dtype, bool vec, cudaStream_t st) {
  if (dtype == AH_DTYPE_F32) return launch_rows<kMode, float>(g, vec, st);
  if (dtype == AH_DTYPE_F16) return launch_rows<kMode, __half>(g, vec, st);
  return launch_rows<kMode, __nv_bfloat16>(g, vec, st);
}

template <typename T, bool kRes>
int launch_norm(const NormArgs& g, bool vec, cudaStream_t st) {
  // Few rows: one piece per thread, up to 1024 threads, for the latency of one
  // round of loads.  Many rows: few threads per row and many pieces each, so that a
  // row's sum costs little and many rows are in flight (16384 x 8192 bf16 with a
  // residual: 144 us with four pieces, 199 with eight, 169 with two, 271 with one); without
  // the residual's registers, eight (89 us, with four 95).
  constexpr int kMany = kRes ? 4 : 8;
  const int64_t pieces = (g.k + Vec<T>::kV - 1) / Vec<T>::kV;
  vec = vec && g.k % Vec<T>::kV == 0;
  const bool many = g.m > 2 * (int64_t)sm_count();
  const int n = !many ? 1 : pieces <= (vec ? 64 : 256) ? 2 : kMany;
  const unsigned tx = (unsigned)std::min<int64_t>(n == 1 ? 1024 : 512, ((pieces + n - 1) / n + 31) / 32 * 32);
  const unsigned ty = tx == 32 ? 8 : 1;
  auto kernel = vec ? (n == 1 ? k_fp8_norm<T, true, kRes, 1>
                       : n == 2 ? k_fp8_norm<T, true, kRes, 2> : k_fp8_norm<T, true, kRes, kMany>)
                    : (n == 1 ? k_fp8_norm<T, false, kRes, 1>
                       : n == 2 ? k_fp8_norm<T, false, kRes, 2> : k_fp8_norm<T, false, kRes, kMany>);
  return launch_pdl(kernel, dim3((unsigned)((g.m + ty - 1) / ty)), dim3(tx, ty), 0, st, g);
}

template <typename T>
int dispatch_norm(const NormArgs& g, bool vec, cudaStream_t st) {
  return g.residual ? launch_norm<T, true>(g, vec, st) : launch_norm<T, false>(g, vec, st);
}

}  // namespace
}  // namespace ah

using namespace ah;

extern "C" {

int ah_fp8_quantize(const void* x, int64_t ldx, uint32_t dtype, int64_t m, int64_t k, uint8_t* q, int64_t ldq,
                    float* scales, int64_t lds, void* stream) {
  const int rc = check_rows("fp8_quantize", m, k, q, ldq, scales, lds, dtype);
  if (rc != AH_OK || m == 0) return rc;
  AH_REQUIRE(x && ldx >= k, "fp8_quantize: null x or ldx below k");
  AH_REQUIRE(element_aligned(x, dtype), "fp8_quantize: x is not aligned to its elements");
  const RowArgs g{x, nullptr, ldx, 0, m, (int)k, q, ldq, scales, lds};
  return dispatch_rows<kRowQuantize>(g, dtype, vec_rows(x, ldx, dtype), as_stream(stream));
}

int ah_fp8_swiglu(const void* gate, int64_t ld_gate, const void* up, int64_t ld_up, uint32_t dtype, int64_t m,
                  int64_t k, uint8_t* q, int64_t ldq, float* scales, int64_t lds, void* stream) {
  const int rc = check_rows("fp8_swiglu", m, k, q, ldq, scales, lds, dtype);
  if (rc != AH_OK || m == 0) return rc;
  AH_REQUIRE(gate && up && ld_gate >= k && ld_up >= k, "fp8_swiglu: null input or a row stride below k");
  AH_REQUIRE(element_aligned(gate, dtype) && element_aligned(up, dtype),
             "fp8_swiglu: an input is not aligned to its elements");
  const RowArgs g{gate, up, ld_gate, ld_up, m, (int)k, q, ldq, scales, lds};
  return dispatch_rows<kRowSwiglu>(g, dtype, vec_rows(gate, ld_gate, dtype) && vec_rows(up, ld_up, dtype),
                                   as_stream(stream));
}

int ah_fp8_add_rms_norm(const void* x, int64_t ldx, void* residual, int64_t ldr, uint32_t dtype, const void* norm_w,
                        uint32_t norm_dtype, float eps, int64_t m, int64_t k, uint8_t* q, int64_t ldq, float* scales,
                        int64_t lds, void* stream) {
  const int rc = check_rows("fp8_add_rms_norm", m, k, q, ldq, scales, lds, dtype);
  if (rc != AH_OK || m == 0) return rc;
  AH_REQUIRE(x && norm_w && ldx >= k, "fp8_add_rms_norm: null input or ldx below k");
  AH_REQUIRE(!residual || ldr >= k, "fp8_add_rms_norm: ldr below k");
  AH_REQUIRE(norm_dtype == AH_DTYPE_F32 || norm_dtype == AH_DTYPE_F16 || norm_dtype == AH_DTYPE_BF16,
             "fp8_add_rms_norm: norm weight dtype %u is not f32, f16 or bf16", norm_dtype);
  AH_REQUIRE(element_aligned(x, dtype) && element_aligned(residual, dtype) && element_aligned(norm_w, norm_dtype),
             "fp8_add_rms_norm: an input is not aligned to its elements");
  AH_REQUIRE(eps >= 0.0f, "fp8_add_rms_norm: eps must be >= 0");
  const NormArgs g{x, residual, norm_w, ldx, ldr, m, (int)k, q, ldq, scales, lds, norm_dtype, aligned16(norm_w), eps};
  const bool vec = vec_rows(x, ldx, dtype) && (!residual || vec_rows(residual, ldr, dtype)) && g.w_aligned;
  if (dtype == AH_DTYPE_F32) return dispatch_norm<float>(g, vec, as_stream(stream));
  if (dtype == AH_DTYPE_F16) return dispatch_norm<__half>(g, vec, as_stream(stream));
  return dispatch_norm<__nv_bfloat16>(g, vec, as_stream(stream));
}

}  // extern "C"
