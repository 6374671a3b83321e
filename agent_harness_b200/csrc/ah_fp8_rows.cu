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
// A group's maximum is taken on the bits of |z|, where a NaN is above every
// number: a group with a NaN or an infinity comes out as NaN.
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

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Columns [c, c + kV) of a row of k columns (zero past it).  `vec`: row + c is
// 16-byte aligned and the piece lies inside the row.
template <typename T>
__device__ __forceinline__ void load_piece(const T* row, int64_t c, int64_t k, bool vec, float (&v)[Vec<T>::kV]) {
  if (vec) {
    const uint4 p = *reinterpret_cast<const uint4*>(row + c);
    const T* e = reinterpret_cast<const T*>(&p);
#pragma unroll
    for (int i = 0; i < Vec<T>::kV; ++i) v[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < Vec<T>::kV; ++i) v[i] = c + i < k ? to_f32(row[c + i]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store_piece(T* row, int64_t c, int64_t k, bool vec, const float (&v)[Vec<T>::kV]) {
  if (vec) {
    uint4 p;
    T* e = reinterpret_cast<T*>(&p);
#pragma unroll
    for (int i = 0; i < Vec<T>::kV; ++i) e[i] = from_f32<T>(v[i]);
    *reinterpret_cast<uint4*>(row + c) = p;
  } else {
#pragma unroll
    for (int i = 0; i < Vec<T>::kV; ++i)
      if (c + i < k) row[c + i] = from_f32<T>(v[i]);
  }
}

// The group maximum of |z| (at least 2^-100) over the group's lanes.
template <typename T>
__device__ __forceinline__ float group_max(const float (&z)[Vec<T>::kV]) {
  uint32_t a = __float_as_uint(kFp8Tiny);
#pragma unroll
  for (int i = 0; i < Vec<T>::kV; ++i) a = max(a, __float_as_uint(z[i]) & 0x7FFFFFFFu);
#pragma unroll
  for (int o = Vec<T>::kLanes / 2; o; o >>= 1) a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, o));
  return __uint_as_float(a);
}

// q bytes of columns [c, c + kV): one 4- or 8-byte store (ldq and q are
// multiples of 16 bytes), bytes at the end of a ragged row.
template <int kV>
__device__ __forceinline__ void store_q(uint8_t* qrow, int64_t c, int64_t k, const float (&z)[kV], float inv) {
  uint32_t w[kV / 4];
#pragma unroll
  for (int i = 0; i < kV / 4; ++i)
    w[i] = cvt_e4m3x4(z[4 * i] * inv, z[4 * i + 1] * inv, z[4 * i + 2] * inv, z[4 * i + 3] * inv);
  if (c + kV <= k) {
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
  int64_t m, k;
  uint8_t* q;
  int64_t ldq;
  float* scales;
  int64_t lds;
  bool vec;  // a and b rows start at multiples of 16 bytes
};

constexpr int kRowThreads = 256;

// One CTA per row and 256 * kV columns.
template <int kMode, typename T>
__global__ void __launch_bounds__(kRowThreads) k_fp8_rows(const RowArgs g) {
  constexpr int kV = Vec<T>::kV;
  const int64_t c = ((int64_t)blockIdx.x * kRowThreads + threadIdx.x) * kV;
  for (int64_t row = blockIdx.y; row < g.m; row += gridDim.y) {
    const bool vec = g.vec && c + kV <= g.k;
    float z[kV];
    load_piece(static_cast<const T*>(g.a) + row * g.lda, c, g.k, vec, z);
    if (kMode == kRowSwiglu) {
      float u[kV];
      load_piece(static_cast<const T*>(g.b) + row * g.ldb, c, g.k, vec, u);
#pragma unroll
      for (int i = 0; i < kV; ++i) z[i] = fp8_silu_mul(z[i], u[i]);
    }
    const float gm = group_max<T>(z);
    if (c < g.k) {
      store_q<kV>(g.q + row * g.ldq, c, g.k, z, __fdiv_rn(kFp8Max, gm));
      if (c % kFp8Group == 0) g.scales[row * g.lds + c / kFp8Group] = gm * (1.0f / kFp8Max);
    }
  }
}

struct NormArgs {
  const void* x;
  void* residual;
  const void* w;
  int64_t ldx, ldr;
  int64_t m, k;
  uint8_t* q;
  int64_t ldq;
  float* scales;
  int64_t lds;
  uint32_t w_dtype;
  float eps;
  bool vec;  // x, residual and w rows start at multiples of 16 bytes
};

__device__ __forceinline__ float norm_weight(const void* w, uint32_t dtype, int64_t c) {
  if (dtype == AH_DTYPE_F32) return static_cast<const float*>(w)[c];
  const unsigned short b = static_cast<const unsigned short*>(w)[c];
  return dtype == AH_DTYPE_F16 ? __half2float(__ushort_as_half(b)) : __uint_as_float((uint32_t)b << 16);
}

// One CTA per row.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) k_fp8_norm(const NormArgs g) {
  constexpr int kV = Vec<T>::kV;
  __shared__ float red[kRowThreads / 32];
  const int64_t row = blockIdx.x;
  float* scales = g.scales + row * g.lds;
  float ss = 0.0f;
  const int64_t sweep = (int64_t)kRowThreads * kV;
  for (int64_t c0 = 0; c0 < g.k; c0 += sweep) {
    const int64_t c = c0 + (int64_t)threadIdx.x * kV;
    const bool vec = g.vec && c + kV <= g.k;
    float h[kV];
    load_piece(static_cast<const T*>(g.x) + row * g.ldx, c, g.k, vec, h);
    if (g.residual) {
      T* rrow = static_cast<T*>(g.residual) + row * g.ldr;
      float r[kV];
      load_piece<T>(rrow, c, g.k, vec, r);
#pragma unroll
      for (int i = 0; i < kV; ++i) h[i] = to_f32(from_f32<T>(h[i] + r[i]));
      store_piece(rrow, c, g.k, vec, h);
    }
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      ss = fmaf(h[i], h[i], ss);
      h[i] *= c + i < g.k ? norm_weight(g.w, g.w_dtype, c + i) : 0.0f;
    }
    const float gm = group_max<T>(h);
    if (c < g.k) {
      store_q<kV>(g.q + row * g.ldq, c, g.k, h, __fdiv_rn(kFp8Max, gm));
      if (c % kFp8Group == 0) scales[c / kFp8Group] = gm * (1.0f / kFp8Max);  // times r below
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  ss = red[0];
#pragma unroll
  for (int i = 1; i < kRowThreads / 32; ++i) ss += red[i];
  const float r = __fdiv_rn(1.0f, sqrtf(__fdiv_rn(ss, (float)g.k) + g.eps));
  for (int64_t c = (int64_t)threadIdx.x * kV; c < g.k; c += sweep)
    if (c % kFp8Group == 0) scales[c / kFp8Group] *= r;  // this thread's own store
}

int check_rows(const char* who, int64_t m, int64_t k, const void* q, int64_t ldq, const void* scales, int64_t lds,
               uint32_t dtype) {
  AH_REQUIRE(m >= 0 && k >= 1, "%s: needs m >= 0 rows of k >= 1 columns", who);
  AH_REQUIRE(m <= 0x7FFFFFFF && k <= 0x7FFFFFFF, "%s: m and k must be below 2^31", who);
  AH_REQUIRE(dtype == AH_DTYPE_F32 || dtype == AH_DTYPE_F16 || dtype == AH_DTYPE_BF16,
             "%s: dtype %u is not f32, f16 or bf16", who, dtype);
  AH_REQUIRE(m == 0 || (q && scales), "%s: null pointer", who);
  AH_REQUIRE(aligned16(q) && ldq % 16 == 0 && ldq >= k, "%s: q rows must start at multiples of 16 bytes, ldq >= k",
             who);
  AH_REQUIRE(lds >= fp8_groups(k), "%s: lds must be at least ceil(k / 128)", who);
  return AH_OK;
}

bool vec_rows(const void* p, int64_t ld, uint32_t dtype) {
  return aligned16(p) && ld * (dtype == AH_DTYPE_F32 ? 4 : 2) % 16 == 0;
}

template <int kMode, typename T>
int launch_rows(const RowArgs& g, cudaStream_t st) {
  const int64_t cols = (int64_t)kRowThreads * Vec<T>::kV;
  const dim3 grid((unsigned)((g.k + cols - 1) / cols), (unsigned)(g.m < 65535 ? g.m : 65535));
  k_fp8_rows<kMode, T><<<grid, kRowThreads, 0, st>>>(g);
  AH_LAUNCH_CHECK();
  return AH_OK;
}

template <int kMode>
int dispatch_rows(const RowArgs& g, uint32_t dtype, cudaStream_t st) {
  if (dtype == AH_DTYPE_F32) return launch_rows<kMode, float>(g, st);
  if (dtype == AH_DTYPE_F16) return launch_rows<kMode, __half>(g, st);
  return launch_rows<kMode, __nv_bfloat16>(g, st);
}

template <typename T>
int launch_norm(const NormArgs& g, cudaStream_t st) {
  k_fp8_norm<T><<<(unsigned)g.m, kRowThreads, 0, st>>>(g);
  AH_LAUNCH_CHECK();
  return AH_OK;
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
  RowArgs g{x, nullptr, ldx, 0, m, k, q, ldq, scales, lds, vec_rows(x, ldx, dtype)};
  return dispatch_rows<kRowQuantize>(g, dtype, as_stream(stream));
}

int ah_fp8_swiglu(const void* gate, int64_t ld_gate, const void* up, int64_t ld_up, uint32_t dtype, int64_t m,
                  int64_t k, uint8_t* q, int64_t ldq, float* scales, int64_t lds, void* stream) {
  const int rc = check_rows("fp8_swiglu", m, k, q, ldq, scales, lds, dtype);
  if (rc != AH_OK || m == 0) return rc;
  AH_REQUIRE(gate && up && ld_gate >= k && ld_up >= k, "fp8_swiglu: null input or a row stride below k");
  RowArgs g{gate, up, ld_gate, ld_up, m, k, q, ldq, scales, lds,
            vec_rows(gate, ld_gate, dtype) && vec_rows(up, ld_up, dtype)};
  return dispatch_rows<kRowSwiglu>(g, dtype, as_stream(stream));
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
  AH_REQUIRE(eps >= 0.0f, "fp8_add_rms_norm: eps must be >= 0");
  NormArgs g{x, residual, norm_w, ldx, ldr, m, k, q, ldq, scales, lds, norm_dtype, eps,
             vec_rows(x, ldx, dtype) && (!residual || vec_rows(residual, ldr, dtype))};
  if (dtype == AH_DTYPE_F32) return launch_norm<float>(g, as_stream(stream));
  if (dtype == AH_DTYPE_F16) return launch_norm<__half>(g, as_stream(stream));
  return launch_norm<__nv_bfloat16>(g, as_stream(stream));
}

}  // extern "C"
