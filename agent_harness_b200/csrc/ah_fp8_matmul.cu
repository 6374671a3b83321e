// ah_fp8_matmul.cu — resident e4m3 weights and their products with quantised
// activations:
//
//   y[i][r] = sum_b a_scale[i][b] * w_scale[r / 128][b] * sum_{j in block b} a[i][j] * w[r][j]
//
// b runs over the blocks of 128 columns.  The inner sums are exact products
// summed in f32; the scales multiply each block's sum in f32.
#include <mutex>
#include <new>

#include "ah_common.cuh"
#include "ah_fp8.cuh"
#include "ah_sm100.cuh"

namespace ah {
namespace {

// ---- building a weight ------------------------------------------------------------

struct TileSource {
  const void* p;  // e4m3 rows, or float rows to quantise
  int64_t ld;
  const float* scales;
  int64_t lds;
};

// Source of tile t: rows [row0, row0 + 128) of s[which].
__device__ __forceinline__ const TileSource& tile_source(const TileSource (&s)[2], bool gate_up, int64_t t,
                                                         int64_t& row0) {
  row0 = (gate_up ? t >> 1 : t) * kFp8Group;
  return s[gate_up ? t & 1 : 0];
}

struct BuildArgs {
  TileSource s[2];
  int64_t rows, cols;  // rows of one source
  uint8_t* tiles;
  float* scales;
  int64_t nt, kb;
  bool gate_up;
};

// Copies one 128 x 128 block of e4m3 bytes into its tile image (one CTA per
// block: x = column block, y = tile).  Runs once per weight.
__global__ void __launch_bounds__(256) k_fp8w_copy(const BuildArgs g) {
  const int64_t b = blockIdx.x;
  for (int64_t t = blockIdx.y; t < g.nt; t += gridDim.y) {
    int64_t row0;
    const TileSource& s = tile_source(g.s, g.gate_up, t, row0);
    const uint8_t* src = static_cast<const uint8_t*>(s.p);
    uint8_t* dst = g.tiles + (t * g.kb + b) * kFp8TileBytes;
    const bool aligned = (reinterpret_cast<uintptr_t>(src) & 15) == 0 && s.ld % 16 == 0;
    for (int i = threadIdx.x; i < kFp8TileBytes / 16; i += 256) {
      const int r = i >> 3, p = i & 7;
      const int64_t row = row0 + r, col = b * kFp8Group + p * 16;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (row < g.rows) {
        const uint8_t* e = src + row * s.ld + col;
        if (aligned && col + 16 <= g.cols) {
          v = *reinterpret_cast<const uint4*>(e);
        } else {
          uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (col + j < g.cols) w[j / 4] |= (uint32_t)e[j] << (8 * (j % 4));
          v = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      *reinterpret_cast<uint4*>(dst + r * 128 + ((p ^ (r & 7)) << 4)) = v;
    }
    if (threadIdx.x == 0) g.scales[t * g.kb + b] = s.scales[(row0 / kFp8Group) * s.lds + b];
  }
}

// Quantises one 128 x 128 block: scale = max(max |w|, 2^-100) / 448, q = e4m3(w * (448 / max)).
template <typename T>
__global__ void __launch_bounds__(256) k_fp8w_quantize(const BuildArgs g) {
  __shared__ uint32_t red[8];
  const int64_t b = blockIdx.x;
  const int r0 = threadIdx.x >> 3, p = threadIdx.x & 7;  // piece p of rows r0, r0 + 32, ...
  for (int64_t t = blockIdx.y; t < g.nt; t += gridDim.y) {
    int64_t row0;
    const TileSource& s = tile_source(g.s, g.gate_up, t, row0);
    float v[4][16];
    uint32_t a = __float_as_uint(kFp8Tiny);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = row0 + r0 + 32 * i, col = b * kFp8Group + p * 16;
      const T* e = static_cast<const T*>(s.p) + row * s.ld + col;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        v[i][j] = row < g.rows && col + j < g.cols ? (float)e[j] : 0.0f;
        a = max(a, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);  // a NaN is above every number
      }
    }
    a = __reduce_max_sync(0xFFFFFFFFu, a);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, red[i]);
    const float gm = __uint_as_float(a), inv = __fdiv_rn(kFp8Max, gm);
    uint8_t* dst = g.tiles + (t * g.kb + b) * kFp8TileBytes;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + 32 * i;
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = cvt_e4m3x4(v[i][4 * j] * inv, v[i][4 * j + 1] * inv, v[i][4 * j + 2] * inv, v[i][4 * j + 3] * inv);
      *reinterpret_cast<uint4*>(dst + r * 128 + ((p ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (threadIdx.x == 0) g.scales[t * g.kb + b] = gm * (1.0f / kFp8Max);
  }
}

enum SourceKind { kSourceE4m3, kSourceF32, kSourceF16, kSourceBf16 };

int source_kind(uint32_t dtype) {
  return dtype == AH_DTYPE_F32 ? kSourceF32 : dtype == AH_DTYPE_F16 ? kSourceF16 : dtype == AH_DTYPE_BF16 ? kSourceBf16 : -1;
}

void destroy(AhFp8Weight* w) {
  int cur = 0;
  cudaGetDevice(&cur);
  cudaSetDevice(w->device);
  cudaFree(w->tiles);
  cudaSetDevice(cur);
  delete w;
}

int build(const TileSource (&s)[2], int kind, bool gate_up, int64_t rows, int64_t cols, AhFp8Weight** out,
          cudaStream_t st) {
  AH_REQUIRE(out, "fp8w: null handle pointer");
  *out = nullptr;
  AH_REQUIRE(kind >= 0, "fp8w: the weight's dtype is not f32, f16 or bf16");
  AH_REQUIRE(rows >= 1 && cols >= 1 && rows <= 0x3FFFFFFF && cols <= 0x3FFFFFFF,
             "fp8w: rows and cols must be 1 .. 2^30 - 1");
  for (int i = 0; i < (gate_up ? 2 : 1); ++i) {
    AH_REQUIRE(s[i].p && s[i].ld >= cols, "fp8w: null source or a row stride below cols");
    AH_REQUIRE(kind != kSourceE4m3 || (s[i].scales && s[i].lds >= fp8_groups(cols)),
               "fp8w: null scales or a scale row stride below ceil(cols / 128)");
  }
  AhFp8Weight* w = new (std::nothrow) AhFp8Weight();
  if (!w) return fail(AH_ENOMEM, "fp8w: out of host memory");
  w->rows = gate_up ? 2 * rows : rows;
  w->cols = cols;
  w->nt = fp8_groups(rows) * (gate_up ? 2 : 1);
  w->kb = fp8_groups(cols);
  w->gate_up = gate_up;
  if (cudaGetDevice(&w->device) != cudaSuccess) {
    delete w;
    return fail(AH_ECUDA, "fp8w: no current device");
  }
  const size_t tile_bytes = (size_t)w->nt * (size_t)w->kb * kFp8TileBytes;
  if (dev_malloc(&w->tiles, tile_bytes + (size_t)w->nt * (size_t)w->kb * sizeof(float)) != cudaSuccess) {
    cudaGetLastError();
    delete w;
    return fail(AH_ENOMEM, "fp8w: device allocation of %zu bytes failed", tile_bytes);
  }
  w->scales = reinterpret_cast<float*>(w->tiles + tile_bytes);
  const BuildArgs g{{s[0], s[1]}, rows, cols, w->tiles, w->scales, w->nt, w->kb, gate_up};
  const dim3 grid((unsigned)w->kb, (unsigned)(w->nt < 65535 ? w->nt : 65535));
  switch (kind) {
    case kSourceE4m3: k_fp8w_copy<<<grid, 256, 0, st>>>(g); break;
    case kSourceF32: k_fp8w_quantize<float><<<grid, 256, 0, st>>>(g); break;
    case kSourceF16: k_fp8w_quantize<__half><<<grid, 256, 0, st>>>(g); break;
    default: k_fp8w_quantize<__nv_bfloat16><<<grid, 256, 0, st>>>(g); break;
  }
  // the handle is complete when it is returned: products may read it before
  // they wait for the grids ahead of them
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) {
    destroy(w);
    return fail(AH_ECUDA, "fp8w: building the weight: %s", cudaGetErrorString(e));
  }
  *out = w;
  return AH_OK;
}

// ---- the product -------------------------------------------------------------------

struct MatmulArgs {
  const uint8_t* tiles;
  const float* wscales;
  int64_t rows, cols, nt, kb;
  bool gate_up;
  const uint8_t* a;
  int64_t lda;
  const float* ascales;
  int64_t lds;
  int64_t m;
  void* y;
  int64_t ldy;
  uint32_t y_dtype;
};

__device__ __forceinline__ void store_y(void* y, int64_t i, uint32_t dtype, float v) {
  if (dtype == AH_DTYPE_F32) static_cast<float*>(y)[i] = v;
  else if (dtype == AH_DTYPE_F16) static_cast<__half*>(y)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
}

// 64 tokens x one tile's 128 rows per CTA of 256 threads, 8 x 4 outputs each;
// every block of 128 columns goes through shared memory as f32, 32 columns at
// a time.
__global__ void __launch_bounds__(256) k_fp8_matmul_simple(const MatmulArgs g) {
  __shared__ float sa[32][64 + 1], sw[32][128 + 1];
  const int64_t t = blockIdx.x, m0 = (int64_t)blockIdx.y * 64;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;  // rows tx + 32 * j, tokens ty + 8 * i
  float acc[8][4] = {};
  for (int64_t b = 0; b < g.kb; ++b) {
    const uint8_t* tile = g.tiles + (t * g.kb + b) * kFp8TileBytes;
    float part[8][4] = {};
    for (int c0 = 0; c0 < 128; c0 += 32) {
      __syncthreads();
      for (int i = threadIdx.x; i < 64 * 32; i += 256) {
        const int tok = i >> 5, c = i & 31;
        const int64_t col = b * kFp8Group + c0 + c;
        sa[c][tok] = m0 + tok < g.m && col < g.cols ? e4m3x2_f32(g.a[(m0 + tok) * g.lda + col]).x : 0.0f;
      }
      for (int i = threadIdx.x; i < 128 * 32; i += 256) {
        const int r = i >> 5, c = c0 + (i & 31);
        sw[i & 31][r] = e4m3x2_f32(tile[r * 128 + (((c >> 4) ^ (r & 7)) << 4) + (c & 15)]).x;
      }
      __syncthreads();
      for (int c = 0; c < 32; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[i][j] = fmaf(sa[c][ty + 8 * i], sw[c][tx + 32 * j], part[i][j]);
    }
    const float ws = g.wscales[t * g.kb + b];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t tok = m0 + ty + 8 * i;
      const float s = tok < g.m ? g.ascales[tok * g.lds + b] * ws : 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(s, part[i][j], acc[i][j]);
    }
  }
  // tile t's first output column and the rows of its source
  const int64_t rows = g.gate_up ? g.rows / 2 : g.rows;
  const int64_t r0 = (g.gate_up ? t >> 1 : t) * kFp8Group;
  const int64_t out0 = g.gate_up && (t & 1) ? rows : 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t tok = m0 + ty + 8 * i, r = r0 + tx + 32 * j;
      if (tok < g.m && r < rows) store_y(g.y, tok * g.ldy + out0 + r, g.y_dtype, acc[i][j]);
    }
}

int check_device(const char* who, const AhFp8Weight* w) {
  int dev = -1;
  AH_CUDA_TRY(cudaGetDevice(&dev));
  AH_REQUIRE(dev == w->device, "%s: the weight lives on device %d, device %d is current", who, w->device, dev);
  return AH_OK;
}

int matmul(const AhFp8Weight* w, const uint8_t* q, int64_t ldq, const float* scales, int64_t lds, int64_t m, void* y,
           int64_t ldy, uint32_t y_dtype, cudaStream_t st) {
  AH_REQUIRE(w, "fp8w_matmul: null weight");
  AH_REQUIRE(m >= 0 && m <= 0x7FFFFFFF, "fp8w_matmul: m must be 0 .. 2^31 - 1");
  AH_REQUIRE(y_dtype == AH_DTYPE_F32 || y_dtype == AH_DTYPE_F16 || y_dtype == AH_DTYPE_BF16,
             "fp8w_matmul: output dtype %u is not f32, f16 or bf16", y_dtype);
  if (m == 0) return AH_OK;
  AH_REQUIRE(q && scales && y, "fp8w_matmul: null pointer");
  AH_REQUIRE(aligned16(q) && ldq % 16 == 0 && ldq >= w->cols,
             "fp8w_matmul: q rows must start at multiples of 16 bytes, ldq >= cols");
  AH_REQUIRE(lds >= w->kb && ldy >= w->rows, "fp8w_matmul: lds below ceil(cols / 128) or ldy below rows");
  const int rc = check_device("fp8w_matmul", w);
  if (rc != AH_OK) return rc;
  const MatmulArgs g{w->tiles, w->scales, w->rows, w->cols, w->nt, w->kb, w->gate_up, q, ldq, scales, lds, m, y, ldy,
                     y_dtype};
  AH_REQUIRE((m + 63) / 64 <= 65535, "fp8w_matmul: m too large for one launch");
  k_fp8_matmul_simple<<<dim3((unsigned)w->nt, (unsigned)((m + 63) / 64)), 256, 0, st>>>(g);
  AH_LAUNCH_CHECK();
  return AH_OK;
}

// ---- the feed-forward block ----------------------------------------------------------

// Workspace: the norm's q and scales, gate | up in f32, the activation's q and scales.
struct FfnLayout {
  int64_t ldq1, lds1, n_ff, ldq2, lds2;
  size_t q1, s1, gu, q2, s2, total;
};

FfnLayout ffn_layout(const AhFp8Weight* gu, const AhFp8Weight* down, int64_t m) {
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  FfnLayout l;
  l.n_ff = gu->rows / 2;
  l.ldq1 = (gu->cols + 15) / 16 * 16;
  l.lds1 = gu->kb;
  l.ldq2 = (l.n_ff + 15) / 16 * 16;
  l.lds2 = down->kb;
  l.q1 = 0;
  l.s1 = l.q1 + up((size_t)m * l.ldq1);
  l.gu = l.s1 + up((size_t)m * l.lds1 * 4);
  l.q2 = l.gu + up((size_t)m * gu->rows * 4);
  l.s2 = l.q2 + up((size_t)m * l.ldq2);
  l.total = l.s2 + up((size_t)m * l.lds2 * 4);
  return l;
}

int check_ffn(const AhFp8Weight* gate_up, const AhFp8Weight* down, int64_t m) {
  AH_REQUIRE(gate_up && down, "fp8_ffn: null weight");
  AH_REQUIRE(gate_up->gate_up && !down->gate_up && down->cols == gate_up->rows / 2 && down->rows == gate_up->cols,
             "fp8_ffn: needs a gate/up weight of 2 * n_ff rows and a down weight [n_embd][n_ff]");
  AH_REQUIRE(m >= 0 && m <= 0x7FFFFFFF, "fp8_ffn: m must be 0 .. 2^31 - 1");
  return AH_OK;
}


}  // namespace
}  // namespace ah

using namespace ah;

extern "C" {

int ah_fp8w_from_blocks(const uint8_t* q, int64_t ldq, const float* scales, int64_t lds, int64_t rows, int64_t cols,
                        AhFp8Weight** out, void* stream) {
  const TileSource s[2] = {{q, ldq, scales, lds}, {}};
  return build(s, kSourceE4m3, false, rows, cols, out, as_stream(stream));
}

int ah_fp8w_from_blocks_gate_up(const uint8_t* gate_q, int64_t ld_gate, const float* gate_scales, int64_t lds_gate,
                                const uint8_t* up_q, int64_t ld_up, const float* up_scales, int64_t lds_up,
                                int64_t n_ff, int64_t n_embd, AhFp8Weight** out, void* stream) {
  const TileSource s[2] = {{gate_q, ld_gate, gate_scales, lds_gate}, {up_q, ld_up, up_scales, lds_up}};
  return build(s, kSourceE4m3, true, n_ff, n_embd, out, as_stream(stream));
}

int ah_fp8w_quantize(const void* w, int64_t ldw, uint32_t dtype, int64_t rows, int64_t cols, AhFp8Weight** out,
                     void* stream) {
  const TileSource s[2] = {{w, ldw, nullptr, 0}, {}};
  return build(s, source_kind(dtype), false, rows, cols, out, as_stream(stream));
}

int ah_fp8w_quantize_gate_up(const void* gate, int64_t ld_gate, const void* up, int64_t ld_up, uint32_t dtype,
                             int64_t n_ff, int64_t n_embd, AhFp8Weight** out, void* stream) {
  const TileSource s[2] = {{gate, ld_gate, nullptr, 0}, {up, ld_up, nullptr, 0}};
  return build(s, source_kind(dtype), true, n_ff, n_embd, out, as_stream(stream));
}

int ah_fp8w_destroy(AhFp8Weight* w) {
  if (w) destroy(w);
  return AH_OK;
}

int ah_fp8w_shape(const AhFp8Weight* w, int64_t* rows, int64_t* cols) {
  AH_REQUIRE(w && rows && cols, "fp8w_shape: null argument");
  *rows = w->rows;
  *cols = w->cols;
  return AH_OK;
}

int64_t ah_fp8w_weight_bytes(const AhFp8Weight* w) {
  if (!w) return 0;
  return w->rows * w->cols + w->nt * w->kb * 4;
}

int ah_fp8w_matmul(const AhFp8Weight* w, const uint8_t* q, int64_t ldq, const float* scales, int64_t lds, int64_t m,
                   void* y, int64_t ldy, uint32_t y_dtype, void* stream) {
  return matmul(w, q, ldq, scales, lds, m, y, ldy, y_dtype, as_stream(stream));
}

int ah_fp8_ffn_workspace_bytes(const AhFp8Weight* gate_up, const AhFp8Weight* down, int64_t m, size_t* bytes) {
  const int rc = check_ffn(gate_up, down, m);
  if (rc != AH_OK) return rc;
  AH_REQUIRE(bytes, "fp8_ffn_workspace_bytes: null output");
  *bytes = ffn_layout(gate_up, down, m).total;
  return AH_OK;
}

int ah_fp8_ffn(const AhFp8Weight* gate_up, const AhFp8Weight* down, const void* x, int64_t ldx, void* residual,
               int64_t ldr, uint32_t dtype, const void* norm_w, uint32_t norm_dtype, float eps, int64_t m, void* y,
               int64_t ldy, uint32_t y_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_ffn(gate_up, down, m);
  if (rc != AH_OK || m == 0) return rc;
  AH_REQUIRE(y && ldy >= down->rows, "fp8_ffn: null y or ldy below n_embd");
  AH_REQUIRE(y_dtype == AH_DTYPE_F32 || y_dtype == AH_DTYPE_F16 || y_dtype == AH_DTYPE_BF16,
             "fp8_ffn: output dtype %u is not f32, f16 or bf16", y_dtype);
  const FfnLayout l = ffn_layout(gate_up, down, m);
  AH_REQUIRE(workspace && aligned16(workspace), "fp8_ffn: the workspace must be 16-byte aligned");
  AH_REQUIRE(workspace_bytes >= l.total, "fp8_ffn: workspace of %zu bytes, %zu needed", workspace_bytes, l.total);
  // every refusal comes before the first launch: the residual is not advanced by a refused call
  if ((rc = check_device("fp8_ffn", gate_up)) != AH_OK || (rc = check_device("fp8_ffn", down)) != AH_OK) return rc;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  uint8_t *q1 = ws + l.q1, *q2 = ws + l.q2;
  float *s1 = reinterpret_cast<float*>(ws + l.s1), *s2 = reinterpret_cast<float*>(ws + l.s2);
  float* gu = reinterpret_cast<float*>(ws + l.gu);
  rc = ah_fp8_add_rms_norm(x, ldx, residual, ldr, dtype, norm_w, norm_dtype, eps, m, gate_up->cols, q1, l.ldq1, s1,
                           l.lds1, stream);
  if (rc != AH_OK) return rc;
  rc = ah_fp8w_matmul(gate_up, q1, l.ldq1, s1, l.lds1, m, gu, gate_up->rows, AH_DTYPE_F32, stream);
  if (rc != AH_OK) return rc;
  rc = ah_fp8_swiglu(gu, gate_up->rows, gu + l.n_ff, gate_up->rows, AH_DTYPE_F32, m, l.n_ff, q2, l.ldq2, s2, l.lds2,
                     stream);
  if (rc != AH_OK) return rc;
  return ah_fp8w_matmul(down, q2, l.ldq2, s2, l.lds2, m, y, ldy, y_dtype, stream);
}

}  // extern "C"
