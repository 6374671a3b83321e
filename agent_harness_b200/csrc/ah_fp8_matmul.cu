// ah_fp8_matmul.cu — resident e4m3 weights and their products with quantised
// activations:
//
//   y[i][r] = sum_b a_scale[i][b] * w_scale[r / 128][b] * sum_{j in block b} a[i][j] * w[r][j]
//
// b runs over the blocks of 128 columns.  The inner sums are exact products
// summed in f32; the scales multiply each block's sum in f32.
#include <algorithm>
#include <climits>
#include <mutex>
#include <new>

#include "ah_common.cuh"
#include "ah_fp8.cuh"
#include "ah_sm100.cuh"
#include "ah_tc.cuh"
#include "ah_tma.cuh"

namespace ah {
namespace {

// Tensor map of an e4m3 matrix [m][ld] read in boxes of 128 columns x box_rows
// with the 128-byte swizzle; zero past column k and row m.
int encode_rows(CUtensorMap* map, const void* base, uint64_t k, uint64_t m, uint64_t ld, uint32_t box_rows) {
  auto fn = tensor_map_encoder();
  if (!fn) return fail(AH_ECUDA, "fp8w_matmul: cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[2] = {k, m}, strides[1] = {ld};
  const cuuint32_t box[2] = {kFp8Group, box_rows}, step[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(AH_ECUDA, "fp8w_matmul: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return AH_OK;
}

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
    uint8_t* dst = g.tiles + fp8_image(g.gate_up, g.kb, t, b) * kFp8TileBytes;
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
    const float gm = __uint_as_float(a), inv = fp8_inverse(gm);
    uint8_t* dst = g.tiles + fp8_image(g.gate_up, g.kb, t, b) * kFp8TileBytes;
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
  // a handle may be collected while its thread captures something else: the free, which
  // is no part of that, would end the capture in its usual mode
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaThreadExchangeStreamCaptureMode(&mode);
  cudaFree(w->tiles);
  cudaThreadExchangeStreamCaptureMode(&mode);
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
    AH_REQUIRE(kind == kSourceE4m3 ? element_aligned(s[i].scales, AH_DTYPE_F32) : element_aligned(s[i].p, kind == kSourceF32 ? AH_DTYPE_F32 : AH_DTYPE_F16),
               "fp8w: a source is not aligned to its elements");
  }
  // an allocation, or the wait below, would end the capture
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(st, &capture) != cudaSuccess) cudaGetLastError();  // no device: the allocation says so
  AH_REQUIRE(capture == cudaStreamCaptureStatusNone, "fp8w: a weight cannot be made on a capturing stream");
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
  (void)device_error_word();  // looked up here, so that a product's first call may be captured
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

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Values at, at + 1, ... (n of 4) of y: one store where they lie on a boundary of
// their size.
__device__ __forceinline__ void store_y4(void* y, int64_t at, uint32_t dtype, const float (&v)[4], int n) {
  if (dtype == AH_DTYPE_F32) {
    float* p = static_cast<float*>(y) + at;
    if (n == 4 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
      return;
    }
  } else {
    uint16_t* p = static_cast<uint16_t*>(y) + at;
    if (n == 4 && (reinterpret_cast<uintptr_t>(p) & 7) == 0) {
      *reinterpret_cast<uint2*>(p) = dtype == AH_DTYPE_F16
                                         ? make_uint2(pack2<__half>(v[0], v[1]), pack2<__half>(v[2], v[3]))
                                         : make_uint2(pack2<__nv_bfloat16>(v[0], v[1]), pack2<__nv_bfloat16>(v[2], v[3]));
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) store_y(y, at + i, dtype, v[i]);
}

// SwiGLU and quantise of one token's group `unit`, four columns per lane, by a warp:
// p.act_q, p.act_scales.  rows = n_ff.
template <typename Args>
__device__ __forceinline__ void store_swiglu4(const Args& p, int64_t token, int64_t unit, int64_t rows,
                                              const float (&gate)[4], const float (&up)[4]) {
  const int lane = threadIdx.x & 31;
  const int64_t r = unit * kFp8Group + lane * 4;
  float o[4];
  fp8_silu_mul(gate, up, o);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = r + i < rows ? o[i] : 0.0f;
  const float fm = max_abs3(max_abs3(kFp8Tiny, o[0], o[1]), o[2], o[3]);
  const float gm = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(fm))), inv = fp8_inverse(gm);
  const uint32_t w = cvt_e4m3x4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  uint8_t* qrow = p.act_q + token * p.ld_act + r;  // ld_act is a multiple of 16
  if (r + 4 <= rows) *reinterpret_cast<uint32_t*>(qrow) = w;
  else
    for (int i = 0; i < 4 && r + i < rows; ++i) qrow[i] = (uint8_t)(w >> (8 * i));
  if (lane == 0) p.act_scales[token * p.lds_act + unit] = gm * (1.0f / kFp8Max);
}

// ---- few tokens: weight rows on the MMA's M, tokens on N ------------------------------
//
// A CTA takes one 128-row tile (or a gate/up pair of tiles) and a run of its
// column blocks for kNt tokens; a cluster of up to 8 CTAs shares a tile's column
// blocks and adds its members' sums through distributed shared memory in rank
// order, so results do not depend on timing.
//
//   warp 0     producer: one bulk copy of kKs column blocks of weights per stage
//              (contiguous, 16 or 32 KB each) and a TMA box of each block's tokens
//   warp 1     TMEM owner, MMA issuer: M = 128, N = kNt, K = 32, four per block
//   warps 2-5  a block's sums from tensor memory, times a_scale * w_scale, added
//              to f32 registers; then the cluster's sum and the output
//
// A block's sums are overwritten, not accumulated, in tensor memory: the scales
// change with every block.  kBufs buffers let the MMAs run ahead of the readers.
//
// Bound by the weight stream (a token costs it nothing up to 32): the first stages'
// weights are requested before the kernel waits for the grid ahead of it (a weight
// is complete once its handle exists), and two CTAs per SM keep 200 KB in flight.
// 128256 x 4096 at 16 tokens 85 us (6.3 TB/s), 28672 x 8192 at one 37 us (6.3), 4096 x
// 4096 at one 6.0 us (2.8: launch, first copies and the cluster's sum take 3 us).  At
// 64 tokens the shared memory's bandwidth is the bound (operands twice, and a
// broadcast read of four scales per four columns): 14336 x 4096 15.9 us (3.7 TB/s).
// Times in this file: calls captured back to back, inputs past the L2, a cool GPU.

constexpr uint32_t kWaitLimit = 1u << 24;
constexpr int kSmallThreads = 192;
constexpr int kMaxCluster = 8;
constexpr int kScaleBlocks = 8;  // column blocks whose scales are staged together

template <int kNt, bool kGlu>
struct Small {
  static constexpr int kTiles = kGlu ? 2 : 1;
  static constexpr int kKs = !kGlu && kNt == 16 ? 2 : 1;  // column blocks per stage
  static constexpr int kBlockBytes = kTiles * kFp8TileBytes;
  static constexpr int kActBytes = kNt * kFp8Group;
  static constexpr int kStageBytes = kKs * (kBlockBytes + kActBytes);
  static constexpr int kCols = kNt * kTiles;  // TMEM columns of one buffer
  static constexpr int kScaleBytes = 2 * kScaleBlocks * kCols * 4;
  static constexpr int kBudget = 113 * 1024 - 1024 - 512;  // two CTAs per SM, barriers, 1 KB alignment
  static constexpr int kStages = (kBudget - kScaleBytes) / kStageBytes;
  static constexpr int kBufs = kCols <= 64 ? 4 : 2;
  static constexpr int kTmemCols = kCols * kBufs < 32 ? 32 : kCols * kBufs;
  static_assert(kTmemCols <= 256, "two CTAs share an SM's 512 tensor-memory columns");
  static_assert(kStages >= 2, "at least two stages");
  // the sums [kCols][128] go over the idle ring for the cluster's reduction
  static_assert(kCols * 128 * 4 <= kStages * kStageBytes, "partial sums must fit the ring");
  static constexpr int kScale = kStages * kStageBytes;
  static constexpr int kBars = kScale + kScaleBytes;
  static constexpr int kMisc = kBars + (2 * kStages + 2 * kBufs + 1) * 8;
  static constexpr int kTotal = kMisc + 16;
  static constexpr size_t kDynamic = (size_t)kTotal + 1024;  // slack for 1 KB alignment
  static_assert(kDynamic <= 113 * 1024, "two CTAs per SM");
};

struct SmallArgs {
  CUtensorMap tm_a;  // e4m3 activations [m][cols], box 128 x kNt, 128-byte swizzle
  MatmulArgs g;
  uint8_t* act_q;    // SwiGLU: output instead of y
  int64_t ld_act;
  float* act_scales;
  int64_t lds_act;
  int* err;
};

// Waits on `bar`'s phase `parity`, up to kWaitLimit polls; then records
// AH_ETIMEOUT, raises the CTA's abort flag and goes on, as every later wait of
// the CTA then does at once: the outputs are lost, but all copies and MMAs stay
// inside the CTA's own stages and buffers and the kernel ends.
__device__ __forceinline__ void wait_bar(uint64_t* bar, uint32_t parity, int* err, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return;
  for (uint32_t it = 0; it < kWaitLimit; ++it) {
    if (mbar_try_wait(bar, parity)) return;
    if ((it & 63) == 0 && *abort_flag) return;
  }
  *abort_flag = 1;
  if (err) atomicExch(err, AH_ETIMEOUT);
}

__device__ __forceinline__ void promote_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <int kNt, bool kGlu>
__global__ void __launch_bounds__(kSmallThreads, 2) k_fp8_small(const __grid_constant__ SmallArgs p) {
  using L = Small<kNt, kGlu>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* empty = full + L::kStages;
  uint64_t* d_full = empty + L::kStages;
  uint64_t* d_empty = d_full + L::kBufs;
  uint64_t* drained = d_empty + L::kBufs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);
  const MatmulArgs& g = p.g;

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int nc = (int)gridDim.x, rank = (int)blockIdx.x;  // the cluster spans x
  const int64_t unit = blockIdx.y;                        // tile, or gate/up pair
  const int64_t m0 = (int64_t)blockIdx.z * kNt;
  const int64_t b0 = g.kb * rank / nc, b1 = g.kb * (rank + 1) / nc;
  const int nb = (int)(b1 - b0);
  const int n_stage = (nb + L::kKs - 1) / L::kKs;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < L::kBufs; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], 4);
    }
    mbar_init(drained, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, L::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // after the allocation: a dependent grid's CTA on this SM must not take the
  // tensor memory first and then wait for this grid
  pdl_launch_dependents();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    const bool elected = elect_one();
    const uint8_t* src = g.tiles + fp8_image(g.gate_up, g.kb, unit * L::kTiles, b0) * kFp8TileBytes;
    const bool halves = !kGlu && g.gate_up;  // one of a pair's two images per column block
    auto weights = [&](int s, int r) {
      const int n = min(L::kKs, nb - s * L::kKs);
      uint8_t* dst = smem + r * L::kStageBytes;
      mbar_arrive_expect_tx(&full[r], (uint32_t)(n * (L::kBlockBytes + L::kActBytes)));
      if (!halves)
        bulk_g2s(dst, src + (int64_t)s * L::kKs * L::kBlockBytes, (uint32_t)(n * L::kBlockBytes), &full[r]);
      else
        for (int i = 0; i < n; ++i)
          bulk_g2s(dst + i * kFp8TileBytes, src + (int64_t)(s * L::kKs + i) * 2 * kFp8TileBytes, kFp8TileBytes,
                   &full[r]);
    };
    const int x0 = (int)b0 * kFp8Group;
    auto tokens = [&](int s, int r) {
      const int n = min(L::kKs, nb - s * L::kKs);
      uint8_t* dst = smem + r * L::kStageBytes + L::kKs * L::kBlockBytes;
      for (int i = 0; i < n; ++i)
        tma_load_2d(dst + i * L::kActBytes, &p.tm_a, x0 + (s * L::kKs + i) * kFp8Group, (int)m0, &full[r]);
    };
    const int ahead = min(n_stage, L::kStages);
    if (elected)
      for (int s = 0; s < ahead; ++s) weights(s, s);
    pdl_wait();  // the tokens come from the preceding grid
    if (elected)
      for (int s = 0; s < ahead; ++s) tokens(s, s);
    int r = 0;
    uint32_t ph = 0;
    for (int s = ahead; s < n_stage; ++s) {
      wait_bar(&empty[r], ph, p.err, abort_flag);
      if (elected) {
        weights(s, r);
        tokens(s, r);
      }
      if (++r == L::kStages) {
        r = 0;
        ph ^= 1;
      }
    }
    // the last releases arrive, too, before the CTA can exit
    for (int i = 0; i < ahead; ++i) {
      wait_bar(&empty[r], ph, p.err, abort_flag);
      if (++r == L::kStages) {
        r = 0;
        ph ^= 1;
      }
    }
    if (*abort_flag)  // the copies in flight land before the CTA can exit
      for (int s = max(0, n_stage - L::kStages); s < n_stage; ++s)
        mbar_wait_bounded(&full[s % L::kStages], (uint32_t)((s / L::kStages) & 1), p.err, AH_ETIMEOUT, 1u << 12);
  } else if (warp == 1) {
    const bool elected = elect_one();
    constexpr uint32_t idesc = idesc_e4m3(128, kNt);
    int r = 0, buf = 0;
    uint32_t ph = 0, dph = 1;  // the buffers start empty
    pdl_wait();  // here, too: the waits for the tokens are counted from the end of the preceding grid
    for (int i = 0; i < nb; ++i) {
      if (i % L::kKs == 0) wait_bar(&full[r], ph, p.err, abort_flag);
      wait_bar(&d_empty[buf], dph, p.err, abort_flag);
      tc_fence_after();
      const uint32_t st = smem_u32(smem + r * L::kStageBytes);
      const uint32_t wb = st + (i % L::kKs) * L::kBlockBytes;
      const uint64_t bdesc = sw128_desc(st + L::kKs * L::kBlockBytes + (i % L::kKs) * L::kActBytes);
      const bool last = i % L::kKs == L::kKs - 1 || i == nb - 1;
      if (elected) {
#pragma unroll
        for (int h = 0; h < L::kTiles; ++h) {
          const uint64_t adesc = sw128_desc(wb + h * kFp8TileBytes);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f8(tmem + buf * L::kCols + h * kNt, adesc + kk * 2, bdesc + kk * 2, idesc, kk > 0);
        }
        mma_commit(&d_full[buf]);
        if (last) mma_commit(&empty[r]);
      }
      if (last && ++r == L::kStages) {
        r = 0;
        ph ^= 1;
      }
      if (++buf == L::kBufs) {
        buf = 0;
        dph ^= 1;
      }
    }
    if (*abort_flag) {  // the MMAs in flight end before the tensor memory is freed
      if (elected) mma_commit(drained);
      mbar_wait_bounded(drained, 0, p.err, AH_ETIMEOUT, kWaitLimit);
    }
  } else {
    const int q = warp & 3, t = threadIdx.x - 64;  // TMEM lane quarter, reader index
    float* sc = reinterpret_cast<float*>(smem + L::kScale);  // [2][kScaleBlocks][kCols]
    constexpr int kPer = kScaleBlocks * L::kCols / 128;
    float next_a[kPer], next_w[kPer];
    // thread t's share of the scales of blocks [i0, i0 + kScaleBlocks), multiplied
    // only when they are put down, eight blocks later; neighbouring threads take
    // neighbouring blocks of a token
    auto fetch = [&](int i0) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int e = t + j * 128, i = i0 + e % kScaleBlocks, c = e / kScaleBlocks;
        const int64_t tok = m0 + c % kNt;
        const bool live = i < nb && tok < g.m;
        next_a[j] = live ? g.ascales[tok * g.lds + b0 + i] : 0.0f;
        next_w[j] = live ? g.wscales[(unit * L::kTiles + c / kNt) * g.kb + b0 + i] : 0.0f;
      }
    };
    pdl_wait();  // the scales come from the preceding grid
    fetch(0);
    float acc[L::kCols];
#pragma unroll
    for (int j = 0; j < L::kCols; ++j) acc[j] = 0.0f;
    int buf = 0;
    uint32_t ph = 0;
    for (int i = 0; i < nb; ++i) {
      float* set = sc + (i / kScaleBlocks & 1) * kScaleBlocks * L::kCols;
      if (i % kScaleBlocks == 0) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int e = t + j * 128;
          set[e % kScaleBlocks * L::kCols + e / kScaleBlocks] = next_a[j] * next_w[j];
        }
        // also: every reader is done with the set before last
        promote_barrier();
        fetch(i + kScaleBlocks);
      }
      wait_bar(&d_full[buf], ph, p.err, abort_flag);
      tc_fence_after();
      const float* s = set + i % kScaleBlocks * L::kCols;
      const uint32_t ta = tmem + ((uint32_t)(q * 32) << 16) + buf * L::kCols;
      auto add = [&](int c, float v0, float v1, float v2, float v3) {
        const float4 f = *reinterpret_cast<const float4*>(s + c);
        acc[c] = fmaf(v0, f.x, acc[c]);
        acc[c + 1] = fmaf(v1, f.y, acc[c + 1]);
        acc[c + 2] = fmaf(v2, f.z, acc[c + 2]);
        acc[c + 3] = fmaf(v3, f.w, acc[c + 3]);
      };
      auto release = [&]() {  // the buffer is read
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&d_empty[buf]);
      };
      if constexpr (L::kCols == 16) {
        float v[16];
        tmem_ld16(ta, v);
        release();
#pragma unroll
        for (int j = 0; j < 16; j += 4) add(j, v[j], v[j + 1], v[j + 2], v[j + 3]);
      } else {
        uint32_t v[L::kCols / 32][32];
#pragma unroll
        for (int c = 0; c < L::kCols / 32; ++c) tmem_ld32_issue(ta + c * 32, v[c]);
#pragma unroll
        for (int c = 0; c < L::kCols / 32; ++c) tmem_ld32_wait(v[c]);
        release();
#pragma unroll
        for (int c = 0; c < L::kCols; c += 4)
          add(c, __uint_as_float(v[c / 32][c % 32]), __uint_as_float(v[c / 32][c % 32 + 1]),
              __uint_as_float(v[c / 32][c % 32 + 2]), __uint_as_float(v[c / 32][c % 32 + 3]));
      }
      if (++buf == L::kBufs) {
        buf = 0;
        ph ^= 1;
      }
    }
    // every block's MMAs have read their stages: the ring is idle
    float* part = reinterpret_cast<float*>(smem);  // [kCols][128]
#pragma unroll
    for (int c = 0; c < L::kCols; ++c) part[c * 128 + q * 32 + lane] = acc[c];
  }

  __syncwarp();
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
  const int live = (int)(g.m - m0 < kNt ? g.m - m0 : kNt);
  if (warp >= 2 && !*abort_flag) {
    // one warp per token, four rows per lane, all members' sums requested at once
    const uint32_t mine = smem_u32(smem) + lane * 16;
    auto sum4 = [&](int c, float (&o)[4]) {
      uint4 v[kMaxCluster];
#pragma unroll
      for (int k = 0; k < kMaxCluster; ++k)
        if (k < nc) v[k] = ld_dsmem_v4(mapa_shared(mine + c * 512, k));
      o[0] = o[1] = o[2] = o[3] = 0.0f;
#pragma unroll
      for (int k = 0; k < kMaxCluster; ++k)
        if (k < nc) {
          o[0] += __uint_as_float(v[k].x);
          o[1] += __uint_as_float(v[k].y);
          o[2] += __uint_as_float(v[k].z);
          o[3] += __uint_as_float(v[k].w);
        }
    };
    const int64_t rows = g.gate_up ? g.rows / 2 : g.rows;  // rows of the tile's source
    const int64_t r = (int64_t)(g.gate_up && !kGlu ? unit >> 1 : unit) * kFp8Group + lane * 4;
    for (int c = rank + (warp - 2) * nc; c < live; c += 4 * nc) {
      float o[4];
      sum4(c, o);
      if constexpr (kGlu) {
        float up[4];
        sum4(kNt + c, up);
        store_swiglu4(p, m0 + c, unit, rows, o, up);
      } else {
        const int64_t at = (m0 + c) * g.ldy + (g.gate_up && (unit & 1) ? rows : 0) + r;
        store_y4(g.y, at, g.y_dtype, o, (int)min((int64_t)4, rows - r));
      }
    }
  }
  // the other members have read this CTA's sums
  __syncwarp();
  cluster_arrive();
  cluster_wait();
}

int device_once(int* dev) {
  AH_CUDA_TRY(cudaGetDevice(dev));
  AH_REQUIRE(*dev >= 0 && *dev < 64, "fp8w_matmul: device %d out of range", *dev);
  return AH_OK;
}

// CTAs that share a tile's column blocks: as many as keep two CTAs per SM
// busy, each with two column blocks at least.
int small_cluster(int64_t units, int64_t kb) {
  int c = 1;
  while (c < kMaxCluster && units * c * 2 <= 2 * sm_count() && kb >= 4 * c) c *= 2;
  return c;
}

template <int kNt, bool kGlu>
int launch_small(SmallArgs& p, cudaStream_t st) {
  using L = Small<kNt, kGlu>;
  const MatmulArgs& g = p.g;
  int rc = encode_rows(&p.tm_a, g.a, (uint64_t)g.cols, (uint64_t)g.m, (uint64_t)g.lda, kNt);
  if (rc != AH_OK) return rc;
  static std::once_flag once[64];
  static cudaError_t attr[64];
  int dev = 0;
  rc = device_once(&dev);
  if (rc != AH_OK) return rc;
  std::call_once(once[dev], [&] {
    attr[dev] = cudaFuncSetAttribute(k_fp8_small<kNt, kGlu>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)L::kDynamic);
  });
  AH_CUDA_TRY(attr[dev]);
  const int64_t units = g.nt / L::kTiles, z = (g.m + kNt - 1) / kNt;
  AH_REQUIRE(units <= 65535 && z <= 65535, "fp8w_matmul: more than 65535 row or token tiles");
  const int c = small_cluster(units * z, g.kb);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)c, (unsigned)units, (unsigned)z);
  cfg.blockDim = dim3(kSmallThreads);
  cfg.dynamicSmemBytes = L::kDynamic;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)c;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  AH_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_fp8_small<kNt, kGlu>, (const SmallArgs)p));
  return AH_OK;
}

template <bool kGlu>
int dispatch_small(SmallArgs& p, cudaStream_t st) {
  if (p.g.m <= 16) return launch_small<16, kGlu>(p, st);
  if (kGlu || p.g.m <= 32) return launch_small<32, kGlu>(p, st);
  if constexpr (!kGlu) return launch_small<64, false>(p, st);
}

// ---- many tokens: CTA pairs, 256 tokens x 256 weight rows ---------------------------------
//
// A persistent pair walks tiles of 256 tokens x two weight tiles (a gate/up pair
// for SwiGLU).  Each CTA loads its 128 tokens and one of the two weight images of
// a column block (32 KB) and holds all 256 columns of its tokens' sums:
//
//   warp 0     producer (both CTAs, all copies complete on the leader's barrier)
//   warp 1     TMEM owner; in the leader the MMA issuer: cta_group::2, M = 256,
//              N = 256, K = 32, four per column block into one of two buffers of
//              256 tensor-memory columns
//   warps 4-11 a thread owns one token (tensor-memory lane) and 64 columns of each
//              weight tile: sums times a_scale * w_scale into 128 f32 registers,
//              one multiply-add each, since w_scale is one number per weight tile
//              and column block; then the tile's output
//
// Up to 128 tokens (!kPair) single CTAs walk tiles of 128 tokens x two weight tiles,
// loading both images (48 KB per column block, M = 128): half of a pair's rows would be
// empty.  A tile's column blocks are shared by a cluster of two, four or eight where
// that many fit the GPU at once; its members add their sums through distributed shared
// memory in rank order (65 x 6144 x 4096 12.6 us, by partial sums in global memory and a
// second launch 14.5; 65 x 8192 x 8192 18.5 against 19.6; requesting several tokens' sums
// at a time was no faster).  128 x 28672 x 8192 45 us (5.2 TB/s of weights; pairs 65), 128 x 32000 x 2048
// 16.4 (21.9), a 4096 x 14336 feed-forward block at 128 tokens 51 (69).  Past 128 tokens
// single CTAs load half as much again (2048 x 28672 x 8192 443 us where pairs took 414).
//
// What bounds it: a column block's MMAs take 560 cycles, and a buffer's way round
// (MMAs, the commit's way to both CTAs, the readers, their arrivals' way back) 1700 to
// 1800, hidden by two buffers down to 850 to 900.  2048 x 28672 x 8192 takes 403 to 420 us
// by the card (2290 to 2390 TFLOP/s; sustained, the power cap leaves 2000).  On one of 414,
// readers that only read tensor memory leave 373 us, that only multiply and add 406, that
// hand the buffers back at once 333 and 570 cycles.  Measured and not kept: half buffers of
// N = 128 (452 us) and tiles of one weight tile with four buffers (506), both bound by the
// readers' fixed cost per wait; scales through shared memory (427); paired multiply-adds
// (fma.f32x2, 561: their register pairs spill).  A release of cluster scope on the arrivals
// cost a memory barrier each (939 against 598 us at the time), issuing copies and MMAs
// outside uniform code another third.

constexpr int kBigThreads = 384;
// Registers: 384 threads start with 168 each (64512); the first four warps drop
// to 24 and the eight readers rise to 240 (128 * 24 + 256 * 240 = 64512).
constexpr int kBigRegsFew = 24, kBigRegsMany = 240;
constexpr int kBigTokens = 256;

template <bool kPair>
struct Big {
  static constexpr int kStages = kPair ? 6 : 4;
  static constexpr int kStageBytes = (kPair ? 2 : 3) * kFp8TileBytes;  // 128 tokens, one or both weight images
  static constexpr int kStage = kStages * kStageBytes;     // output staging: 4 KB per reader warp
  static constexpr int kMax = kStage + 8 * 4096;           // SwiGLU: group maxima [2][128]
  static constexpr int kBars = kMax + 1024;
  static constexpr int kMisc = kBars + (2 * kStages + 4 + 1) * 8;
  static constexpr int kTotal = kMisc + 16;
  static constexpr size_t kDynamic = (size_t)kTotal + 1024;
  static_assert(kDynamic <= 227 * 1024, "one CTA per SM");
};

// How the tiles are dealt out to pairs (or single CTAs).  Tiles [0, whole) go round robin to the
// grid, each over all column blocks.  Each of the `rest` tiles, fewer than a full
// round, is cut along the column blocks into `parts` pieces for as many pairs: pair
// p's sums go to partial slot p as f32 [256 columns][256 tokens], and k_fp8_join adds
// a tile's slots in K order.
struct BigSplit {
  int whole, rest, parts;
};

// The tiles of one pair or CTA, in order: tile, column blocks [b0, b1), partial slot (or
// -1: the whole tile).  What does not change stays in the kernel's arguments.
template <bool kPair>
struct BigWalk {
  static constexpr int kCtas = kPair ? 2 : 1;
  int tile, b0, b1, slot, at;
  __device__ __forceinline__ BigWalk() : at((int)blockIdx.x / kCtas) {}
  __device__ __forceinline__ bool next(const BigSplit& s, int kb) {
    b0 = 0;
    b1 = kb;
    slot = -1;
    tile = at;
    if (at < s.whole) {
      at += (int)gridDim.x / kCtas;
      return true;
    }
    const int pair = (int)blockIdx.x / kCtas;
    if (at == INT_MAX || pair >= s.rest * s.parts) return false;
    at = INT_MAX;
    const int piece = pair % s.parts;
    tile = s.whole + pair / s.parts;
    b0 = (int)((int64_t)kb * piece / s.parts);
    b1 = (int)((int64_t)kb * (piece + 1) / s.parts);
    slot = pair;
    return true;
  }
};

struct BigArgs {
  CUtensorMap tm_a;  // e4m3 activations [m][cols], box 128 x 128, 128-byte swizzle
  CUtensorMap tm_w;  // weight images as bytes [images * 128][128], box 128 x 128
  CUtensorMap tm_y;  // y [m][rows], box 128 bytes x 32 rows, 128-byte swizzle (when y_map)
  MatmulArgs g;
  bool y_map, y_whole;  // y has a map; its rows are whole 16-byte pieces, which a tiled store writes
  bool cluster;  // single CTAs: a split tile's parts are a cluster and add their sums in it
  BigSplit split;
  float* partial;
  uint8_t* act_q;
  int64_t ld_act;
  float* act_scales;
  int64_t lds_act;
  int* err;
};

// Four consecutive column blocks' scales of one row, from block b (zero past kb).
__device__ __forceinline__ void load_scales4(const float* row, int b, int kb, bool vec, float (&v)[4]) {
  if (vec && b + 4 <= kb) {
    const float4 f = *reinterpret_cast<const float4*>(row + b);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = b + i < kb ? row[b + i] : 0.0f;
  }
}

// One token of a tile that a cluster of nc CTAs shares: the members' sums at `at` in their
// shared memory (four columns of weight tile 0, tile 1's 64 KB on), in rank order, by
// one warp, and the token's output.
template <bool kGlu>
__device__ __forceinline__ void join_token(const BigArgs& p, int unit, int token, uint32_t at, int nc) {
  const MatmulArgs& g = p.g;
  const int lane = threadIdx.x & 31;
  float o[2][4];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    uint4 v[kMaxCluster];
#pragma unroll
    for (int k = 0; k < kMaxCluster; ++k)
      if (k < nc) v[k] = ld_dsmem_v4(mapa_shared(at + t * 65536, k));
    o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.0f;
#pragma unroll
    for (int k = 0; k < kMaxCluster; ++k)
      if (k < nc) {
        o[t][0] += __uint_as_float(v[k].x);
        o[t][1] += __uint_as_float(v[k].y);
        o[t][2] += __uint_as_float(v[k].z);
        o[t][3] += __uint_as_float(v[k].w);
      }
  }
  const int64_t rows = g.gate_up ? g.rows / 2 : g.rows;  // rows of a tile's source
  if constexpr (kGlu) {
    store_swiglu4(p, token, unit, rows, o[0], o[1]);
  } else {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t r = (int64_t)(g.gate_up ? unit : unit * 2 + t) * kFp8Group + lane * 4;
      store_y4(g.y, (int64_t)token * g.ldy + (g.gate_up ? t * rows : 0) + r, g.y_dtype, o[t],
               (int)max((int64_t)0, min((int64_t)4, rows - r)));
    }
  }
}

template <bool kGlu, bool kPair>
__global__ void __launch_bounds__(kBigThreads, 1) k_fp8_big(const __grid_constant__ BigArgs p) {
  using L = Big<kPair>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBars);  // the leader's are used
  uint64_t* empty = full + L::kStages;
  uint64_t* d_full = empty + L::kStages;
  uint64_t* d_empty = d_full + 2;  // the leader's are used
  uint64_t* drained = d_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);
  const MatmulArgs& g = p.g;

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int rank = kPair ? (int)cluster_ctarank() : 0;
  const int mt = (int)((g.m + kBigTokens - 1) / kBigTokens), nt = (int)g.nt, kb = (int)g.kb;
  BigWalk<kPair> walk;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], kPair ? 16 : 8);  // eight reader warps in each CTA
    }
    mbar_init(drained, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    if constexpr (kPair) tmem_alloc_pair(tmem_slot, 512);
    else tmem_alloc(tmem_slot, 512);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (kPair) {
    cluster_arrive();
    cluster_wait();
  }
  tc_fence_after();
  pdl_launch_dependents();  // after the allocation, as in k_fp8_small
  const uint32_t tmem = *tmem_slot;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kBigRegsFew));
    if (warp == 0) {
      const bool elected = elect_one();
      // a stage's copies land in both CTAs and complete on the leader's barrier
      const uint32_t full0 = mapa_shared(smem_u32(full), 0), st0 = smem_u32(smem);
      auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y, int s) {
        if constexpr (kPair) tma_load_2d_pair(dst, map, x, y, full0 + s * 8);
        else tma_load_2d(smem + (dst - st0), map, x, y, &full[s]);
      };
      auto weights = [&](int s, int unit, int b) {
        if (rank == 0) mbar_arrive_expect_tx(&full[s], (kPair ? 2 : 1) * L::kStageBytes);
        const uint32_t dst = st0 + s * L::kStageBytes + kFp8TileBytes;
#pragma unroll
        for (int i = 0; i < (kPair ? 1 : 2); ++i) {
          const int t = min(unit * 2 + rank + i, nt - 1);  // past an odd last tile: read again, not stored
          load(dst + i * kFp8TileBytes, &p.tm_w, 0, (int)fp8_image(g.gate_up, kb, t, b) * kFp8Group, s);
        }
      };
      bool more = walk.next(p.split, kb);
      int left = more ? min(walk.b1 - walk.b0, L::kStages) : 0;  // blocks whose weights are under way
      if (elected)
        for (int i = 0; i < left; ++i) weights(i, walk.tile / mt, walk.b0 + i);
      pdl_wait();  // the tokens come from the preceding grid
      int s = 0;
      uint32_t ph = 1;  // the stages start empty
      for (; more; more = walk.next(p.split, kb)) {
        const int unit = walk.tile / mt, row = walk.tile % mt * kBigTokens + rank * 128;
        for (int b = walk.b0; b < walk.b1; ++b) {
          wait_bar(&empty[s], ph, p.err, abort_flag);
          if (elected) {
            if (left <= 0) weights(s, unit, b);
            load(st0 + s * L::kStageBytes, &p.tm_a, b * kFp8Group, row, s);
          }
          --left;
          if (++s == L::kStages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      // the last releases, which the leader sends to both CTAs, arrive before either can exit
      for (int i = 0; i < L::kStages; ++i)
        wait_bar(&empty[(s + i) % L::kStages], s + i < L::kStages ? ph : ph ^ 1, p.err, abort_flag);
      if (*abort_flag && rank == 0)  // the copies in flight land before the pair can exit
        for (int i = 0; i < L::kStages; ++i)
          mbar_wait_bounded(&full[i], i < s ? ph ^ 1 : ph, p.err, AH_ETIMEOUT, 1u << 12);
    } else if (warp == 1 && rank == 0) {
      const bool elected = elect_one();
      constexpr uint32_t idesc = idesc_e4m3(kPair ? 256 : 128, 256);
      auto commit = [](uint64_t* bar) {
        if constexpr (kPair) mma_commit_pair(bar);
        else mma_commit(bar);
      };
      int s = 0, buf = 0;
      uint32_t ph = 0, dph = 1;  // the buffers start empty
      pdl_wait();  // here, too: the waits for the tokens are counted from the end of the preceding grid
      while (walk.next(p.split, kb))
        for (int b = walk.b0; b < walk.b1; ++b) {
          wait_bar(&full[s], ph, p.err, abort_flag);
          wait_bar(&d_empty[buf], dph, p.err, abort_flag);
          tc_fence_after();
          const uint32_t st = smem_u32(smem + s * L::kStageBytes);
          const uint64_t adesc = sw128_desc(st), bdesc = sw128_desc(st + kFp8TileBytes);
          if (elected) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              if constexpr (kPair) mma_f8_pair(tmem + buf * 256, adesc + kk * 2, bdesc + kk * 2, idesc, kk > 0);
              else mma_f8(tmem + buf * 256, adesc + kk * 2, bdesc + kk * 2, idesc, kk > 0);
            }
            commit(&d_full[buf]);
            commit(&empty[s]);
          }
          if (++s == L::kStages) {
            s = 0;
            ph ^= 1;
          }
          buf ^= 1;
          dph ^= buf == 0;
        }
      if (*abort_flag) {  // the MMAs in flight end before the tensor memory is freed
        if (elected) {  // an arrival in this CTA alone: the other one does not wait for it
          if constexpr (kPair) mma_commit_pair_self(drained);
          else mma_commit(drained);
        }
        mbar_wait_bounded(drained, 0, p.err, AH_ETIMEOUT, kWaitLimit);
      }
    }
    if (!kPair && p.cluster) {  // the readers' exchange
      __syncwarp();
      cluster_arrive();
      cluster_wait();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kBigRegsMany));
    const int q = warp & 3, h = (warp - 4) >> 2;  // TMEM lane quarter, column half
    const uint32_t d_empty0 = kPair ? mapa_shared(smem_u32(d_empty), 0) : smem_u32(d_empty);
    const uint32_t lane_addr = tmem + ((uint32_t)(q * 32) << 16) + h * 64;
    const bool vec = (reinterpret_cast<uintptr_t>(g.ascales) & 15) == 0 && g.lds % 4 == 0;
    const bool wvec = kb % 4 == 0;  // rows of scales start at multiples of 16 bytes
    uint8_t* stage = smem + L::kStage + (warp - 4) * 4096;
    pdl_wait();  // the scales come from the preceding grid
    int buf = 0;
    uint32_t ph = 0;
    while (walk.next(p.split, kb)) {
      const int unit = walk.tile / mt, m0 = walk.tile % mt * kBigTokens + rank * 128 + q * 32;
      const int b0 = walk.b0, b1 = walk.b1;
      const bool va = vec && b0 % 4 == 0, vw = wvec && b0 % 4 == 0;
      const int64_t tok = m0 + lane;
      const float* arow = g.ascales + (tok < g.m ? tok : 0) * g.lds;  // past m: stored nowhere
      const float* w0 = g.wscales + (int64_t)(unit * 2) * kb;
      const float* w1 = g.wscales + (int64_t)min(unit * 2 + 1, nt - 1) * kb;
      float acc[2][64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[0][j] = acc[1][j] = 0.0f;
      float a4[4];
      load_scales4(arow, b0, b1, va, a4);
      for (int b4 = b0; b4 < b1; b4 += 4) {
        float s0[4], s1[4];
        load_scales4(w0, b4, b1, vw, s0);
        load_scales4(w1, b4, b1, vw, s1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s0[i] *= a4[i];
          s1[i] *= a4[i];
        }
        load_scales4(arow, b4 + 4, b1, va, a4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (b4 + i >= b1) break;
          wait_bar(&d_full[buf], ph, p.err, abort_flag);
          tc_fence_after();
          const uint32_t ta = lane_addr + buf * 256;
          uint32_t v[2][32];
          tmem_ld32_issue(ta, v[0]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            tmem_ld32_wait(v[c & 1]);
            if (c < 3) {
              tmem_ld32_issue(ta + (c + 1) / 2 * 128 + (c + 1) % 2 * 32, v[(c + 1) & 1]);
            } else {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) {
                if constexpr (kPair) mbar_arrive_cluster(d_empty0 + buf * 8);
                else mbar_arrive(&d_empty[buf]);
              }
            }
            const float f = c < 2 ? s0[i] : s1[i];
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              float& o = acc[c / 2][c % 2 * 32 + j];
              o = fmaf(__uint_as_float(v[c & 1][j]), f, o);
            }
          }
          buf ^= 1;
          ph ^= buf == 0;
        }
      }
      const bool ok = !__any_sync(0xFFFFFFFFu, *abort_flag);  // after a give-up nothing is stored
      if (!kPair && walk.slot >= 0 && p.cluster) {
        // to the idle ring as [tile][token][128 columns], 16-byte pieces of a token's row
        // at piece ^ (token % 32)
        if (ok) {
          const uint32_t row = smem_u32(smem) + (q * 32 + lane) * 512;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 16; ++j)
              asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(row + t * 65536 + (((h * 16 + j) ^ lane) << 4)),
                           "f"(acc[t][4 * j]), "f"(acc[t][4 * j + 1]), "f"(acc[t][4 * j + 2]), "f"(acc[t][4 * j + 3])
                           : "memory");
        }
        continue;
      }
      if (walk.slot >= 0) {
        // columns 64 h + j of weight tile t at 128 t + 64 h + j: a warp stores 32 tokens
        float* out = p.partial + ((int64_t)walk.slot * 256 + h * 64) * kBigTokens + rank * 128 + q * 32 + lane;
        if (ok && tok < g.m) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 64; ++j) out[(t * 128 + j) * kBigTokens] = acc[t][j];
        }
        continue;
      }
      if constexpr (kGlu) {
        const int64_t n_ff = g.rows / 2, c0 = (int64_t)unit * kFp8Group + h * 64;
        // rows past n_ff are zero in the images: their products are zero
        fp8_silu_mul(acc[0], acc[1], acc[0]);
        float fm = kFp8Tiny;
#pragma unroll
        for (int j = 0; j < 64; j += 2) fm = max_abs3(fm, acc[0][j], acc[0][j + 1]);
        uint32_t mx = __float_as_uint(fm);  // a NaN's bits are above every number's
        uint32_t* maxima = reinterpret_cast<uint32_t*>(smem + L::kMax);
        maxima[h * 128 + q * 32 + lane] = mx;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        mx = max(mx, maxima[(h ^ 1) * 128 + q * 32 + lane]);
        asm volatile("bar.sync 1, 256;" ::: "memory");  // read before the next tile writes
        const float gm = __uint_as_float(mx), inv = fp8_inverse(gm);
        if (ok && tok < g.m) {
          uint8_t* qrow = p.act_q + tok * p.ld_act + c0;  // 16-byte aligned: ld_act is a multiple of 16
#pragma unroll
          for (int j = 0; j < 64; j += 16) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = cvt_e4m3x4(acc[0][j + 4 * i] * inv, acc[0][j + 4 * i + 1] * inv, acc[0][j + 4 * i + 2] * inv,
                                acc[0][j + 4 * i + 3] * inv);
            if (c0 + j + 16 <= n_ff) {
              *reinterpret_cast<uint4*>(qrow + j) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (c0 + j + i < n_ff) qrow[j + i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
            }
          }
          if (h == 0) p.act_scales[tok * p.lds_act + unit] = gm * (1.0f / kFp8Max);
        }
      } else if (!ok) {
        continue;
      } else if (p.y_map && (p.y_whole || (int64_t)(unit + 1) * 2 * kFp8Group <= g.rows)) {
        // 128-byte rows through the warp's 4 KB stage (16-byte pieces swizzled as
        // the map does), one tiled store per 32 rows
        const bool wide = g.y_dtype == AH_DTYPE_F32;
        const uint32_t row = smem_u32(stage) + lane * 128, sw = lane & 7;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (!wide && (c & 1)) continue;
          const int64_t col = (int64_t)(unit * 2 + c / 2) * kFp8Group + h * 64 + c % 2 * 32;
          if (lane == 0) bulk_wait_read0();  // the last store has read the stage
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float* o = &acc[c / 2][0];
              if (wide) w[i] = __float_as_uint(o[c % 2 * 32 + 4 * j + i]);
              else if (c % 2 == 0) {
                const int k = (8 * j + 2 * i) & 63;
                w[i] = g.y_dtype == AH_DTYPE_F16 ? pack2<__half>(o[k], o[k + 1]) : pack2<__nv_bfloat16>(o[k], o[k + 1]);
              }
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + ((j ^ sw) << 4)), "r"(w[0]), "r"(w[1]),
                         "r"(w[2]), "r"(w[3])
                         : "memory");
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && col < g.rows && m0 < g.m) {
            tma_store_2d(&p.tm_y, (int)col, (int)m0, smem_u32(stage));
            bulk_commit();
          }
        }
      } else {
        // y that no tensor map can address, or rows that end inside a 16-byte piece: 32 x 32
        // f32 boxes through the warp's stage, each token's 32 columns written by the whole warp
        const int64_t rows = g.gate_up ? g.rows / 2 : g.rows;  // rows of a tile's source
        float* box = reinterpret_cast<float*>(stage);
        if (lane == 0) bulk_wait_read0();  // another tile's last store has read the stage
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; ++j) box[lane * 32 + (j ^ lane)] = acc[c / 2][c % 2 * 32 + j];
          __syncwarp();
          const int64_t r = (int64_t)(g.gate_up ? unit : unit * 2 + c / 2) * kFp8Group + h * 64 + c % 2 * 32 + lane;
          if (r < rows) {
            const int64_t at = (g.gate_up ? c / 2 * rows : 0) + r;
            const int live = (int)min((int64_t)32, g.m - m0);
            auto write = [&](auto* y, auto convert) {
              y += (int64_t)m0 * g.ldy + at;
#pragma unroll 8
              for (int i = 0; i < live; ++i, y += g.ldy) *y = convert(box[i * 32 + (lane ^ i)]);
            };
            if (g.y_dtype == AH_DTYPE_F32) write(static_cast<float*>(g.y), [](float v) { return v; });
            else if (g.y_dtype == AH_DTYPE_F16) write(static_cast<__half*>(g.y), [](float v) { return __float2half_rn(v); });
            else write(static_cast<__nv_bfloat16*>(g.y), [](float v) { return __float2bfloat16_rn(v); });
          }
        }
      }
    }
    if (lane == 0) bulk_wait_all();  // the stage is read, the stores complete
    if (!kPair && p.cluster) {
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      if (!*abort_flag) {
        const int nc = p.split.parts;
        for (int c = (int)cluster_ctarank() + (warp - 4) * nc; c < (int)g.m; c += 8 * nc)
          join_token<kGlu>(p, (int)blockIdx.x / nc, c, smem_u32(smem) + c * 512 + ((lane ^ (c & 31)) << 4), nc);
      }
    }
  }

  __syncwarp();
  __syncthreads();
  if (kPair || p.cluster) {  // the other CTAs are done with this one's shared memory
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after();
    if constexpr (kPair) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

// Joins one split tile's partial sums for 32 tokens (x: chunk of tokens, y: tile of
// the rest): 32 warps of eight columns, lanes over the tokens.
constexpr int kJoinThreads = 1024;
template <bool kGlu>
__global__ void __launch_bounds__(kJoinThreads) k_fp8_join(const __grid_constant__ BigArgs p) {
  __shared__ float tr[kGlu ? 1 : 32][256 + 1];  // [token][column]
  __shared__ uint32_t maxima[kGlu ? 32 * 32 : 1];
  pdl_launch_dependents();
  pdl_wait();
  const MatmulArgs& g = p.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int mt = (int)((g.m + kBigTokens - 1) / kBigTokens), parts = p.split.parts;
  const int r = blockIdx.y, tile = p.split.whole + r, unit = tile / mt;
  const int64_t m0 = (int64_t)(tile % mt) * kBigTokens + blockIdx.x * 32, tok = m0 + lane;
  if (m0 >= g.m) return;
  // this warp's columns: SwiGLU, four gate columns and the same four up columns
  const int c0 = kGlu ? warp * 4 : warp * 8;
  auto column = [&](int j) { return kGlu ? j / 4 * 128 + c0 + j % 4 : c0 + j; };
  const float* in = p.partial + (int64_t)r * parts * 256 * kBigTokens + blockIdx.x * 32 + lane;
  float acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
  if (tok < g.m) {
    for (int q = 0; q < parts; q += 4) {  // four pieces' loads in flight
      float v[4][8];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = q + i < parts ? in[((q + i) * 256 + column(j)) * kBigTokens] : 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += v[i][j];
    }
  }
  if constexpr (kGlu) {
    const int64_t n_ff = g.rows / 2, col = (int64_t)unit * kFp8Group + c0;
    float o[4];
    fp8_silu_mul({acc[0], acc[1], acc[2], acc[3]}, {acc[4], acc[5], acc[6], acc[7]}, o);
    maxima[warp * 32 + lane] = __float_as_uint(max_abs3(max_abs3(kFp8Tiny, o[0], o[1]), o[2], o[3]));
    __syncthreads();
    uint32_t mx = 0;  // a NaN's bits are above every number's
#pragma unroll
    for (int i = 0; i < 32; ++i) mx = max(mx, maxima[i * 32 + lane]);
    const float gm = __uint_as_float(mx), inv = fp8_inverse(gm);
    if (tok < g.m) {
      const uint32_t w = cvt_e4m3x4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
      uint8_t* qrow = p.act_q + tok * p.ld_act + col;  // ld_act is a multiple of 16
      if (col + 4 <= n_ff) *reinterpret_cast<uint32_t*>(qrow) = w;
      else
        for (int i = 0; i < 4 && col + i < n_ff; ++i) qrow[i] = (uint8_t)(w >> (8 * i));
      if (warp == 0) p.act_scales[tok * p.lds_act + unit] = gm * (1.0f / kFp8Max);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) tr[lane][c0 + j] = acc[j];
    __syncthreads();
    // warp w writes token w's 256 columns
    const int64_t rows = g.gate_up ? g.rows / 2 : g.rows;
    if (m0 + warp < g.m) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = i / 4;  // weight tile of the pair
        const int64_t row = (int64_t)(g.gate_up ? unit : unit * 2 + t) * kFp8Group + i % 4 * 32 + lane;
        if (row < rows)
          store_y(g.y, (m0 + warp) * g.ldy + (g.gate_up ? t * rows : 0) + row, g.y_dtype, tr[warp][i * 32 + lane]);
      }
    }
  }
}

int check_device(const char* who, const AhFp8Weight* w) {
  int dev = -1;
  AH_CUDA_TRY(cudaGetDevice(&dev));
  AH_REQUIRE(dev == w->device, "%s: the weight lives on device %d, device %d is current", who, w->device, dev);
  return AH_OK;
}

// Makes a weight's device current while plans are made for it.
struct DeviceScope {
  int before = -1;
  cudaError_t error;
  explicit DeviceScope(int device) {
    error = cudaGetDevice(&before);
    if (error == cudaSuccess && device != before) error = cudaSetDevice(device);
    if (error != cudaSuccess) cudaGetLastError();
  }
  ~DeviceScope() {
    int now = before;
    if (before >= 0 && cudaGetDevice(&now) == cudaSuccess && now != before) cudaSetDevice(before);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
};

// The pairs (or single CTAs) of a launch and how its tiles are dealt out.  Splitting the tiles past
// the last full round saves column blocks' time (about 0.45 us each) and costs a
// launch (3 us) and the partial sums' way to L2 and back (about 6 TB/s).
struct BigPlan {
  bool pair;     // CTA pairs of 256 tokens, or single CTAs of 128
  bool cluster;  // single CTAs: tiles cut along K over clusters
  int pairs;     // pairs, or CTAs
  BigSplit split;
  size_t bytes;  // partial sums
};

// Clusters of c single CTAs that the current device holds at a time.
int max_clusters(int c) {
  static std::once_flag once[64];
  static int most[64][kMaxCluster + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::call_once(once[dev], [&] {
    if (cudaFuncSetAttribute(k_fp8_big<false, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)Big<false>::kDynamic) != cudaSuccess) {
      cudaGetLastError();
      return;
    }
    for (int n = 2; n <= kMaxCluster; n *= 2) {
      cudaLaunchAttribute at{};
      at.id = cudaLaunchAttributeClusterDimension;
      at.val.clusterDim.x = (unsigned)n;
      at.val.clusterDim.y = at.val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3((unsigned)n);
      cfg.blockDim = dim3(kBigThreads);
      cfg.dynamicSmemBytes = Big<false>::kDynamic;
      cfg.attrs = &at;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&most[dev][n], k_fp8_big<false, false>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        most[dev][n] = 0;
      }
    }
  });
  return most[dev][c];
}

BigPlan big_plan(const AhFp8Weight* w, int64_t m) {
  const int64_t tiles = (m + kBigTokens - 1) / kBigTokens * ((w->nt + 1) / 2);
  const bool pair = m > kBigTokens / 2;
  const int64_t pairs = pair ? std::max(1, sm_count() / 2) : sm_count();
  const int64_t rest = tiles % pairs, kb = w->kb;
  BigPlan p{pair, false, (int)std::min(tiles, pairs), {(int)tiles, 0, 0}, 0};
  for (int c = kMaxCluster; !pair && c >= 2; c /= 2)
    if (kb >= 4 * c && tiles <= max_clusters(c)) {  // four column blocks each at least
      p.cluster = true;
      p.pairs = (int)tiles * c;
      p.split = BigSplit{0, (int)tiles, c};
      return p;
    }
  const int64_t parts = rest ? std::min<int64_t>(pairs / rest, kb / 2) : 0;  // two column blocks each at least
  if (parts < 2) return p;
  const double saved = 0.45e-6 * (double)(kb - (kb + parts - 1) / parts);
  const double moved = 2.0 * (double)(rest * parts) * (double)std::min<int64_t>(m, kBigTokens) * 256 * sizeof(float);
  if (saved < 3e-6 + moved / 6e12) return p;
  p.pairs = (int)(tiles > pairs ? pairs : rest * parts);
  p.split = BigSplit{(int)(tiles - rest), (int)rest, (int)parts};
  p.bytes = (size_t)(rest * parts) * 256 * kBigTokens * sizeof(float);
  return p;
}

template <bool kGlu, bool kPair>
int launch_big(BigArgs& p, const BigPlan& plan, cudaStream_t st) {
  const MatmulArgs& g = p.g;
  int rc = encode_rows(&p.tm_a, g.a, (uint64_t)g.cols, (uint64_t)g.m, (uint64_t)g.lda, 128);
  if (rc != AH_OK) return rc;
  rc = encode_2d(&p.tm_w, g.tiles, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, kFp8Group, (uint64_t)g.nt * g.kb * kFp8Group,
                 kFp8Group, kFp8Group, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (rc != AH_OK) return rc;
  const int elem = g.y_dtype == AH_DTYPE_F32 ? 4 : 2;
  p.y_map = !kGlu && !g.gate_up && aligned16(g.y) && g.ldy * elem % 16 == 0;
  p.y_whole = g.rows * elem % 16 == 0;
  if (p.y_map) {
    const CUtensorMapDataType dt = elem == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    auto fn = tensor_map_encoder();
    const cuuint64_t dims[2] = {(cuuint64_t)g.rows, (cuuint64_t)g.m}, strides[1] = {(cuuint64_t)g.ldy * elem};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / elem), 32}, one[2] = {1, 1};
    const CUresult r = fn(&p.tm_y, dt, 2, g.y, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(AH_ECUDA, "fp8w_matmul: cuTensorMapEncodeTiled failed (%d)", (int)r);
  }
  static std::once_flag once[64];
  static cudaError_t attr[64];
  int dev = 0;
  rc = device_once(&dev);
  if (rc != AH_OK) return rc;
  static int regs[64];
  std::call_once(once[dev], [&] {
    attr[dev] = cudaFuncSetAttribute(k_fp8_big<kGlu, kPair>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Big<kPair>::kDynamic);
    cudaFuncAttributes a{};
    if (attr[dev] == cudaSuccess) attr[dev] = cudaFuncGetAttributes(&a, k_fp8_big<kGlu, kPair>);
    regs[dev] = a.numRegs;
  });
  AH_CUDA_TRY(attr[dev]);
  // raising the readers' registers waits for ever where the launch brought fewer
  if (regs[dev] * kBigThreads < kBigRegsFew * 128 + kBigRegsMany * 256)
    return fail(AH_EUNSUPPORTED, "fp8w_matmul: built with %d registers per thread, too few to redistribute", regs[dev]);
  p.split = plan.split;
  p.cluster = plan.cluster;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((kPair ? 2 : 1) * plan.pairs));
  cfg.blockDim = dim3(kBigThreads);
  cfg.dynamicSmemBytes = Big<kPair>::kDynamic;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = kPair ? 2 : plan.cluster ? (unsigned)plan.split.parts : 1;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  AH_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_fp8_big<kGlu, kPair>, (const BigArgs)p));
  if (plan.split.rest == 0 || plan.cluster) return AH_OK;
  const unsigned chunks = (unsigned)std::min<int64_t>(kBigTokens / 32, (g.m + 31) / 32);
  return launch_pdl(k_fp8_join<kGlu>, dim3(chunks, (unsigned)plan.split.rest), dim3(kJoinThreads), 0, st, (const BigArgs)p);
}

// Whether a product goes to k_fp8_big.  The weight-streaming kernel
// takes up to 32, and 33 to 64 while the tiles of single CTAs would leave a third of the
// SMs idle (64 tokens: 14336 x 4096 15.9 us against 17.4, but 28672 x 8192 45.5 against
// 42.5, a 4096 x 14336 feed-forward block 54 with its gate/up product there against 44).
// It takes more while its tiles, one per 64 tokens (32 for a gate/up pair), leave
// clusters of four (two) on two CTAs per SM: 4096 x 4096 at 128 tokens 10.7 us against
// 13.6 of single CTAs, but at 192 15.1 against 14.0 of pairs, and 8192 x 512 at 128 7.4
// against 6.5.
bool use_big(const AhFp8Weight* w, bool glu, int64_t m) {
  if (m <= 32) return false;
  if (m <= 64) return (w->nt + 1) / 2 * 3 > sm_count() * 2;
  return glu ? w->nt / 2 * ((m + 31) / 32) > sm_count() : w->nt * ((m + 63) / 64) > sm_count() / 2;
}

// Bytes of partial sums a product of m rows uses.
size_t matmul_bytes(const AhFp8Weight* w, bool glu, int64_t m) { return m > 0 && use_big(w, glu, m) ? big_plan(w, m).bytes : 0; }

int check_matmul(const AhFp8Weight* w, int64_t m) {
  AH_REQUIRE(w, "fp8w_matmul: null weight");
  AH_REQUIRE(m >= 0 && m <= 0x7FFFFF00, "fp8w_matmul: m must be 0 .. 2^31 - 256");
  AH_REQUIRE((m + kBigTokens - 1) / kBigTokens * ((w->nt + 1) / 2) < (1 << 30) && w->nt * w->kb < (1 << 24),
             "fp8w_matmul: too many tiles for one launch");
  return AH_OK;
}

// The rest of a product's launch, for y or for SwiGLU's outputs (set in p by `set`).
template <bool kGlu, typename Set>
int run_matmul(const MatmulArgs& g, const AhFp8Weight* w, float* partial, size_t bytes, cudaStream_t st, Set set) {
  if (use_big(w, kGlu, g.m)) {
    BigPlan plan = big_plan(w, g.m);
    AH_REQUIRE(!partial || bytes >= plan.bytes, "fp8w_matmul: workspace of %zu bytes, %zu needed", bytes, plan.bytes);
    if (plan.split.rest && !plan.cluster && !partial) {  // no workspace: no split
      const int64_t tiles = plan.split.whole + plan.split.rest;
      plan.pairs = (int)std::min<int64_t>(tiles, plan.pair ? std::max(1, sm_count() / 2) : sm_count());
      plan.split = BigSplit{(int)tiles, 0, 0};
    }
    BigArgs p{};
    p.g = g;
    p.partial = partial;
    p.err = device_error_word();
    set(p);
    return plan.pair ? launch_big<kGlu, true>(p, plan, st) : launch_big<kGlu, false>(p, plan, st);
  }
  SmallArgs p{};
  p.g = g;
  p.err = device_error_word();
  set(p);
  return dispatch_small<kGlu>(p, st);
}

int matmul(const AhFp8Weight* w, const uint8_t* q, int64_t ldq, const float* scales, int64_t lds, int64_t m, void* y,
           int64_t ldy, uint32_t y_dtype, void* workspace, size_t bytes, cudaStream_t st) {
  int rc = check_matmul(w, m);
  if (rc != AH_OK) return rc;
  AH_REQUIRE(y_dtype == AH_DTYPE_F32 || y_dtype == AH_DTYPE_F16 || y_dtype == AH_DTYPE_BF16,
             "fp8w_matmul: output dtype %u is not f32, f16 or bf16", y_dtype);
  if (m == 0) return AH_OK;
  AH_REQUIRE(q && scales && y, "fp8w_matmul: null pointer");
  AH_REQUIRE(aligned16(q) && ldq % 16 == 0 && ldq >= w->cols,
             "fp8w_matmul: q rows must start at multiples of 16 bytes, ldq >= cols");
  AH_REQUIRE(lds >= w->kb && ldy >= w->rows, "fp8w_matmul: lds below ceil(cols / 128) or ldy below rows");
  AH_REQUIRE(element_aligned(scales, AH_DTYPE_F32) && element_aligned(y, y_dtype),
             "fp8w_matmul: scales or y are not aligned to their elements");
  AH_REQUIRE(aligned16(workspace), "fp8w_matmul: the workspace must be 16-byte aligned");
  rc = check_device("fp8w_matmul", w);
  if (rc != AH_OK) return rc;
  const MatmulArgs g{w->tiles, w->scales, w->rows, w->cols, w->nt, w->kb, w->gate_up, q, ldq, scales, lds, m, y, ldy,
                     y_dtype};
  return run_matmul<false>(g, w, static_cast<float*>(workspace), bytes, st, [](auto&) {});
}

// silu(gate) * up of the products with a gate/up weight, quantised from f32.
int matmul_swiglu(const AhFp8Weight* w, const uint8_t* q, int64_t ldq, const float* scales, int64_t lds, int64_t m,
                  uint8_t* act_q, int64_t ld_act, float* act_scales, int64_t lds_act, float* partial, size_t bytes,
                  cudaStream_t st) {
  const MatmulArgs g{w->tiles, w->scales, w->rows, w->cols, w->nt, w->kb, true, q, ldq, scales, lds, m, nullptr, 0, 0};
  return run_matmul<true>(g, w, partial, bytes, st, [&](auto& p) {
    p.act_q = act_q;
    p.ld_act = ld_act;
    p.act_scales = act_scales;
    p.lds_act = lds_act;
  });
}

// ---- the feed-forward block ----------------------------------------------------------

// Workspace: the norm's q and scales, the activation's q and scales, the products'
// partial sums.
struct FfnLayout {
  int64_t ldq1, lds1, ldq2, lds2;
  size_t q1, s1, q2, s2, partial, partial_bytes, total;
};

FfnLayout ffn_layout(const AhFp8Weight* gu, const AhFp8Weight* down, int64_t m) {
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  FfnLayout l;
  l.ldq1 = (gu->cols + 15) / 16 * 16;
  l.lds1 = gu->kb;
  l.ldq2 = (down->cols + 15) / 16 * 16;
  l.lds2 = down->kb;
  l.q1 = 0;
  l.s1 = l.q1 + up((size_t)m * l.ldq1);
  l.q2 = l.s1 + up((size_t)m * l.lds1 * 4);
  l.s2 = l.q2 + up((size_t)m * l.ldq2);
  l.partial = l.s2 + up((size_t)m * l.lds2 * 4);
  l.partial_bytes = std::max(matmul_bytes(gu, true, m), matmul_bytes(down, false, m));
  l.total = l.partial + l.partial_bytes;
  return l;
}

int check_ffn(const AhFp8Weight* gate_up, const AhFp8Weight* down, int64_t m) {
  AH_REQUIRE(gate_up && down, "fp8_ffn: null weight");
  AH_REQUIRE(gate_up->gate_up && !down->gate_up && down->cols == gate_up->rows / 2 && down->rows == gate_up->cols,
             "fp8_ffn: needs a gate/up weight of 2 * n_ff rows and a down weight [n_embd][n_ff]");
  AH_REQUIRE(gate_up->device == down->device, "fp8_ffn: the weights live on devices %d and %d", gate_up->device,
             down->device);
  AH_REQUIRE(gate_up->nt / 2 <= 65535 && down->nt <= 65535, "fp8_ffn: more than 65535 row tiles");
  const int rc = check_matmul(gate_up, m);
  return rc != AH_OK ? rc : check_matmul(down, m);
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

int ah_fp8w_matmul_workspace_bytes(const AhFp8Weight* w, int64_t m, size_t* bytes) {
  const int rc = check_matmul(w, m);
  if (rc != AH_OK) return rc;
  AH_REQUIRE(bytes, "fp8w_matmul_workspace_bytes: null output");
  const DeviceScope on(w->device);  // the plan goes by the device that will run it
  if (on.error != cudaSuccess)
    return fail(AH_ECUDA, "fp8w_matmul_workspace_bytes: device %d: %s", w->device, cudaGetErrorString(on.error));
  *bytes = matmul_bytes(w, false, m);
  return AH_OK;
}

int ah_fp8w_matmul(const AhFp8Weight* w, const uint8_t* q, int64_t ldq, const float* scales, int64_t lds, int64_t m,
                   void* y, int64_t ldy, uint32_t y_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  return matmul(w, q, ldq, scales, lds, m, y, ldy, y_dtype, workspace, workspace_bytes, as_stream(stream));
}

int ah_fp8_ffn_workspace_bytes(const AhFp8Weight* gate_up, const AhFp8Weight* down, int64_t m, size_t* bytes) {
  const int rc = check_ffn(gate_up, down, m);
  if (rc != AH_OK) return rc;
  AH_REQUIRE(bytes, "fp8_ffn_workspace_bytes: null output");
  const DeviceScope on(down->device);
  if (on.error != cudaSuccess)
    return fail(AH_ECUDA, "fp8_ffn_workspace_bytes: device %d: %s", down->device, cudaGetErrorString(on.error));
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
  AH_REQUIRE(element_aligned(y, y_dtype), "fp8_ffn: y is not aligned to its elements");
  const FfnLayout l = ffn_layout(gate_up, down, m);
  AH_REQUIRE(workspace && aligned16(workspace), "fp8_ffn: the workspace must be 16-byte aligned");
  AH_REQUIRE(workspace_bytes >= l.total, "fp8_ffn: workspace of %zu bytes, %zu needed", workspace_bytes, l.total);
  // every refusal comes before the first launch: the residual is not advanced by a refused call
  if ((rc = check_device("fp8_ffn", gate_up)) != AH_OK || (rc = check_device("fp8_ffn", down)) != AH_OK) return rc;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  uint8_t *q1 = ws + l.q1, *q2 = ws + l.q2;
  float *s1 = reinterpret_cast<float*>(ws + l.s1), *s2 = reinterpret_cast<float*>(ws + l.s2);
  float* partial = l.partial_bytes ? reinterpret_cast<float*>(ws + l.partial) : nullptr;
  rc = ah_fp8_add_rms_norm(x, ldx, residual, ldr, dtype, norm_w, norm_dtype, eps, m, gate_up->cols, q1, l.ldq1, s1,
                           l.lds1, stream);
  if (rc != AH_OK) return rc;
  rc = matmul_swiglu(gate_up, q1, l.ldq1, s1, l.lds1, m, q2, l.ldq2, s2, l.lds2, partial, l.partial_bytes,
                     as_stream(stream));
  if (rc != AH_OK) return rc;
  return matmul(down, q2, l.ldq2, s2, l.lds2, m, y, ldy, y_dtype, partial, l.partial_bytes, as_stream(stream));
}

}  // extern "C"
