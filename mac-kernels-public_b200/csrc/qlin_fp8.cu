// Block-scaled 8-bit linear and its input gradient: the row quantizer, the GEMM's host launcher and the
// C ABI (include/qlin.h).
#include <cuda.h>
#include <cuda_runtime.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "../../include/qlin.h"
#include "qlin_fp8.cuh"
#include "qlin_internal.h"

namespace qlin {

// ---------------------------------------------------------------------------------------------
// Row quantizer: for every row and block of 128 columns, in fp32,
//   a = max(max |x|, 2^-100),  q = e4m3(x * (448 / a)),  scale = a / 448
// (448 is e4m3's largest value; the floor keeps both quotients normal for blocks of zeros).  The
// maximum is taken over the values' bit patterns, so a NaN or an infinity makes its block's scale
// non-finite and with it every output of the row.  Columns past K are zeros.
//
// One pass over x, bound by HBM: a warp takes 8 rows of two blocks, 16 lanes to a block and 8 values
// to a lane, with all its loads issued before the first reduction; the 8 scales of a block, which lie
// side by side in the block-major scale array, go out as one 32-byte piece.
// ---------------------------------------------------------------------------------------------
constexpr float kE4m3Max = 448.f;
constexpr uint32_t kAmaxFloorBits = (127 - 100) << 23;  // 2^-100

struct QuantFp8Params {
  const void* x;
  long long ldx;
  int M, K, kb;      // kb = blocks of 128, the last one padded with zeros
  int k_tiles;       // CTAs along the blocks
  uint8_t* q;
  long long ldq;
  float* scale;      // [kb][ld_scale]
  long long ld_scale;
  long long lim_x, lim_q, lim_scale;  // element counts for the QLIN_CHECKS build
};

template <int DT>
__device__ __forceinline__ float load_elem(const void* x, long long i) {
  if constexpr (DT == QLIN_F16) return __half2float(reinterpret_cast<const __half*>(x)[i]);
  else if constexpr (DT == QLIN_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(x)[i]);
  else return reinterpret_cast<const float*>(x)[i];
}

// 8 consecutive values as stored: 16 bytes of a 2-byte type, 32 of fp32.
template <int DT>
struct Raw8 {
  uint4 v[DT == QLIN_F32 ? 2 : 1];
};

template <int DT>
__device__ __forceinline__ Raw8<DT> load_raw8(const void* x, long long i) {
  Raw8<DT> r;
  constexpr int kBytes = DT == QLIN_F32 ? 4 : 2;
  const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(x) + i * kBytes);
  r.v[0] = __ldg(p);
  if constexpr (DT == QLIN_F32) r.v[1] = __ldg(p + 1);
  return r;
}

template <int DT>
__device__ __forceinline__ void raw8_to_float(const Raw8<DT>& r, float (&f)[8]) {
  const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (DT == QLIN_F32) {
      f[j] = __uint_as_float(w[j]);
    } else if constexpr (DT == QLIN_F16) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      f[2 * j] = t.x;
      f[2 * j + 1] = t.y;
    } else {
      f[2 * j] = __uint_as_float(w[j] << 16);
      f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  }
  if constexpr (DT == QLIN_F32) {
    f[4] = __uint_as_float(r.v[1].x);
    f[5] = __uint_as_float(r.v[1].y);
    f[6] = __uint_as_float(r.v[1].z);
    f[7] = __uint_as_float(r.v[1].w);
  }
}

// 4 values times r in e4m3, the first in the low byte.
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d, float r) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a * r, b * r), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c * r, d * r), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

template <int DT, bool kVec>
__global__ void __launch_bounds__(256) quant_rows_fp8_kernel(const QuantFp8Params p) {
  constexpr int kRows = 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row_tile = blockIdx.x / p.k_tiles;
  const int b = ((blockIdx.x - row_tile * p.k_tiles) * 8 + warp) * 2 + (lane >> 4);
  const int m0 = row_tile * kRows;
  const int c = b * 128 + (lane & 15) * 8;
  const int rows = min(kRows, p.M - m0);
  float f[kRows][8];
  if (kVec && c + 8 <= p.K) {
    Raw8<DT> raw[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const long long at = (long long)(m0 + min(i, rows - 1)) * p.ldx + c;
      if (qchk_span(BS_FP8_QUANT, at, 8, p.lim_x)) raw[i] = load_raw8<DT>(p.x, at);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) raw8_to_float<DT>(raw[i], f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const long long at = (long long)(m0 + i) * p.ldx + c + j;
        f[i][j] = (i < rows && c + j < p.K && qchk(BS_FP8_QUANT, at, p.lim_x)) ? load_elem<DT>(p.x, at) : 0.f;
      }
  }
  float mine = 0.f;  // the scale this lane writes: row lane & 15
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    uint32_t a = kAmaxFloorBits;
#pragma unroll
    for (int j = 0; j < 8; ++j) a = max(a, __float_as_uint(f[i][j]) & 0x7fffffffu);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
    const float amax = __uint_as_float(a);
    const float r = __fdiv_rn(kE4m3Max, amax);
    if ((lane & 15) == i) mine = __fdiv_rn(amax, kE4m3Max);
    if (i < rows && b < p.kb) {
      const long long at = (long long)(m0 + i) * p.ldq + c;
      if (qchk_span(BS_FP8_QUANT, at, 8, p.lim_q))
        *reinterpret_cast<uint2*>(p.q + at) = make_uint2(to_e4m3x4(f[i][0], f[i][1], f[i][2], f[i][3], r),
                                                         to_e4m3x4(f[i][4], f[i][5], f[i][6], f[i][7], r));
    }
  }
  if ((lane & 15) < rows && b < p.kb) {
    const long long at = (long long)b * p.ld_scale + m0 + (lane & 15);
    if (qchk(BS_FP8_QUANT, at, p.lim_scale)) p.scale[at] = mine;
  }
}

static int launch_quant_rows_fp8(const void* x, int x_dtype, long long ldx, int M, int K, uint8_t* q, long long ldq,
                                 float* scale, long long ld_scale, cudaStream_t stream) {
  QuantFp8Params p{};
  p.x = x;
  p.ldx = ldx;
  p.M = M;
  p.K = K;
  p.kb = (K + 127) / 128;
  p.k_tiles = (p.kb + 15) / 16;
  p.q = q;
  p.ldq = ldq;
  p.scale = scale;
  p.ld_scale = ld_scale;
  p.lim_x = (long long)(M - 1) * ldx + K;
  p.lim_q = (long long)(M - 1) * ldq + (long long)p.kb * 128;
  p.lim_scale = (long long)(p.kb - 1) * ld_scale + M;
  const long long grid = (long long)((M + 7) / 8) * p.k_tiles;
  if (grid > 0x7fffffff) {
    set_error("fp8 quantizer: %d rows of %d columns are too many", M, K);
    return QLIN_EINVAL;
  }
  const int esz = x_dtype == QLIN_F32 ? 4 : 2;
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * esz) % 16 == 0;
#define QLIN_QUANT_FP8(DT)                                                              \
  if (vec) quant_rows_fp8_kernel<DT, true><<<(unsigned)grid, 256, 0, stream>>>(p);      \
  else quant_rows_fp8_kernel<DT, false><<<(unsigned)grid, 256, 0, stream>>>(p);
  if (x_dtype == QLIN_F16) { QLIN_QUANT_FP8(QLIN_F16) }
  else if (x_dtype == QLIN_BF16) { QLIN_QUANT_FP8(QLIN_BF16) }
  else { QLIN_QUANT_FP8(QLIN_F32) }
#undef QLIN_QUANT_FP8
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error("fp8 quantizer launch failed: %s", cudaGetErrorString(e));
    return QLIN_ECUDA;
  }
  return QLIN_OK;
}

// ---------------------------------------------------------------------------------------------
// GEMM launch
// ---------------------------------------------------------------------------------------------
template <int CTAS, int TN, bool kTrans>
static int launch_fp8(const CUtensorMap& tx, const CUtensorMap& tw, const Fp8Params& p, cudaStream_t stream) {
  using Cfg = Fp8Cfg<CTAS, TN>;
  static_assert(Cfg::kSmem <= 232448, "shared memory per CTA");
  auto kern = fp8_gemm_kernel<CTAS, TN, kTrans>;
  static bool attr_done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem) != cudaSuccess) {
      set_error("cudaFuncSetAttribute(max dynamic smem %d) failed", Cfg::kSmem);
      return QLIN_ECUDA;
    }
    attr_done[dev] = true;
  }
  const int tiles = p.m_tiles * p.n_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CTAS * std::min(tiles, sm_count() / CTAS));
  cfg.blockDim = dim3(Cfg::kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CTAS;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tx, tw, p);
  if (e != cudaSuccess) {
    set_error("fp8 gemm launch failed: %s", cudaGetErrorString(e));
    return QLIN_ECUDA;
  }
  return QLIN_OK;
}

static size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

// Workspace: the e4m3 activations [m, round_up(depth, 128)] and their scales [blocks][m].
static size_t fp8_workspace(int64_t m, int64_t depth) {
  if (m <= 0 || depth <= 0) return 0;
  const int64_t kb = (depth + 127) / 128;
  return align256((size_t)m * kb * 128) + align256((size_t)kb * m * 4);
}

static int bias_kind_of(const void* bias, int dt) {
  if (bias == nullptr) return 0;
  return dt == QLIN_F16 ? 1 : dt == QLIN_F32 ? 2 : dt == QLIN_BF16 ? 3 : -1;
}
static bool is_float(int d) { return d == QLIN_F32 || d == QLIN_F16 || d == QLIN_BF16; }

// y[m, out] = quantized x[m, depth] times the weight q [rows, cols]: rows = out and cols = depth for the
// linear, the other way round (trans) for its input gradient.
static int fp8_product(const char* what, const void* x, int x_dtype, int64_t m, int64_t depth, int64_t ldx,
                       const void* q, int64_t ldq, int64_t out, bool trans, const float* scale, int64_t ld_scale,
                       const void* bias, int bias_dtype, void* y, int y_dtype, int64_t ldy, void* workspace,
                       size_t workspace_bytes, cudaStream_t stream) {
  const int64_t rows = trans ? depth : out, cols = trans ? out : depth;
  const int64_t most = 0x7fffffff - 512;
  if (m < 0 || depth < 0 || out < 0 || m > most || depth > most || out > most || (m > 1 && (ldx < depth || ldy < out)) ||
      (rows > 1 && ldq < cols) || (rows > 128 && ld_scale < (cols + 127) / 128)) {
    set_error("%s: bad sizes m=%lld rows=%lld cols=%lld ldx=%lld ldq=%lld ldy=%lld ld_scale=%lld", what, (long long)m,
              (long long)rows, (long long)cols, (long long)ldx, (long long)ldq, (long long)ldy, (long long)ld_scale);
    return QLIN_EINVAL;
  }
  const int bk = bias_kind_of(bias, bias_dtype);
  if (!is_float(x_dtype) || !is_float(y_dtype) || bk < 0) {
    set_error("%s: x, y and the bias are f32, f16 or bf16", what);
    return QLIN_EDECLINE;
  }
  if (cols % 16 != 0 || (ldq % 16 != 0 && rows > 1) || (reinterpret_cast<uintptr_t>(q) & 15)) {
    set_error("%s: the weight needs 16-byte aligned rows of a multiple of 16 columns (cols=%lld, ldq=%lld)", what,
              (long long)cols, (long long)ldq);
    return QLIN_EDECLINE;
  }
  if (m == 0 || out == 0) return QLIN_OK;
  if (y == nullptr) {
    set_error("%s: null output", what);
    return QLIN_EINVAL;
  }
  if (depth > 0 && (x == nullptr || q == nullptr || scale == nullptr)) {
    set_error("%s: null pointer", what);
    return QLIN_EINVAL;
  }
  if (workspace_bytes < fp8_workspace(m, depth) || (workspace == nullptr && fp8_workspace(m, depth) > 0)) {
    set_error("%s: workspace too small: need %zu bytes", what, fp8_workspace(m, depth));
    return QLIN_EINVAL;
  }
  const int kb = (int)((depth + 127) / 128);
  const int64_t kp = (int64_t)kb * 128;
  uint8_t* xq = reinterpret_cast<uint8_t*>(workspace);
  float* sx = reinterpret_cast<float*>(xq + align256((size_t)m * kp));
  Fp8Params p{};
  p.M = (int)m;
  p.N = (int)out;
  p.kb = kb;
  p.sx = sx;
  p.ld_sx = m;
  p.sw = scale;
  p.sw_out = trans ? 1 : ld_scale;
  p.sw_red = trans ? ld_scale : 1;
  p.bias = bias;
  p.bias_kind = bk;
  p.y = y;
  p.y_dtype = y_dtype == QLIN_F32 ? OUT_F32 : y_dtype == QLIN_F16 ? OUT_F16 : OUT_BF16;
  p.ldy = ldy;
  const int esz = y_dtype == QLIN_F32 ? 4 : 2;
  p.vec_out = (reinterpret_cast<uintptr_t>(y) & 15) == 0 && (ldy * esz) % 16 == 0;
  p.status = reinterpret_cast<DeviceStatus*>(device_status_ptr());
  p.lim_y = (m - 1) * ldy + out;
  p.lim_sx = (long long)kb * m;
  p.lim_sw = (long long)((rows + 127) / 128 - 1) * ld_scale + (cols + 127) / 128;
  const bool pair = m > 128 && out > 128;
  const int64_t m_tiles = (m + 127) / 128, n_tiles = (out + 127) / 128;
  if (m_tiles * n_tiles > 0x7fffffff) {
    set_error("%s: too many output tiles", what);
    return QLIN_EINVAL;
  }
  p.m_tiles = (int)(pair ? (m_tiles + 1) / 2 : m_tiles);
  p.n_tiles = (int)(pair ? (n_tiles + 1) / 2 : n_tiles);
  CUtensorMap tx{}, tw{};
  if (kb > 0) {
    int rc = launch_quant_rows_fp8(x, x_dtype, ldx, (int)m, (int)depth, xq, kp, sx, m, stream);
    if (rc) return rc;
    rc = make_tmap_2d(&tx, xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)kp, (uint64_t)m, (uint64_t)kp, 128, 128,
                      CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    rc = make_tmap_2d(&tw, q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)cols, (uint64_t)rows,
                      rows > 1 ? (uint64_t)ldq : (uint64_t)cols, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  if (pair) return trans ? launch_fp8<2, 256, true>(tx, tw, p, stream) : launch_fp8<2, 256, false>(tx, tw, p, stream);
  return trans ? launch_fp8<1, 128, true>(tx, tw, p, stream) : launch_fp8<1, 128, false>(tx, tw, p, stream);
}

// This translation unit's bounds record (QLIN_CHECKS build).
QLIN_BOUNDS_READER(bounds_read_fp8)

}  // namespace qlin

using namespace qlin;

extern "C" {

size_t qlin_fp8_linear_workspace(int64_t m, int64_t n, int64_t k) {
  (void)n;
  return fp8_workspace(m, k);
}

int qlin_fp8_linear(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const void* q, int64_t ldq,
                    int64_t n, const float* scale, int64_t ld_scale, const void* bias, int bias_dtype, void* y,
                    int y_dtype, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
  return fp8_product("qlin_fp8_linear", x, x_dtype, m, k, ldx, q, ldq, n, false, scale, ld_scale, bias, bias_dtype, y,
                     y_dtype, ldy, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

size_t qlin_fp8_linear_grad_input_workspace(int64_t m, int64_t n, int64_t k) {
  (void)k;
  return fp8_workspace(m, n);
}

int qlin_fp8_linear_grad_input(const void* dy, int dy_dtype, int64_t m, int64_t n, int64_t lddy, const void* q,
                               int64_t ldq, int64_t k, const float* scale, int64_t ld_scale, void* dx, int dx_dtype,
                               int64_t lddx, void* workspace, size_t workspace_bytes, void* stream) {
  return fp8_product("qlin_fp8_linear_grad_input", dy, dy_dtype, m, n, lddy, q, ldq, k, true, scale, ld_scale, nullptr,
                     0, dx, dx_dtype, lddx, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

int qlin_quantize_rows_fp8(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, void* out, int64_t ldo,
                           float* scale, int64_t ld_scale, void* stream) {
  const int64_t kp = (k + 127) / 128 * 128;
  const int64_t most = 0x7fffffff - 512;
  if (m < 0 || k < 0 || m > most || k > most || (m > 1 && (ldx < k || ldo < kp)) || ld_scale < m) {
    set_error("qlin_quantize_rows_fp8: bad sizes m=%lld k=%lld ldx=%lld ldo=%lld ld_scale=%lld", (long long)m,
              (long long)k, (long long)ldx, (long long)ldo, (long long)ld_scale);
    return QLIN_EINVAL;
  }
  if (!is_float(x_dtype) || (reinterpret_cast<uintptr_t>(out) & 7) || ldo % 8 != 0) {
    set_error("qlin_quantize_rows_fp8: x is f32, f16 or bf16, rows of out are 8-byte aligned");
    return QLIN_EDECLINE;
  }
  if (m == 0 || k == 0) return QLIN_OK;
  if (x == nullptr || out == nullptr || scale == nullptr) {
    set_error("qlin_quantize_rows_fp8: null pointer");
    return QLIN_EINVAL;
  }
  return launch_quant_rows_fp8(x, x_dtype, ldx, (int)m, (int)k, reinterpret_cast<uint8_t*>(out), ldo, scale, ld_scale,
                               reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
