// Block-scaled 8-bit linear and its input gradient: the row quantizer, the GEMM's host launcher and the
// C ABI (include/qlin.h).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/qlin.h"
#include "qlin_fp8.cuh"
#include "qlin_fp8_quant.cuh"
#include "qlin_fp8_small.cuh"
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
// side by side in the block-major scale array, go out as one 32-byte piece.  Values stay as they are stored until
// they are scaled: four CTAs on an SM in 16 bits.  Measured: 4608 x 16384 bf16 in 37 us (6.1 TB/s read and
// written), 4608 x 6144 in 17; rows off 16-byte boundaries, 7993 x 4565 bf16, 27 us (4.1 TB/s), where 7993 x 4568 on
// them takes 21: a row's words are shifted to their places with nine shuffles instead of one.
// ---------------------------------------------------------------------------------------------
struct QuantFp8Params {
  const void* x;
  long long ldx;
  int M, K, kb;      // kb = blocks of 128, the last one padded with zeros
  int k_pairs;       // pairs of blocks
  uint8_t* q;
  long long ldq;
  float* scale;      // [kb][ld_scale]
  long long ld_scale;
  long long lim_x, lim_q, lim_scale;  // element counts for the QLIN_CHECKS build
};

// The w-th aligned 16-byte word around address at; zeros from the row's end on.  A word that reaches past the caller's
// values [base, end) is read value by value.
template <int kBytes>
__device__ __forceinline__ uint4 aligned_word(const uint8_t* at, int w, const uint8_t* row_end, const uint8_t* base,
                                              const uint8_t* end) {
  const uint8_t* from = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(at) & ~uintptr_t(15)) + w * 16;
  if (from >= row_end) return uint4{};
  if (from >= base && from + 16 <= end) return *reinterpret_cast<const uint4*>(from);
  uint32_t o[4] = {};
#pragma unroll
  for (int j = 0; j < 16 / kBytes; ++j) {
    const uint8_t* e = from + j * kBytes;
    if (e < base || e >= end) continue;
    if constexpr (kBytes == 4) o[j] = *reinterpret_cast<const uint32_t*>(e);
    else o[j / 2] |= (uint32_t) * reinterpret_cast<const uint16_t*>(e) << (16 * (j & 1));
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <int DT, bool kVec>
__global__ void __launch_bounds__(256, DT == QLIN_F32 ? 2 : 4) quant_rows_fp8_kernel(const QuantFp8Params p) {
  constexpr int kRows = 8;
  griddep_launch();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t item = blockIdx.x * 8u + warp;  // a warp takes 8 rows of two blocks; neighbours the next blocks
  const int row_tile = (int)(item / (uint32_t)p.k_pairs);
  const int b = (int)(item - (uint32_t)row_tile * (uint32_t)p.k_pairs) * 2 + (lane >> 4);
  const int m0 = row_tile * kRows;
  if (m0 >= p.M) return;
  const int c = b * 128 + (lane & 15) * 8;
  const int rows = min(kRows, p.M - m0);
  Raw8<DT> raw[kRows];  // kept as stored: as fp32 they would take twice the registers
  if constexpr (!kVec) {
    // Rows that start off a 16-byte boundary: every lane reads the aligned words its values begin in, and takes
    // what they end in from the next lane; the words after the last lane's are read by a lane for each row.
    constexpr int kBytes = DT == QLIN_F32 ? 4 : 2;
    constexpr int kOwn = kBytes / 2;  // words of 16 bytes
    const int b0 = b - (lane >> 4);
    const uint8_t* base = reinterpret_cast<const uint8_t*>(p.x);
    const uint8_t* end = base + p.lim_x * kBytes;
    uint4 own[kRows][kOwn];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const uint8_t* row = base + (long long)(m0 + min(i, rows - 1)) * p.ldx * kBytes;
#pragma unroll
      for (int w = 0; w < kOwn; ++w)
        own[i][w] = aligned_word<kBytes>(row + (long long)c * kBytes, w, row + (long long)p.K * kBytes, base, end);
    }
    const uint8_t* my_row = base + (long long)(m0 + min(lane & 7, rows - 1)) * p.ldx * kBytes;
    const uint4 past = lane < 8 ? aligned_word<kBytes>(my_row + (b0 * 128ll + 256) * kBytes, 0,
                                                       my_row + (long long)p.K * kBytes, base, end)
                                : uint4{};
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      Around8<DT> a;
      const uint8_t* at = base + ((long long)(m0 + min(i, rows - 1)) * p.ldx + c) * kBytes;
      a.off = (uint32_t)(reinterpret_cast<uintptr_t>(at) & 15);
#pragma unroll
      for (int w = 0; w < kOwn; ++w) a.v[w] = own[i][w];
      uint4 next;
      next.x = __shfl_down_sync(0xffffffffu, own[i][0].x, 1);
      next.y = __shfl_down_sync(0xffffffffu, own[i][0].y, 1);
      next.z = __shfl_down_sync(0xffffffffu, own[i][0].z, 1);
      next.w = __shfl_down_sync(0xffffffffu, own[i][0].w, 1);
      uint4 last;
      last.x = __shfl_sync(0xffffffffu, past.x, i);
      last.y = __shfl_sync(0xffffffffu, past.y, i);
      last.z = __shfl_sync(0xffffffffu, past.z, i);
      last.w = __shfl_sync(0xffffffffu, past.w, i);
      a.v[kOwn] = lane == 31 ? last : next;
      raw[i] = a.values();
      if (c + 8 > p.K) raw[i] = raw8_first<DT>(raw[i], p.K - c);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const long long at = (long long)(m0 + min(i, rows - 1)) * p.ldx + c;
      raw[i] = Raw8<DT>{};
      if (c < p.K && qchk_span(BS_FP8_QUANT, at, min(8, p.K - c), p.lim_x))
        raw[i] = c + 8 <= p.K ? load_raw8<DT>(p.x, at) : gather_raw8<DT>(p.x, at, p.K - c);
    }
  }
  // Each of the 16 lanes ends up with the maximum of one of the 8 rows (two lanes to a row): at every
  // step a lane hands the half of its rows to its partner that it does not keep.
  uint32_t a[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    a[i] = max(kAmaxFloorBits, raw8_amax_bits<DT>(raw[i]));
  }
#pragma unroll
  for (int o = 8, n = 4; o > 1; o >>= 1, n >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const uint32_t give = up ? a[i] : a[i + n], keep = up ? a[i + n] : a[i];
      a[i] = max(keep, __shfl_xor_sync(0xffffffffu, give, o));
    }
  }
  a[0] = max(a[0], __shfl_xor_sync(0xffffffffu, a[0], 1));
  const float amax = __uint_as_float(a[0]);  // of row (lane >> 1) & 7
  const float up = __fdiv_rn(kE4m3Max, amax);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const float r = __shfl_sync(0xffffffffu, up, (lane & 16) | (i << 1));
    if (i < rows && b < p.kb) {
      const long long at = (long long)(m0 + i) * p.ldq + c;
      float f[8];
      raw8_to_float<DT>(raw[i], f);
      if (qchk_span(BS_FP8_QUANT, at, 8, p.lim_q))
        *reinterpret_cast<uint2*>(p.q + at) = make_uint2(to_e4m3x4(f[0], f[1], f[2], f[3], r),
                                                         to_e4m3x4(f[4], f[5], f[6], f[7], r));
    }
  }
  const int row = (lane >> 1) & 7;
  if ((lane & 1) == 0 && row < rows && b < p.kb) {
    const long long at = (long long)b * p.ld_scale + m0 + row;
    if (qchk(BS_FP8_QUANT, at, p.lim_scale)) p.scale[at] = __fdiv_rn(amax, kE4m3Max);
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
  p.k_pairs = (p.kb + 1) / 2;
  p.q = q;
  p.ldq = ldq;
  p.scale = scale;
  p.ld_scale = ld_scale;
  p.lim_x = (long long)(M - 1) * ldx + K;
  p.lim_q = (long long)(M - 1) * ldq + (long long)p.kb * 128;
  p.lim_scale = (long long)(p.kb - 1) * ld_scale + M;
  const long long grid = ((long long)((M + 7) / 8) * p.k_pairs + 7) / 8;
  if (grid > 0x7fffffff / 8) {
    set_error("fp8 quantizer: %d rows of %d columns are too many", M, K);
    return QLIN_EINVAL;
  }
  const int esz = x_dtype == QLIN_F32 ? 4 : 2;
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * esz) % 16 == 0;
  const dim3 ctas((unsigned)grid), threads(256);
  cudaError_t e;
#define QLIN_QUANT_FP8(DT)                                                                    \
  e = vec ? launch_dependent(quant_rows_fp8_kernel<DT, true>, ctas, threads, 0, stream, 0, p) \
          : launch_dependent(quant_rows_fp8_kernel<DT, false>, ctas, threads, 0, stream, 0, p);
  if (x_dtype == QLIN_F16) { QLIN_QUANT_FP8(QLIN_F16) }
  else if (x_dtype == QLIN_BF16) { QLIN_QUANT_FP8(QLIN_BF16) }
  else { QLIN_QUANT_FP8(QLIN_F32) }
#undef QLIN_QUANT_FP8
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
static int launch_fp8(const CUtensorMap& tx, const CUtensorMap& tw, const CUtensorMap& ty, const Fp8Params& p,
                      cudaStream_t stream) {
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
  const int share = CTAS == 2 ? 2 : p.splits;
  const cudaError_t e = launch_dependent(kern, dim3((unsigned)(share * std::min(tiles, sm_count() / share))),
                                         dim3(Cfg::kThreads), Cfg::kSmem, stream, (unsigned)share, tx, tw, ty, p);
  if (e != cudaSuccess) {
    set_error("fp8 gemm launch failed: %s", cudaGetErrorString(e));
    return QLIN_ECUDA;
  }
  return QLIN_OK;
}

template <bool kTrans, int DT>
static int launch_fp8_small(const CUtensorMap& tw, const Fp8SmallParams& p, cudaStream_t stream) {
  using Cfg = Fp8SmallCfg;
  auto kern = fp8_small_kernel<kTrans, DT>;
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
  // CTAs that share a tile's contraction: as many (up to 8, three blocks each at least: one token 256 -> 5120 takes
  // 4.9 us alone and 5.3 shared by two) as the machine takes at once.
  const int tiles = (p.N + 127) / 128;
  const int at_once = sm_count() * Cfg::kCtas;
  int splits = 1;
  while (splits < 8 && splits * 2 * 3 <= p.kb && tiles * splits * 2 <= at_once) splits *= 2;
  const cudaError_t e = launch_dependent(kern, dim3((unsigned)(tiles * splits)), dim3(Cfg::kThreads), Cfg::kSmem, stream,
                                         (unsigned)splits, tw, p, splits);
  if (e != cudaSuccess) {
    set_error("fp8 small-M launch failed: %s", cudaGetErrorString(e));
    return QLIN_ECUDA;
  }
  return QLIN_OK;
}

template <bool kTrans>
static int run_fp8_small(int x_dtype, const CUtensorMap& tw, const Fp8SmallParams& p, cudaStream_t stream) {
  if (x_dtype == QLIN_F16) return launch_fp8_small<kTrans, QLIN_F16>(tw, p, stream);
  if (x_dtype == QLIN_BF16) return launch_fp8_small<kTrans, QLIN_BF16>(tw, p, stream);
  return launch_fp8_small<kTrans, QLIN_F32>(tw, p, stream);
}

// Up to this many tokens the small-M kernel runs, which quantizes them itself and needs no workspace.
constexpr int64_t kSmallM = Fp8SmallCfg::TN;

// Which kernel and how many CTAs to a tile.  Measured with warm operands, a block of 128 contraction indices takes
// a pair's 256 x 256 tile about 790 clocks and a single CTA's 128 x 128 tile about 560, so the pair wins where
// both fill their last wave alike (1024 x 4096 x 4096: 22 us against two waves of single tiles), the single tiles
// where the pair's leave SMs idle (333 x 4096 x 5120: 14.8 us, the pair 21.9).  Where they leave half of the
// machine free, 2, 4 or 8 CTAs share a tile's contraction, at least 4 blocks each; their join costs about 5500
// clocks (128 x 4096 x 5120: 12.8 us shared by two, 17 alone; 128 x 1024 x 5120: 10 and 8).
struct Fp8Plan {
  bool pair;
  int splits;
};

constexpr int64_t kGroupBytes = 40 << 20;  // measured 8 to 80 MB: 4608 x 6144 x 16384 474, 471, 465, 455, 455, 456 us

static Fp8Plan plan_fp8(int64_t m_tiles, int64_t n_tiles, int64_t kb) {
  const int64_t sms = sm_count();
  const auto waves = [](int64_t tiles, int64_t at_once) { return (tiles + at_once - 1) / at_once; };
  Fp8Plan best{true, 1};
  int64_t cost = waves(((m_tiles + 1) / 2) * ((n_tiles + 1) / 2), sms / 2) * kb * 790;
  for (int s = 1; s <= 8; s *= 2) {
    if (s > 1 && (m_tiles * n_tiles * s > sms || kb < 4 * s)) break;
    const int64_t c = waves(m_tiles * n_tiles, sms / s) * ((kb + s - 1) / s) * 560 + (s > 1 ? 5500 : 0);
    if (c < cost) {
      cost = c;
      best = Fp8Plan{false, s};
    }
  }
  return best;
}

static size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

// Workspace: the e4m3 activations [m, round_up(depth, 128)] and their scales [blocks][m].
static size_t fp8_workspace(int64_t m, int64_t depth) {
  if (m <= kSmallM || depth <= 0) return 0;
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
  const int esz = y_dtype == QLIN_F32 ? 4 : 2;
  const int y_kind = y_dtype == QLIN_F32 ? OUT_F32 : y_dtype == QLIN_F16 ? OUT_F16 : OUT_BF16;
  const int64_t sw_out = trans ? 1 : ld_scale, sw_red = trans ? ld_scale : 1;
  const int64_t lim_sw = ((rows + 127) / 128 - 1) * ld_scale + (cols + 127) / 128;
  CUtensorMap tx{}, tw{}, ty{};
  if (kb > 0) {
    const int rc = make_tmap_2d(&tw, q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)cols, (uint64_t)rows,
                                rows > 1 ? (uint64_t)ldq : (uint64_t)cols, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  if (m <= kSmallM && kb > 0) {
    Fp8SmallParams p{};
    p.x = x;
    p.x_vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (m == 1 || (ldx * (x_dtype == QLIN_F32 ? 4 : 2)) % 16 == 0);
    p.ldx = ldx;
    p.M = (int)m;
    p.N = (int)out;
    p.K = (int)depth;
    p.kb = kb;
    p.sw = scale;
    p.sw_out = sw_out;
    p.sw_red = sw_red;
    p.bias = bias;
    p.bias_kind = bk;
    p.y = y;
    p.y_dtype = y_kind;
    p.ldy = ldy;
    p.status = reinterpret_cast<DeviceStatus*>(device_status_ptr());
    p.lim_x = (m - 1) * ldx + depth;
    p.lim_y = (m - 1) * ldy + out;
    p.lim_sw = lim_sw;
    return trans ? run_fp8_small<true>(x_dtype, tw, p, stream) : run_fp8_small<false>(x_dtype, tw, p, stream);
  }
  uint8_t* xq = reinterpret_cast<uint8_t*>(workspace);
  float* sx = reinterpret_cast<float*>(xq + align256((size_t)m * kp));
  Fp8Params p{};
  p.M = (int)m;
  p.N = (int)out;
  p.kb = kb;
  p.sx = sx;
  p.ld_sx = m;
  p.sw = scale;
  p.sw_out = sw_out;
  p.sw_red = sw_red;
  p.bias = bias;
  p.bias_kind = bk;
  p.y = y;
  p.y_dtype = y_kind;
  p.ldy = ldy;
  p.tma_out = (reinterpret_cast<uintptr_t>(y) & 15) == 0 && (ldy * esz) % 16 == 0;
  p.status = reinterpret_cast<DeviceStatus*>(device_status_ptr());
  p.lim_y = (m - 1) * ldy + out;
  p.lim_sx = (long long)kb * m;
  p.lim_sw = lim_sw;
  const int64_t m_tiles = (m + 127) / 128, n_tiles = (out + 127) / 128;
  if (m_tiles * n_tiles > 0x7fffffff) {
    set_error("%s: too many output tiles", what);
    return QLIN_EINVAL;
  }
  const Fp8Plan plan = plan_fp8(m_tiles, n_tiles, kb);
  const bool pair = plan.pair;
  p.splits = plan.splits;
  p.m_tiles = (int)(pair ? (m_tiles + 1) / 2 : m_tiles);
  p.n_tiles = (int)(pair ? (n_tiles + 1) / 2 : n_tiles);
  // Groups of equal size whose e4m3 tokens take at most kGroupBytes of L2: every group streams the weight once.
  const int64_t tile_bytes = (pair ? 256 : 128) * std::max<int64_t>(kp, 128);
  const int64_t fit = std::min<int64_t>(std::max<int64_t>(kGroupBytes / tile_bytes, 1), 1 << 16);
  const int64_t groups = (p.m_tiles + fit - 1) / fit;
  p.group = (int)((p.m_tiles + groups - 1) / groups);
  if (p.tma_out) {
    const int rc = make_tmap_2d(&ty, y, y_dtype == QLIN_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                        : y_dtype == QLIN_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                              : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                                esz, (uint64_t)out, (uint64_t)m, (uint64_t)ldy * esz, 128 / esz, 32,
                                CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  if (kb > 0) {
    int rc = launch_quant_rows_fp8(x, x_dtype, ldx, (int)m, (int)depth, xq, kp, sx, m, stream);
    if (rc) return rc;
    rc = make_tmap_2d(&tx, xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)kp, (uint64_t)m, (uint64_t)kp, 128, 128,
                      CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  if (pair) return trans ? launch_fp8<2, 256, true>(tx, tw, ty, p, stream) : launch_fp8<2, 256, false>(tx, tw, ty, p, stream);
  return trans ? launch_fp8<1, 128, true>(tx, tw, ty, p, stream) : launch_fp8<1, 128, false>(tx, tw, ty, p, stream);
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
