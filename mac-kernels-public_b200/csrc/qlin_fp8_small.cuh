// The block-scaled 8-bit linear for few tokens (up to 16), in one launch without a workspace.
//
// With few tokens the weight's bytes are everything, so the roles of the operands are exchanged: a CTA
// streams 128 output channels' weight tiles through TMA and multiplies them, as the MMA's 128 rows, by the
// tokens as its TN = 16 columns.  The tokens' values are quantized here, block by block
// beside the stream, straight into the swizzled operand tile: every CTA does it again from L2, which costs less
// than a launch of its own and its round trip through memory.  Where the channels alone give too few CTAs to
// keep HBM busy, a cluster of up to 8 CTAs shares the contraction and joins its sums through distributed shared
// memory in a fixed order.
//
// Every block's products have a TMEM buffer of their own, as in the large kernel; a thread owns one channel,
// each token's scale comes from shared memory.
//
// Measured: 2 x 5120 -> 30720 in 27.2 us, 5.8 TB/s of weights (88% of a copy's rate; two CTAs of six 18 KB stages
// on an SM keep it busy), one token 256 -> 5120 in 3.8 us, of which the products are the smallest part.  Sixteen tokens
// 5120 -> 30720 take 30 us in 16 bits and 51 in fp32, whose quantizers hold twice the bytes: 28 of a thread's spill at
// the 80 registers that two CTAs on an SM leave.
//
// Warp roles (384 threads, one tile to a CTA):
//   warp 0       weight stream (TMA)       warp 1   TMEM alloc + MMA issuer
//   warps 2..7   quantizers                warps 8..11   rescale, join, output
#pragma once
#include <cuda.h>

#include "qlin_fp8_quant.cuh"
#include "qlin_ptx.cuh"

namespace qlin {

struct Fp8SmallParams {
  const void* x;
  int x_vec;        // rows of x take 16-byte loads
  long long ldx;
  int M, N, K;      // tokens, output channels, contraction
  int kb;           // blocks of 128 along the contraction
  const float* sw;  // block (output o, contraction r) at o * sw_out + r * sw_red
  long long sw_out, sw_red;
  const void* bias;
  int bias_kind;
  void* y;
  int y_dtype;
  long long ldy;
  DeviceStatus* status;
  // Element counts of the caller's buffers for the QLIN_CHECKS build (unused otherwise).
  long long lim_x, lim_y, lim_sw;
};

struct Fp8SmallCfg {
  static constexpr int TN = 16;
  static constexpr int kThreads = 384;
  static constexpr int kCtas = 2;  // resident on an SM
  static constexpr int kRing = 6;  // stages, TMEM buffers and scale slots
  static constexpr uint32_t kWStage = 128 * 128;
  static constexpr uint32_t kXStage = TN * 128;
  static constexpr uint32_t kTmemCols = 128;  // a power of two of at least kRing * TN
  static constexpr int kSmem = 1024 + kRing * (int)(kWStage + kXStage) + kRing * TN * 4 + 256;
  static_assert(kRing * TN <= kTmemCols && kCtas * kTmemCols <= 512 && kCtas * kSmem <= 228 * 1024, "resident CTAs");
  static_assert(TN * 128 * 4 <= kRing * (int)kWStage, "the joined sums fit into the weight ring");
};

// 8 consecutive values of row m from column c as they are stored, zeros past M and K.
template <int DT>
__device__ __forceinline__ Raw8<DT> small_load8(const Fp8SmallParams& p, int m, int c) {
  Raw8<DT> raw{};
  const long long at = (long long)m * p.ldx + c;
  if (m >= p.M || c >= p.K) return raw;
  if (c + 8 <= p.K) {
    if (qchk_span(BS_FP8_X, at, 8, p.lim_x))
      raw = p.x_vec ? load_raw8<DT>(p.x, at) : load_raw8_any<DT>(p.x, at, p.lim_x);
    return raw;
  }
  return qchk_span(BS_FP8_X, at, p.K - c, p.lim_x) ? gather_raw8<DT>(p.x, at, p.K - c) : raw;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <bool kTrans, int DT>
__global__ void __launch_bounds__(384, Fp8SmallCfg::kCtas)
fp8_small_kernel(const __grid_constant__ CUtensorMap tmap_w, const Fp8SmallParams p, int splits) {
  using Cfg = Fp8SmallCfg;
  constexpr int TN = Cfg::TN;
  constexpr int R = Cfg::kRing;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sw = smem;
  uint8_t* sx = sw + R * Cfg::kWStage;
  float* scale = reinterpret_cast<float*>(sx + R * Cfg::kXStage);  // [R][TN]
  uint64_t* bars = reinterpret_cast<uint64_t*>(scale + R * TN);
  uint64_t* w_full = bars;            // weight tile landed
  uint64_t* x_full = w_full + R;      // quantized tile and its scales written
  uint64_t* empty = x_full + R;       // MMAs that read the stage completed
  uint64_t* acc_full = empty + R;     // products ready
  uint64_t* acc_empty = acc_full + R; // products and scales read
  uint64_t* drain = acc_empty + R;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = blockIdx.x % splits;
  const int nt = blockIdx.x / splits;
  const int b_begin = (int)((long long)p.kb * rank / splits), b_end = (int)((long long)p.kb * (rank + 1) / splits);
  const int blocks = b_end - b_begin;

  if (threadIdx.x == 0) {
    for (int s = 0; s < R; ++s) {
      mbar_init(&w_full[s], 1);
      mbar_init(&x_full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], 4);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    // the carve-out (rings, barriers, flags) lies inside the launch's shared memory
    if (!qchk_smem(BS_FP8_SMEM, smem_raw, bars, reinterpret_cast<volatile uint8_t*>(abort_flag + 1) -
                                          reinterpret_cast<volatile uint8_t*>(bars)))
      *abort_flag = 1;
    fence_mbar_init();
    prefetch_tmap(&tmap_w);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_launch();
  griddep_wait();
  float acc[TN];  // rescale warps: this channel's sums, a token each

  if (warp == 0) {
    // --------------------------------------------------------------------- weight stream
    if (elect_one()) {
      bool ok = true;
      int i = 0;
      for (; i < blocks; ++i) {
        const int s = i % R, b = b_begin + i;
        if (!mbar_wait(&empty[s], ((i / R) & 1) ^ 1, abort_flag, p.status, 0x51)) { ok = false; break; }
        mbar_arrive_expect_tx(&w_full[s], Cfg::kWStage);
        tma_load_2d(sw + s * Cfg::kWStage, &tmap_w, &w_full[s], kTrans ? nt * 128 : b * 128, kTrans ? b * 128 : nt * 128);
      }
      if (!ok) {  // wait for the copies in flight
        for (int j = (i >= R ? i - R : 0); j < i; ++j) {
          const uint64_t t0 = globaltimer();
          while (!mbar_try_wait(smem_u32(&w_full[j % R]), (j / R) & 1)) {
            if (globaltimer() - t0 > QLIN_WAIT_TIMEOUT_NS) break;
          }
        }
      }
    }
  } else if (warp == 1) {
    // --------------------------------------------------------------------- MMA issuer
    if (elect_one()) {
      constexpr uint32_t idesc = idesc_e4m3_f32(128, TN, kTrans, false);
      constexpr uint64_t kAStep = kTrans ? (32 * 128) >> 4 : 32 >> 4;  // 32 contraction indices of one MMA
      for (int i = 0; i < blocks; ++i) {
        const int s = i % R;
        const uint32_t ph = (i / R) & 1;
        if (!mbar_wait(&w_full[s], ph, abort_flag, p.status, 0x52) ||
            !mbar_wait(&x_full[s], ph, abort_flag, p.status, 0x53) ||
            !mbar_wait(&acc_empty[s], ph ^ 1, abort_flag, p.status, 0x54))
          break;
        tc_fence_after();
        const uint32_t sw_u = smem_u32(sw + s * Cfg::kWStage);
        const uint64_t a_desc = kTrans ? smem_desc_sw128_mn(sw_u) : smem_desc_sw128(sw_u);
        const uint64_t b_desc = smem_desc_sw128(smem_u32(sx + s * Cfg::kXStage));
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_f8_ss(tmem_base + s * TN, a_desc + (uint64_t)kk * kAStep, b_desc + (uint64_t)(kk * 2), idesc, kk > 0);
        tc_commit(&acc_full[s]);
        tc_commit(&empty[s]);
      }
      tc_commit(drain);
      const uint64_t t0 = globaltimer();
      while (!mbar_try_wait(smem_u32(drain), 0)) {
        if (globaltimer() - t0 > QLIN_WAIT_TIMEOUT_NS) break;
      }
    }
  } else if (warp < 8) {
    // --------------------------------------------------------------------- quantizers
    // A warp takes every sixth block, 8 tokens of it at a time, 16 lanes to a token's block; the next 8
    // tokens' values (of this or of its next block) are in flight meanwhile.
    constexpr int kPairs = 4, kWarps = 6;
    const int groups = (min(p.M, TN) + 7) / 8;
    const int col = (lane & 15) * 8;
    Raw8<DT> raw[kPairs];
    auto load = [&](int i, int g) {
#pragma unroll
      for (int u = 0; u < kPairs; ++u)
        raw[u] = small_load8<DT>(p, g * 8 + u * 2 + (lane >> 4), (b_begin + i) * 128 + col);
    };
    bool ok = true;
    if (warp - 2 < blocks) load(warp - 2, 0);
    for (int i = warp - 2; i < blocks && ok; i += kWarps) {
      const int s = i % R;
      uint8_t* tile = sx + s * Cfg::kXStage;
      for (int g = 0; g < groups; ++g) {
        Raw8<DT> now[kPairs];  // kept as stored: as fp32 they would take twice the registers
        uint32_t a[kPairs];
#pragma unroll
        for (int u = 0; u < kPairs; ++u) {
          now[u] = raw[u];
          a[u] = max(kAmaxFloorBits, raw8_amax_bits<DT>(now[u]));
        }
        if (g + 1 < groups) load(i, g + 1);
        else if (i + kWarps < blocks) load(i + kWarps, 0);
        // each lane ends up with the maximum of pair (lane >> 2) & 3 of its half, as in the row quantizer
#pragma unroll
        for (int o = 8, n = 2; o > 2; o >>= 1, n >>= 1) {
          const bool up = lane & o;
#pragma unroll
          for (int u = 0; u < n; ++u) {
            const uint32_t give = up ? a[u] : a[u + n], keep = up ? a[u + n] : a[u];
            a[u] = max(keep, __shfl_xor_sync(0xffffffffu, give, o));
          }
        }
        a[0] = max(a[0], __shfl_xor_sync(0xffffffffu, a[0], 2));
        a[0] = max(a[0], __shfl_xor_sync(0xffffffffu, a[0], 1));
        const float amax = __uint_as_float(a[0]);
        const float up = __fdiv_rn(kE4m3Max, amax);
        if (g == 0) {
          const uint32_t ph = ((i / R) & 1) ^ 1;
          if (!mbar_wait(&empty[s], ph, abort_flag, p.status, 0x55) ||
              !mbar_wait(&acc_empty[s], ph, abort_flag, p.status, 0x56)) {
            ok = false;
            break;
          }
        }
        if ((lane & 3) == 0) scale[s * TN + g * 8 + ((lane >> 2) & 3) * 2 + (lane >> 4)] = __fdiv_rn(amax, kE4m3Max);
#pragma unroll
        for (int u = 0; u < kPairs; ++u) {
          const float r = __shfl_sync(0xffffffffu, up, (lane & 16) | (u << 2));
          const int j = g * 8 + u * 2 + (lane >> 4);
          float f[8];
          raw8_to_float<DT>(now[u], f);
          uint8_t* at = tile + j * 128 + ((((lane & 15) >> 1) ^ (j & 7)) << 4) + (lane & 1) * 8;
          if (qchk_smem(BS_FP8_SMEM, smem_raw, at, 8))
            *reinterpret_cast<uint2*>(at) = make_uint2(to_e4m3x4(f[0], f[1], f[2], f[3], r),
                                                       to_e4m3x4(f[4], f[5], f[6], f[7], r));
        }
      }
      if (!ok) break;
      fence_proxy_async_smem();  // the MMA reads the tile through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive(&x_full[s]);
    }
  } else {
    // --------------------------------------------------------------------- rescale
    const int quarter = warp & 3;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[j] = 0.f;
    const long long sw_off = (long long)nt * p.sw_out;
    auto load_sw = [&](int i) {
      const long long at = sw_off + (long long)(b_begin + min(i, blocks - 1)) * p.sw_red;
      return qchk(BS_FP8_SCALE, at, p.lim_sw) ? p.sw[at] : 0.f;
    };
    float w_next = blocks > 0 ? load_sw(0) : 0.f;
    for (int i = 0; i < blocks; ++i) {
      const int s = i % R;
      const uint32_t ph = (i / R) & 1;
      const float w = w_next;
      w_next = load_sw(i + 1);
      if (!mbar_wait(&x_full[s], ph, abort_flag, p.status, 0x57) ||  // the scales were written before it
          !mbar_wait(&acc_full[s], ph, abort_flag, p.status, 0x58))
        break;
      tc_fence_after();
      uint32_t v[TN];
      tmem_ld_cols<TN>(tmem_base + lanes + s * TN, v);
      tmem_wait_ld_of(v);
#pragma unroll
      for (int j = 0; j < TN; j += 4) {
        const float4 t = *reinterpret_cast<const float4*>(&scale[s * TN + j]);
        acc[j] = fmaf(__uint_as_float(v[j]), t.x * w, acc[j]);
        acc[j + 1] = fmaf(__uint_as_float(v[j + 1]), t.y * w, acc[j + 1]);
        acc[j + 2] = fmaf(__uint_as_float(v[j + 2]), t.z * w, acc[j + 2]);
        acc[j + 3] = fmaf(__uint_as_float(v[j + 3]), t.w * w, acc[j + 3]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[s]);
    }
  }

  // Warps 0 and 1 ran their loops on one elected lane; reconverge before the block barriers.  Every copy
  // has landed and every MMA completed (the issuer waited for its last commit), so the ring is free.
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
  const bool aborted = *abort_flag != 0;
  float* joint = reinterpret_cast<float*>(sw);  // [TN][128]
  const int r = (warp & 3) * 32 + lane;
  const int n = nt * 128 + r;
  auto put = [&](int j, float v) {
    const long long at = (long long)j * p.ldy + n;
    if (!qchk(BS_FP8_Y, at, p.lim_y)) return;
    if (p.y_dtype == OUT_F32) reinterpret_cast<float*>(p.y)[at] = v;
    else if (p.y_dtype == OUT_F16) reinterpret_cast<__half*>(p.y)[at] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v);
  };
  if (splits == 1) {
    if (warp >= 8 && n < p.N && !aborted) {
      const float bias = fp8_bias(p.bias, p.bias_kind, n, p.N);
#pragma unroll
      for (int j = 0; j < TN; ++j)
        if (j < p.M) put(j, acc[j] + bias);
    }
    return;
  }
  if (warp >= 8) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
      if (j < p.M) joint[j * 128 + r] = acc[j];
  }
  cluster_sync();
  // Token j is joined by CTA j % splits, all twelve warps of it: three sets of 128 channels' threads.
  if (n < p.N && !aborted) {
    const float bias = fp8_bias(p.bias, p.bias_kind, n, p.N);
    for (int j = rank + splits * (warp >> 2); j < p.M; j += splits * 3) {
      float part[8], v = bias;  // all parts' loads in flight
#pragma unroll
      for (int c = 0; c < 8; ++c) part[c] = c < splits ? ld_cluster_f32(cluster_map(&joint[j * 128 + r], c)) : 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) v += c < splits ? part[c] : 0.f;
      put(j, v);
    }
  }
  cluster_sync();  // no CTA leaves while another reads its sums
}

}  // namespace qlin
