// Block-scaled 8-bit linear on the tensor cores (tcgen05.mma kind::f8f6f4, fp32 accumulation).
//
//   Y[m, n] = sum_b sx[b][m] * S[n / 128][b] * P_b[m, n]  (+ bias[n]),
//   P_b[m, n] = sum_{d in block b of 128} xq[m, d] * W[n, d]
//
// xq are the activations in e4m3 with one scale per row and block (the row quantizer below), W the
// stored e4m3 weight with one scale S per 128 x 128 block.  The input gradient is the same sum with the
// weight's rows as the contraction (kTrans): W is then read as it lies, as a transposed operand.
//
// The scales change with every block, so each block's products go to a TMEM buffer of their own and
// the epilogue warps fold them into fp32 registers, one packed FMA per two values, while the tensor
// cores fill the next buffer.  Tokens lie on the TMEM lanes: a thread owns one token, whose scale times
// the warp's block scale is one factor for all of its values.
//
// Measured at 4608 x 6144 x 16384 (bf16): 388 us for this kernel in short bursts (2.4 PFLOP/s, tensor pipe 66%
// busy), 440 in a long row of calls, where the card's power limit sets the clock to 1.46 GHz.  Without the rescale
// it takes a fifth less; L2 (36%) and DRAM (8%) wait.  The rescale's own cost is its instructions, about 160 a
// warp and block, 64 of them packed FMAs; TMEM loads of 16 or 32 columns and one or two in flight take the same.
//
// Warp roles (384 threads, one CTA per SM, persistent over the tiles):
//   warp 0        TMA producer            warp 1   TMEM alloc + MMA issuer       (warps 2, 3 idle)
//   warps 4..11   rescale + epilogue: two warps per TMEM lane quarter, half the columns each
// A pair's epilogue warps hold 128 running sums a thread and take over most of the first warpgroup's
// registers.
#pragma once
#include <cuda.h>

#include <type_traits>

#include "qlin_ptx.cuh"

namespace qlin {

struct Fp8Params {
  int M, N;       // tokens, output channels
  int kb;         // blocks of 128 along the contraction
  int m_tiles, n_tiles;
  int group;        // token tiles that stay in L2 together
  const float* sx;  // [kb][ld_sx]
  long long ld_sx;
  const float* sw;  // block (output o, contraction r) at o * sw_out + r * sw_red
  long long sw_out, sw_red;
  const void* bias;
  int bias_kind;    // 0 none, 1 f16, 2 f32, 3 bf16
  void* y;
  int y_dtype;      // OutDType
  long long ldy;
  int splits;       // single CTAs only: CTAs (a cluster) that share a tile's contraction
  int tma_out;      // y's rows are 16-byte aligned: the output leaves through tmap_y
  DeviceStatus* status;
  // Element counts of the caller's buffers for the QLIN_CHECKS build (unused otherwise).
  long long lim_y, lim_sx, lim_sw;
};

// Tokens by channels of one tile: CTAS = 2 is a cluster of two CTAs that share cta_group::2 MMAs of
// 256 tokens x TN channels, each CTA holding its 128 tokens and half of the channels.
template <int CTAS, int TN>
struct Fp8Cfg {
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 128 + 32 * kEpiWarps;
  static constexpr int kBuf = 512 / TN;        // accumulator buffers in TMEM
  static constexpr int kBRows = TN / CTAS;     // channels this CTA loads per stage
  static constexpr uint32_t kAStage = 128 * 128;
  static constexpr uint32_t kBStage = kBRows * 128;
  static constexpr int kStages = 5;
  static constexpr int kCols = TN / (kEpiWarps / 4);  // accumulator columns per epilogue warp
  // output staging of a warp: its tokens' rows, 2 bytes a value, or one piece of them with kOddPitch
  static constexpr uint32_t kOutWarp = kCols == 128 ? 32 * 256 : 5 * 1024;
  static constexpr int kSmem = 1024 + kStages * (int)(kAStage + kBStage) + kEpiWarps * (int)kOutWarp + 512;
  static_assert(CTAS == 1 || CTAS == 2, "one CTA or a pair");
  static_assert(128 * 132 * 4 <= kStages * (int)(kAStage + kBStage), "the joined sums fit over the operand ring");
  static_assert(kBRows == 128, "the transposed operand is one 128-column block");
};

// Tiles in groups of `group` token tiles, tokens fastest and then channels within a group: the tiles that run at
// one time share a few token tiles and a few channel tiles, and a group's tokens stay in L2 while the channels
// stream past them.
__device__ __forceinline__ void fp8_tile(int t, int m_tiles, int n_tiles, int group, int& mt, int& nt) {
  const int per = group * n_tiles;
  const int g = t / per, r = t - g * per;
  const int rows = min(group, m_tiles - g * group);
  nt = r / rows;
  mt = g * group + (r - nt * rows);
}

// Pitch of a token's sums in shared memory, in floats: 16 bytes past a multiple of 128, so that the lanes of a
// store (a token each) fall on different banks.
constexpr int kJoinPitch = 132;

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// An ordinary load, volatile so that it stays where it is written: behind griddep_wait, and ahead of its use.
__device__ __forceinline__ float ld_f32(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}

// (a0, a1) += s * (p0, p1)
__device__ __forceinline__ void ffma2(float s, uint32_t p0, uint32_t p1, float& a0, float& a1) {
  asm("{\n\t.reg .b64 f, sc, acc;\n\t"
      "mov.b64 f, {%2, %3};\n\t"
      "mov.b64 sc, {%4, %4};\n\t"
      "mov.b64 acc, {%0, %1};\n\t"
      "fma.rn.f32x2 acc, sc, f, acc;\n\t"
      "mov.b64 {%0, %1}, acc;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "r"(p0), "r"(p1), "f"(s));
}

__device__ __forceinline__ float fp8_bias(const void* bias, int kind, long long n, long long lim) {
  if (kind == 0 || !qchk(BS_FP8_SCALE, n, lim)) return 0.f;
  if (kind == 1) return __half2float(reinterpret_cast<const __half*>(bias)[n]);
  if (kind == 2) return reinterpret_cast<const float*>(bias)[n];
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(bias)[n]);
}

__device__ __forceinline__ uint32_t pack_out2(int dtype, float a, float b) {
  if (dtype == OUT_F16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Pitch of a staged row's piece: 8 words of 16 bytes and, behind the last piece, what is left of the row.
constexpr int kOddPitch = 144;

// The first bytes of a row, up to a 16-byte boundary (or its end before that), and the last ones, from a boundary
// on, from shared memory at the same address modulo 16.
template <int kBytes>
__device__ __forceinline__ void store_head(uint8_t* g, const uint8_t* s, int bytes) {
  if (((reinterpret_cast<uintptr_t>(g) + bytes) & 15) != 0) {  // a few columns at the end of y
    for (int i = 0; i < bytes; i += kBytes) {
      if constexpr (kBytes == 2) *reinterpret_cast<uint16_t*>(g + i) = *reinterpret_cast<const uint16_t*>(s + i);
      else *reinterpret_cast<uint32_t*>(g + i) = *reinterpret_cast<const uint32_t*>(s + i);
    }
    return;
  }
  int i = 0;
  if (kBytes == 2 && (bytes & 2)) {
    *reinterpret_cast<uint16_t*>(g) = *reinterpret_cast<const uint16_t*>(s);
    i = 2;
  }
  if (bytes & 4) {
    *reinterpret_cast<uint32_t*>(g + i) = *reinterpret_cast<const uint32_t*>(s + i);
    i += 4;
  }
  if (bytes & 8) *reinterpret_cast<uint2*>(g + i) = *reinterpret_cast<const uint2*>(s + i);
}
template <int kBytes>
__device__ __forceinline__ void store_tail(uint8_t* g, const uint8_t* s, int bytes) {
  int i = 0;
  if (bytes & 8) {
    *reinterpret_cast<uint2*>(g) = *reinterpret_cast<const uint2*>(s);
    i = 8;
  }
  if (bytes & 4) {
    *reinterpret_cast<uint32_t*>(g + i) = *reinterpret_cast<const uint32_t*>(s + i);
    i += 4;
  }
  if (kBytes == 2 && (bytes & 2)) *reinterpret_cast<uint16_t*>(g + i) = *reinterpret_cast<const uint16_t*>(s + i);
}

template <int CTAS, int TN, bool kTrans>
__global__ void __launch_bounds__(Fp8Cfg<CTAS, TN>::kThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                const __grid_constant__ CUtensorMap tmap_y, const Fp8Params p) {
  using Cfg = Fp8Cfg<CTAS, TN>;
  constexpr int STAGES = Cfg::kStages;
  constexpr int NB = Cfg::kBuf;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sa = smem;
  uint8_t* sb = sa + STAGES * Cfg::kAStage;
  uint8_t* so = sb + STAGES * Cfg::kBStage;  // 8 x kOutWarp
  uint64_t* bars = reinterpret_cast<uint64_t*>(so + Cfg::kEpiWarps * Cfg::kOutWarp);
  uint64_t* full = bars;              // [STAGES] both CTAs' operands landed (even CTA's)
  uint64_t* empty = full + STAGES;    // [STAGES] MMAs that read the stage completed (each CTA's)
  uint64_t* acc_full = empty + STAGES;   // [NB] products ready (each CTA's)
  uint64_t* acc_empty = acc_full + NB;   // [NB] read out by the epilogue warps of both CTAs (even CTA's)
  uint64_t* drain = acc_empty + NB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = CTAS == 2 ? cluster_ctarank() : 0;
  const int num_tiles = p.m_tiles * p.n_tiles;
  const int share = CTAS == 2 ? 2 : p.splits;  // CTAs to a tile
  const int tile0 = blockIdx.x / share;
  const int tile_step = gridDim.x / share;
  const int part_k = CTAS == 2 ? 0 : blockIdx.x % share;
  const int b_begin = CTAS == 2 ? 0 : (int)((long long)p.kb * part_k / share);
  const int b_end = CTAS == 2 ? p.kb : (int)((long long)p.kb * (part_k + 1) / share);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < NB; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], Cfg::kEpiWarps * CTAS);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    // the carve-out (rings, barriers, flags) lies inside the launch's shared memory
    if (!qchk_smem(BS_FP8_SMEM, smem_raw, bars, reinterpret_cast<volatile uint8_t*>(abort_flag + 1) -
                                          reinterpret_cast<volatile uint8_t*>(bars)))
      *abort_flag = 1;
    fence_mbar_init();
  }
  if (warp == 1) {
    if constexpr (CTAS == 2) {
      tmem_alloc_pair(tmem_slot, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
    }
  }
  if (warp == 0 && lane == 0 && p.kb > 0) {
    prefetch_tmap(&tmap_x);
    prefetch_tmap(&tmap_w);
    if (p.tma_out) prefetch_tmap(&tmap_y);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) cluster_sync();  // both CTAs' barriers are initialized before any remote arrive
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // The quantizer's codes and scales.  No griddep_launch here: the next call's quantizer would crowd onto the SMs that
  // this kernel leaves free (333 x 4096 -> 5120: 15.8 us a call without, 17.8 with).
  griddep_wait();

  // setmaxnreg (pairs): 2 x 224 + 56 = 3 x 168, the registers of an SM quarter's three warps at launch
  if (warp < 4) {
    if constexpr (CTAS == 2) setmaxnreg_dec<56>();
    if (warp == 0) {
      // --------------------------------------------------------------------- producer (both CTAs)
      if (elect_one()) {
        const uint32_t full_leader = CTAS == 2 ? cluster_map(full, 0) : smem_u32(full);
        uint32_t it = 0;
        bool ok = true;
        for (int t = tile0; t < num_tiles && ok; t += tile_step) {
          int mt, nt;
          fp8_tile(t, p.m_tiles, p.n_tiles, p.group, mt, nt);
          const int m0 = (mt * CTAS + (int)rank) * 128;
          const int n0 = nt * TN + (int)rank * Cfg::kBRows;
          for (int b = b_begin; b < b_end; ++b, ++it) {
            const int s = it % STAGES;
            if (!mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1, abort_flag, p.status, 0x41)) { ok = false; break; }
            if (rank == 0) mbar_arrive_expect_tx(&full[s], CTAS * (Cfg::kAStage + Cfg::kBStage));
            const int wx = kTrans ? n0 : b * 128, wy = kTrans ? b * 128 : n0;
            if constexpr (CTAS == 2) {
              const uint32_t bar = full_leader + (uint32_t)(s * 8);
              tma_load_2d_pair(sa + s * Cfg::kAStage, &tmap_x, bar, b * 128, m0);
              tma_load_2d_pair(sb + s * Cfg::kBStage, &tmap_w, bar, wx, wy);
            } else {
              tma_load_2d(sa + s * Cfg::kAStage, &tmap_x, &full[s], b * 128, m0);
              tma_load_2d(sb + s * Cfg::kBStage, &tmap_w, &full[s], wx, wy);
            }
          }
        }
        if (!ok && rank == 0) {  // wait for the copies in flight (the even CTA's barriers count both CTAs' bytes)
          for (uint32_t j = (it >= (uint32_t)STAGES ? it - STAGES : 0); j < it; ++j) {
            const uint64_t t0 = globaltimer();
            while (!mbar_try_wait(smem_u32(&full[j % STAGES]), (j / STAGES) & 1)) {
              if (globaltimer() - t0 > QLIN_WAIT_TIMEOUT_NS) break;
            }
          }
        }
      }
    } else if (warp == 1) {
      // --------------------------------------------------------------------- MMA issuer (even CTA)
      if (rank == 0 && elect_one()) {
        constexpr uint32_t idesc = idesc_e4m3_f32(128 * CTAS, TN, false, kTrans);
        // 32 contraction indices of one MMA: 32 bytes of a K-major row, or 32 rows of a transposed tile
        constexpr uint64_t kBStep = kTrans ? (32 * 128) >> 4 : 32 >> 4;
        uint32_t it = 0;
        bool ok = true;
        for (int t = tile0; t < num_tiles && ok; t += tile_step) {
          for (int b = b_begin; b < b_end; ++b, ++it) {
            const int s = it % STAGES;
            const uint32_t buf = it % NB;
            if (!mbar_wait<CTAS == 2>(&full[s], (it / STAGES) & 1, abort_flag, p.status, 0x42) ||
                !mbar_wait<CTAS == 2>(&acc_empty[buf], ((it / NB) & 1) ^ 1, abort_flag, p.status, 0x43)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint64_t a_desc = smem_desc_sw128(smem_u32(sa + s * Cfg::kAStage));
            const uint32_t sb_u = smem_u32(sb + s * Cfg::kBStage);
            const uint64_t b_desc = kTrans ? smem_desc_sw128_mn(sb_u) : smem_desc_sw128(sb_u);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const uint64_t ad = a_desc + (uint64_t)(kk * 2), bd = b_desc + (uint64_t)kk * kBStep;
              if constexpr (CTAS == 2) mma_f8_ss_pair(tmem_base + buf * TN, ad, bd, idesc, kk > 0);
              else mma_f8_ss(tmem_base + buf * TN, ad, bd, idesc, kk > 0);
            }
            if constexpr (CTAS == 2) {
              tc_commit_pair(cluster_map(&acc_full[buf], 0));
              tc_commit_pair(cluster_map(&acc_full[buf], 1));
              tc_commit_pair(cluster_map(&empty[s], 0));
              tc_commit_pair(cluster_map(&empty[s], 1));
            } else {
              tc_commit(&acc_full[buf]);
              tc_commit(&empty[s]);
            }
          }
        }
        if constexpr (CTAS == 2) tc_commit_pair(cluster_map(drain, 0));
        else tc_commit(drain);
        const uint64_t t0 = globaltimer();
        while (!mbar_try_wait(smem_u32(drain), 0)) {
          if (globaltimer() - t0 > QLIN_WAIT_TIMEOUT_NS) break;
        }
      }
    }
    if (CTAS == 1 && share > 1) {  // the two cluster barriers around the join
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
  } else {
    if constexpr (CTAS == 2) setmaxnreg_inc<224>();
    // --------------------------------------------------------------------- rescale + epilogue
    constexpr int kCols = Cfg::kCols;
    constexpr int kChunk = 16;
    const int quarter = warp & 3;
    const int part = (warp - 4) >> 2;
    const int r = quarter * 32 + lane;  // TMEM lane == token within this CTA's 128
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t acc_empty_leader = CTAS == 2 ? cluster_map(acc_empty, 0) : smem_u32(acc_empty);
    uint32_t it = 0;
    bool ok = true;
    for (int t = tile0; t < num_tiles && ok; t += tile_step) {
      int mt, nt;
      fp8_tile(t, p.m_tiles, p.n_tiles, p.group, mt, nt);
      const int m = (mt * CTAS + (int)rank) * 128 + r;
      const int n0 = nt * TN + part * kCols;  // kCols channels from here, inside one 128-channel block
      const long long sw_off = (long long)min(n0 / 128, (p.N - 1) / 128) * p.sw_out;
      float acc[kCols];  // the sums start from the bias
      if (p.bias_kind != 0 && part_k == 0) {
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += 32) {
          const float mine = n0 + c0 + lane < p.N ? fp8_bias(p.bias, p.bias_kind, n0 + c0 + lane, p.N) : 0.f;
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[c0 + j] = __shfl_sync(0xffffffffu, mine, j);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kCols; ++j) acc[j] = 0.f;
      }
      // Scales come from L2, at times from HBM: a token's are asked for kAhead blocks before their use, and
      // the weight's, one for all lanes, 32 blocks at a time, a lane each.
      constexpr int kAhead = 4;
      const float* sx_next = p.sx + (long long)b_begin * p.ld_sx + min(m, p.M - 1);
      int left = b_end - b_begin - 1;  // blocks after the one sx_next points at
      auto take_sx = [&]() {
        const float v = qchk(BS_FP8_SCALE, sx_next - p.sx, p.lim_sx) ? ld_f32(sx_next) : 0.f;
        if (left > 0) sx_next += p.ld_sx;
        --left;
        return v;
      };
      auto take_sw = [&](int b) {
        const long long i = sw_off + (long long)min(b_begin + b + lane, p.kb - 1) * p.sw_red;
        return qchk(BS_FP8_SCALE, i, p.lim_sw) ? ld_f32(p.sw + i) : 0.f;
      };
      float sx[kAhead], sw = p.kb > 0 ? take_sw(0) : 0.f;  // b counts from b_begin here
      const int blocks = b_end - b_begin;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) sx[u] = p.kb > 0 ? take_sx() : 0.f;
      for (int b0 = 0; b0 < blocks && ok; b0 += kAhead) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int b = b0 + u;
          if (b >= blocks) break;
          const float s = sx[u] * __shfl_sync(0xffffffffu, sw, b & 31);
          if ((b & 31) == 31) sw = take_sw(b + 1);
          sx[u] = take_sx();
          const uint32_t buf = it % NB;
          if (!mbar_wait(&acc_full[buf], (it / NB) & 1, abort_flag, p.status, 0x44)) { ok = false; break; }
          tc_fence_after();
          const uint32_t taddr = tmem_base + lanes + buf * TN + part * kCols;
          // the next chunk's load is in flight during a chunk's arithmetic
          uint32_t v[2][kChunk];
          tmem_ld_cols<kChunk>(taddr, v[0]);
#pragma unroll
          for (int c = 0; c < kCols / kChunk; ++c) {
            tmem_wait_ld_of(v[c & 1]);
            if (c + 1 < kCols / kChunk) {
              tmem_ld_cols<kChunk>(taddr + (c + 1) * kChunk, v[(c + 1) & 1]);
            } else {  // the last values are in registers: the buffer goes back to the issuer
              tc_fence_before();
              __syncwarp();
              if (lane == 0) {
                if constexpr (CTAS == 2) mbar_arrive_cluster(acc_empty_leader + buf * 8);
                else mbar_arrive(&acc_empty[buf]);
              }
            }
#pragma unroll
            for (int j = 0; j < kChunk; j += 2)
              ffma2(s, v[c & 1][j], v[c & 1][j + 1], acc[c * kChunk + j], acc[c * kChunk + j + 1]);
          }
          ++it;
        }
      }
      if (!ok) break;
      if (CTAS == 1 && share > 1) {  // this CTA's sums, for the cluster: rows of kJoinPitch floats over the operand ring
        float* row = reinterpret_cast<float*>(sa) + r * kJoinPitch + part * kCols;
        if (qchk_smem(BS_FP8_SMEM, smem_raw, row, kCols * 4)) {
#pragma unroll
          for (int j = 0; j < kCols; j += 4)
            *reinterpret_cast<float4*>(row + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
        }
        break;
      }
      // The warp's 32 rows go through its own staging buffer, 128 bytes of each row at a time.  Where y's rows are
      // 16-byte aligned they leave as TMA stores, which the next tile's products do not wait for,
      // clipped at M and N, the 16-byte pieces swizzled by the row.  Else a row is staged at its global address
      // modulo 16, so that all but its first and last bytes leave in 16-byte stores, 8 lanes to a row.  (A bulk copy
      // for each row and piece, 1024 a tile in fp32, took longer than the tile's products.)
      const int m_warp = (mt * CTAS + (int)rank) * 128 + quarter * 32;
      uint8_t* stage = so + (warp - 4) * Cfg::kOutWarp;
      constexpr int kPieceBytes = 32 * 128;
      constexpr int kPieces = kCols == 128 ? 2 : 1;
      bool used[kPieces] = {};
      const bool wide = p.y_dtype == OUT_F32;
      if (lane == 0) bulk_wait_read<0>();  // the last tile's stores have left the buffer
      __syncwarp();
      auto piece = [&](auto wide_c, int c0) {  // 128 bytes of every row: the values from column c0
        constexpr bool kWide = decltype(wide_c)::value;
        constexpr int kN = kWide ? 32 : 64;
        const int n = n0 + c0;
        if (!p.tma_out) {
          // The row in 32-bit words, shifted in registers to its address modulo 16: word j of this piece is what
          // belongs at the row's first 16-byte boundary at or below its start, plus 4 (w0 + j).
          constexpr int kBytes = kWide ? 4 : 2;
          const int w0 = c0 * kBytes / 4;
          const bool last_piece = c0 + kN == kCols;
          const int bytes = min(kCols, p.N - n0) * kBytes;  // of the row's part that this warp has
          uint8_t* g0 = reinterpret_cast<uint8_t*>(p.y) + ((long long)m_warp * p.ldy + n0) * kBytes;
          const long long pitch = p.ldy * kBytes;
          if (bytes <= 0 || !qchk_smem(BS_FP8_SMEM, smem_raw, stage, 32 * kOddPitch)) return;
          uint8_t* g = g0 + lane * pitch;
          uint8_t* row = stage + lane * kOddPitch;
          const int off = (int)(reinterpret_cast<uintptr_t>(g) & 15);
          uint32_t r[40];  // words w0 - 4 .. w0 + 35
#pragma unroll
          for (int k = 0; k < 40; ++k) {
            const int j = w0 + k - 4;
            if (j < 0 || k >= 36 || j * 4 / kBytes >= kCols) r[k] = 0;
            else if constexpr (kWide) r[k] = __float_as_uint(acc[j]);
            else r[k] = pack_out2(p.y_dtype, acc[2 * j], acc[2 * j + 1]);
          }
          if constexpr (!kWide) {
#pragma unroll
            for (int k = 39; k > 0; --k) r[k] = (off & 2) ? __funnelshift_l(r[k - 1], r[k], 16) : r[k];
          }
#pragma unroll
          for (int k = 39; k > 1; --k) r[k] = (off & 4) ? r[k - 1] : r[k];
#pragma unroll
          for (int k = 39; k > 3; --k) r[k] = (off & 8) ? r[k - 2] : r[k];
          __syncwarp();  // the last piece has left
#pragma unroll
          for (int w = 0; w < 9; ++w)
            if (w < 8 || last_piece)
              *reinterpret_cast<uint4*>(row + w * 16) = make_uint4(r[4 * w + 4], r[4 * w + 5], r[4 * w + 6], r[4 * w + 7]);
          __syncwarp();
          const int rows = min(32, p.M - m_warp);
#pragma unroll
          for (int i = 0; i < 8; ++i) {  // 8 lanes to a row, 4 rows at a time
            const int rr = i * 4 + (lane >> 3), w = lane & 7;
            uint8_t* gr = g0 + rr * pitch;
            const int o = (int)(reinterpret_cast<uintptr_t>(gr) & 15), rel = w0 * 4 + w * 16;
            if (rr < rows && rel >= o && rel + 16 <= o + bytes &&
                qchk_span(BS_FP8_Y, (gr - o + rel - reinterpret_cast<uint8_t*>(p.y)) / kBytes, 16 / kBytes, p.lim_y))
              *reinterpret_cast<uint4*>(gr - o + rel) = *reinterpret_cast<const uint4*>(stage + rr * kOddPitch + w * 16);
          }
          if (lane < rows) {
            const int end = off + bytes, tail = end & ~15;
            if (c0 == 0 && off > 0 &&
                qchk_span(BS_FP8_Y, (g - reinterpret_cast<uint8_t*>(p.y)) / kBytes, (min(16, end) - off) / kBytes, p.lim_y))
              store_head<kBytes>(g, row + off, min(16, end) - off);
            const int in = tail - w0 * 4;  // where the row's last word lies in this piece
            if (end > tail && in >= 0 && in < (last_piece ? 144 : 128) && (tail > 0 || off == 0) &&
                qchk_span(BS_FP8_Y, (g - off + tail - reinterpret_cast<uint8_t*>(p.y)) / kBytes, (end - tail) / kBytes, p.lim_y))
              store_tail<kBytes>(g - off + tail, row + in, end - tail);
          }
          return;
        }
        const int slot = (c0 / kN) % kPieces;
        uint8_t* dst = stage + slot * kPieceBytes;
        if (used[slot]) {  // the buffer holds a part of the row
          if (lane == 0) bulk_wait_read<0>();
          __syncwarp();
        }
        used[slot] = true;
        if (qchk_smem(BS_FP8_SMEM, smem_raw, dst, kPieceBytes)) {
#pragma unroll
          for (int ch = 0; ch < 8; ++ch) {
            uint4 w;
            if constexpr (kWide) {
              w = make_uint4(__float_as_uint(acc[c0 + 4 * ch]), __float_as_uint(acc[c0 + 4 * ch + 1]),
                             __float_as_uint(acc[c0 + 4 * ch + 2]), __float_as_uint(acc[c0 + 4 * ch + 3]));
            } else {
              w = make_uint4(pack_out2(p.y_dtype, acc[c0 + 8 * ch], acc[c0 + 8 * ch + 1]),
                             pack_out2(p.y_dtype, acc[c0 + 8 * ch + 2], acc[c0 + 8 * ch + 3]),
                             pack_out2(p.y_dtype, acc[c0 + 8 * ch + 4], acc[c0 + 8 * ch + 5]),
                             pack_out2(p.y_dtype, acc[c0 + 8 * ch + 6], acc[c0 + 8 * ch + 7]));
            }
            *reinterpret_cast<uint4*>(dst + lane * 128 + ((ch ^ (lane & 7)) << 4)) = w;
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (n < p.N && m_warp < p.M) tma_store_2d(&tmap_y, dst, n, m_warp);
          bulk_commit();
        }
      };
      if (wide) {
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += 32) piece(std::true_type{}, c0);
      } else {
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += 64) piece(std::false_type{}, c0);
      }
    }
    if (lane == 0) bulk_wait_all();
    if (CTAS == 1 && share > 1) {
      // Every CTA of the cluster joins its share of the tile's tokens, in the order of the parts: four channels
      // to a thread, two tokens at a time, with all of their loads in flight.
      cluster_sync();
      const bool aborted = *abort_flag != 0;
      int mt, nt;
      fp8_tile(tile0, p.m_tiles, p.n_tiles, p.group, mt, nt);
      const int n = nt * TN + lane * 4;
      const int valid = min(128, p.M - mt * 128);
      constexpr int kWarps = Cfg::kEpiWarps;
      const uint32_t mine = smem_u32(reinterpret_cast<float*>(sa) + lane * 4);
      for (int r0 = part_k + share * (warp - 4); r0 < valid && n < p.N && !aborted; r0 += share * kWarps * 2) {
        float4 v[2][8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int r = r0 + u * share * kWarps;
#pragma unroll
          for (int c = 0; c < 8; ++c)
            if (c < share && r < valid) v[u][c] = ld_cluster_f32x4(cluster_map_addr(mine + r * (kJoinPitch * 4), c));
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int r = r0 + u * share * kWarps;
          if (r >= valid) break;
          float o[4] = {};
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            if (c >= share) break;
            o[0] += v[u][c].x;
            o[1] += v[u][c].y;
            o[2] += v[u][c].z;
            o[3] += v[u][c].w;
          }
          const long long at = (long long)(mt * 128 + r) * p.ldy + n;
          if (p.tma_out && n + 4 <= p.N && qchk_span(BS_FP8_Y, at, 4, p.lim_y)) {
            if (p.y_dtype == OUT_F32)
              *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.y) + at) = make_float4(o[0], o[1], o[2], o[3]);
            else
              *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.y) + at) =
                  make_uint2(pack_out2(p.y_dtype, o[0], o[1]), pack_out2(p.y_dtype, o[2], o[3]));
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (n + j >= p.N || !qchk(BS_FP8_Y, at + j, p.lim_y)) continue;
              if (p.y_dtype == OUT_F32) reinterpret_cast<float*>(p.y)[at + j] = o[j];
              else if (p.y_dtype == OUT_F16) reinterpret_cast<__half*>(p.y)[at + j] = __float2half_rn(o[j]);
              else reinterpret_cast<__nv_bfloat16*>(p.y)[at + j] = __float2bfloat16_rn(o[j]);
            }
          }
        }
      }
      cluster_sync();  // no CTA leaves while another reads its sums
    }
  }

  // Warps 0 and 1 ran their loops on one elected lane; reconverge before the block barrier
  // (barrier.sync is .aligned) and before the warp-wide TMEM dealloc.
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  // The even CTA's MMAs (which write the odd CTA's TMEM and read its shared memory) have all
  // completed once its issuer's drain wait returned; neither CTA frees TMEM or exits before.
  if constexpr (CTAS == 2) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CTAS == 2) tmem_dealloc_pair(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace qlin
