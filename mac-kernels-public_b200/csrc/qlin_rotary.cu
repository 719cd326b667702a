// Rotary positions with several axes, and the RMS norm of every query and key head with the position
// rotation in the same pass, forward and backward.
//
// Table: pair p of a head belongs to one axis a and turns by angle = pos[a] * theta^(-2 i / dim_a), i its
// index within the axis; the table holds (cos, sin) in fp32, [tokens][pairs][2].
//
// Head norm with rotation, for each head's row x of D values with weight w:
//   v = x * rstd * w,  rstd = (mean(x^2) + eps)^-1/2
//   (y_a, y_b) = (v_a c - v_b s, v_a s + v_b c) for each rotated pair; the values past 2 * pairs stay v
// A pair is two neighbours (interleaved) or the same place of the rotated part's two halves.
// Backward, with g the gradient rotated back and xhat = x * rstd:
//   dx = rstd * (g w - xhat * mean(g w xhat)),  dw = sum over all rows of g * xhat
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/qlin.h"
#include "qlin_internal.h"
#include "qlin_ptx.cuh"

namespace qlin {

// ---------------------------------------------------------------------------------------------
// Table
// ---------------------------------------------------------------------------------------------
constexpr int kMaxPairs = 256;

template <int CAP>
struct RotTableParams {
  const void* pos;  // [tokens, axes]
  long long tokens;
  int axes, pairs;
  float2* out;      // [tokens, pairs]
  unsigned long long turn[CAP];  // theta^(-2 i / dim) / (2 pi) of each pair, times 2^64
  unsigned char axis[CAP];
};

// A position times a frequency in turns, modulo a whole turn, times 2^64.  The product of integers wraps by
// itself; a float position is its 24-bit mantissa's product, shifted.
__device__ __forceinline__ unsigned long long turns_of(long long pos, unsigned long long turn) {
  return (unsigned long long)pos * turn;
}
__device__ __forceinline__ unsigned long long turns_of(float pos, unsigned long long turn) {
  const uint32_t bits = __float_as_uint(pos);
  const int e = max((int)((bits >> 23) & 255), 1) - 150;  // pos = +- mantissa * 2^e
  const uint32_t mant = (bits & 0x7fffff) | ((bits & 0x7f800000) ? 0x800000 : 0);
  // the 88-bit product, by the turn's halves
  const unsigned long long p0 = (unsigned long long)mant * (uint32_t)turn;
  const unsigned long long p1 = (unsigned long long)mant * (uint32_t)(turn >> 32);
  const unsigned long long lo = (p1 << 32) + p0, hi = (p1 + (p0 >> 32)) >> 32;
  unsigned long long u;
  if (e >= 0) u = e < 64 ? lo << e : 0;
  else if (e > -64) u = (lo >> -e) | (hi << (64 + e));
  else u = e > -128 ? hi >> (-64 - e) : 0;
  return (bits >> 31) ? 0 - u : u;
}

// (cos, sin) of u / 2^64 turns: the nearest quarter turn goes by exchange and sign, the rest, at most an eighth,
// by the Taylor sums to the 10th and 9th power (the first terms left out are below 2^-33 and 2^-29, a
// sixteenth of the fp32 rounding of the sine's largest values).
__device__ __forceinline__ float2 cos_sin_of(unsigned long long u) {
  const uint32_t quarter = (uint32_t)((u + (1ull << 61)) >> 62) & 3;
  const long long rest = (long long)(u - ((unsigned long long)quarter << 62));  // wraps for the last half quarter
  const float t = fmaf((float)(uint32_t)rest, 5.421010862427522e-20f,          // 2^-64
                       (float)(int)(rest >> 32) * 2.3283064365386963e-10f);    // 2^-32
  const float a = t * 6.283185307179586f, z = a * a;
  float c = fmaf(z, -1.f / 3628800.f, 1.f / 40320.f);
  c = fmaf(z, c, -1.f / 720.f);
  c = fmaf(z, c, 1.f / 24.f);
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.f);
  float s = fmaf(z, 1.f / 362880.f, -1.f / 5040.f);
  s = fmaf(z, s, 1.f / 120.f);
  s = fmaf(z, s, -1.f / 6.f);
  s = fmaf(z * a, s, a);
  const float x = quarter & 1 ? s : c, y = quarter & 1 ? c : s;
  return make_float2((quarter == 1 || quarter == 2) ? -x : x, quarter >= 2 ? -y : y);
}

// The angle is kept in turns as a 64-bit fraction until its whole turns are gone; a position multiplies the
// frequency's own error, at most 2^-57 of a turn and 2^-61 from a theta of 10^4 on.  A thread keeps its pair's
// frequency and walks over tokens, four at a time; a warp writes 256 consecutive bytes.  Bound by instructions.
// Measured at 32760 tokens of 64 pairs (16.8 MB written): 6.3 us from int64 positions, 9.4 us from fp32 ones; with the
// frequencies read through the constant cache, one lane's entry at a time, 14 us; with 8 CTAs on each SM and 64-bit
// divisions instead of walking pointers, 8.6 us.
template <int CAP, typename POS>
__global__ void __launch_bounds__(256) rotary_table_kernel(const __grid_constant__ RotTableParams<CAP> p) {
  griddep_launch();
  const int pair = blockIdx.y * 32 + threadIdx.x;
  if (pair >= p.pairs) return;
  // Read by address, as ordinary memory: the constant cache serves one lane's entry at a time.
  const RotTableParams<CAP>* params = &p;
  asm volatile("" : "+l"(params));
  const unsigned long long turn = params->turn[pair];
  const int axis = params->axis[pair];
  const POS* pos = reinterpret_cast<const POS*>(p.pos);
  constexpr int kTokens = 4;
  griddep_wait();
  const long long step = (long long)gridDim.x * 8, first = (long long)blockIdx.x * 8 + threadIdx.y;
  const POS* from = pos + first * p.axes + axis;
  float2* to = p.out + first * p.pairs + pair;
  const long long from_step = step * p.axes, to_step = step * p.pairs;
  for (long long left = p.tokens - first; left > 0; left -= kTokens * step) {
    POS x[kTokens];
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      x[u] = (u * step < left && qchk(BS_ROT_IN, from - pos, p.tokens * p.axes)) ? *from : POS(0);
      from += from_step;
    }
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      float2 v;
      if constexpr (std::is_same<POS, float>::value) {
        v = cos_sin_of(turns_of(x[u], turn));
        if ((__float_as_uint(x[u]) & 0x7f800000) == 0x7f800000) v = make_float2(nanf(""), nanf(""));
      } else {
        v = cos_sin_of(turns_of((long long)x[u], turn));
      }
      if (u * step < left && qchk(BS_ROT_OUT, to - p.out, p.tokens * p.pairs)) *to = v;
      to += to_step;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Head norm with rotation
// ---------------------------------------------------------------------------------------------
struct HeadParams;
__device__ __forceinline__ void put_dw(const HeadParams& p, int which, int cta, int i, float sum);

// One of q and k: [B, L, heads, D] with element strides, values of a row side by side.
struct HeadSide {
  const void* x;
  const void* dy;      // backward: the output's gradient
  void* y;             // forward: the output; backward: dx
  const void* w;       // [D] or null
  float* dw;           // backward: partial sums [ctas][D]
  void* dw_out;        // backward: the gradient itself, where one CTA has all of the side's rows
  int heads, chunks;   // chunks: warps that share a token's heads
  long long x_b, x_l, x_h, y_b, y_l, y_h, dy_b, dy_l, dy_h;
  long long lim_x, lim_y, lim_dy;  // element counts for the QLIN_CHECKS build
};

struct HeadParams {
  HeadSide side[2];    // q, k
  const float2* table;
  long long table_b;   // float2 between batches (0: shared)
  long long tokens;    // B * L
  int L, D, pairs;     // pairs: rotated pairs of a head
  int interleaved;
  float eps;
  int w_dtype;
  int heads_per_warp;
  int ctas[2];         // backward: CTAs of each side
  long long lim_table;
};

template <int DT>
__device__ __forceinline__ float head_load(const void* x, long long i) {
  if constexpr (DT == QLIN_F16) return __half2float(reinterpret_cast<const __half*>(x)[i]);
  else if constexpr (DT == QLIN_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(x)[i]);
  else return reinterpret_cast<const float*>(x)[i];
}
template <int DT>
__device__ __forceinline__ void head_store(void* x, long long i, float v) {
  if constexpr (DT == QLIN_F16) reinterpret_cast<__half*>(x)[i] = __float2half_rn(v);
  else if constexpr (DT == QLIN_BF16) reinterpret_cast<__nv_bfloat16*>(x)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<float*>(x)[i] = v;
}
__device__ __forceinline__ float weight_at(const void* w, int dt, int i, int D) {
  if (w == nullptr || !qchk(BS_ROT_IN, i, D)) return 1.f;
  if (dt == QLIN_F16) return __half2float(reinterpret_cast<const __half*>(w)[i]);
  if (dt == QLIN_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[i]);
  return reinterpret_cast<const float*>(w)[i];
}

// A lane's 8 values of a row: two pieces of 4, at o0 and o1.  Interleaved (and past the rotated part) the
// pieces are neighbours and hold pairs (0,1) (2,3) | (4,5) (6,7); with halves, pair i is value i of each piece.
template <int DT>
struct Pieces {
  uint2 v[DT == QLIN_F32 ? 4 : 2];
};

template <int DT, bool kInter>
__device__ __forceinline__ Pieces<DT> load_pieces(const void* x, long long row, int o0, int o1) {
  Pieces<DT> r;
  if constexpr (DT == QLIN_F32) {
    const uint4 a = *reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(x) + row + o0);
    const uint4 b = *reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(x) + row + o1);
    r.v[0] = make_uint2(a.x, a.y);
    r.v[1] = make_uint2(a.z, a.w);
    r.v[2] = make_uint2(b.x, b.y);
    r.v[3] = make_uint2(b.z, b.w);
  } else if constexpr (kInter) {
    const uint4 a = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(x) + row + o0);
    r.v[0] = make_uint2(a.x, a.y);
    r.v[1] = make_uint2(a.z, a.w);
  } else {
    r.v[0] = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(x) + row + o0);
    r.v[1] = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(x) + row + o1);
  }
  return r;
}

template <int DT>
__device__ __forceinline__ void pieces_to_float(const Pieces<DT>& r, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < (DT == QLIN_F32 ? 4 : 2); ++i) {
    const uint32_t w[2] = {r.v[i].x, r.v[i].y};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if constexpr (DT == QLIN_F32) {
        f[2 * i + j] = __uint_as_float(w[j]);
      } else if constexpr (DT == QLIN_F16) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        f[4 * i + 2 * j] = t.x;
        f[4 * i + 2 * j + 1] = t.y;
      } else {
        f[4 * i + 2 * j] = __uint_as_float(w[j] << 16);
        f[4 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    }
  }
}

template <int DT, bool kInter>
__device__ __forceinline__ void store_pieces(void* y, long long row, int o0, int o1, const float (&f)[8]) {
  if constexpr (DT == QLIN_F32) {
    float* p = reinterpret_cast<float*>(y) + row;
    *reinterpret_cast<float4*>(p + o0) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + o1) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == QLIN_F16) {
        const __half2 h = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    uint16_t* p = reinterpret_cast<uint16_t*>(y) + row;
    if constexpr (kInter) {
      *reinterpret_cast<uint4*>(p + o0) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      *reinterpret_cast<uint2*>(p + o0) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(p + o1) = make_uint2(w[2], w[3]);
    }
  }
}

// Rotates the lane's 4 pairs in place by (c, s); kBack by (c, -s).
template <bool kInter, bool kBack>
__device__ __forceinline__ void rotate4(float (&f)[8], const float (&c)[4], const float (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int a = kInter ? 2 * i : i, b = kInter ? 2 * i + 1 : i + 4;
    const float sn = kBack ? -s[i] : s[i];
    const float t = f[a] * c[i] - f[b] * sn;
    f[b] = f[a] * sn + f[b] * c[i];
    f[a] = t;
  }
}

// What a lane does in every row: where its values lie, and its pairs' place in the table (-1: not rotated).
template <int G>
struct LanePlan {
  int o0, o1, pair0;
  bool on;
  __device__ __forceinline__ LanePlan(int lane, int D, int pairs, bool inter) {
    const int j = lane & (G - 1);
    on = j * 8 < D;
    o0 = j * 8;
    o1 = o0 + 4;
    pair0 = -1;
    if (j * 4 < pairs) {
      pair0 = j * 4;
      if (!inter) {
        o0 = j * 4;
        o1 = o0 + pairs;
      }
    }
  }
};

__device__ __forceinline__ void load_turn(const HeadParams& p, long long token_row, int pair0, float (&c)[4],
                                          float (&s)[4]) {
  if (pair0 >= 0 && qchk_span(BS_ROT_IN, token_row + pair0, 4, p.lim_table)) {
    const float4 a = reinterpret_cast<const float4*>(p.table + token_row + pair0)[0];
    const float4 b = reinterpret_cast<const float4*>(p.table + token_row + pair0)[1];
    c[0] = a.x; s[0] = a.y; c[1] = a.z; s[1] = a.w;
    c[2] = b.x; s[2] = b.y; c[3] = b.z; s[3] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = 1.f;
      s[i] = 0.f;
    }
  }
}

// The lane's 8 values of the weight; its two pieces start on multiples of 4 values (the vector kernels take
// weights whose address is a multiple of 4 values too).
template <class Plan>
__device__ __forceinline__ void load_weight(const void* w, int dt, const Plan& plan, int D, float (&f)[8]) {
  if (w == nullptr || !plan.on || !qchk_span(BS_ROT_IN, plan.o0, 4, D) || !qchk_span(BS_ROT_IN, plan.o1, 4, D)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = plan.on ? 1.f : 0.f;
  } else if (dt == QLIN_F32) {
    pieces_to_float<QLIN_F32>(load_pieces<QLIN_F32, false>(w, 0, plan.o0, plan.o1), f);
  } else if (dt == QLIN_F16) {
    pieces_to_float<QLIN_F16>(load_pieces<QLIN_F16, false>(w, 0, plan.o0, plan.o1), f);
  } else {
    pieces_to_float<QLIN_BF16>(load_pieces<QLIN_BF16, false>(w, 0, plan.o0, plan.o1), f);
  }
}

// Column i of a CTA's sum of g * xhat: to its partial row, or rounded once to the gradient.
__device__ __forceinline__ void put_dw(const HeadParams& p, int which, int cta, int i, float sum) {
  const HeadSide& sd = p.side[which];
  if (sd.dw_out != nullptr) {
    if (!qchk(BS_ROT_OUT, i, p.D)) return;
    if (p.w_dtype == QLIN_F16) head_store<QLIN_F16>(sd.dw_out, i, sum);
    else if (p.w_dtype == QLIN_BF16) head_store<QLIN_BF16>(sd.dw_out, i, sum);
    else head_store<QLIN_F32>(sd.dw_out, i, sum);
    return;
  }
  const long long at = (long long)cta * p.D + i;
  if (qchk(BS_ROT_OUT, at, (long long)p.ctas[which] * p.D)) sd.dw[at] = sum;
}

// Batch and position of a token.
__device__ __forceinline__ void token_of(const HeadParams& p, long long token, long long& b, long long& l) {
  if (p.tokens <= 0x7fffffff) {
    const uint32_t q = (uint32_t)token / (uint32_t)p.L;
    b = q;
    l = (uint32_t)token - q * (uint32_t)p.L;
  } else {
    b = token / p.L;
    l = token - b * p.L;
  }
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Forward.  A row is G lanes of 8 values; a warp takes a share of a token's q or k heads (all of them where
// there are tokens enough), 32 / G rows at a time with kUnroll loads in flight, and keeps the token's cosines
// and sines and the weight in registers.  blockIdx.y is the share.  Bound by HBM: 32760 tokens of 80 heads of 128
// in bf16 take 209 us (6.5 TB/s) with 32 warps on an SM; walking over tokens with fewer CTAs took 217 to 250, more
// loads ahead at 24 or 16 warps 223 to 250.
template <int DT, int G, bool kInter>
__global__ void __launch_bounds__(256, 4) qk_norm_rotary_kernel(const __grid_constant__ HeadParams p) {
  constexpr int R = 32 / G;
  constexpr int kUnroll = DT == QLIN_F32 ? 2 : 4;
  griddep_launch();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  int chunk = blockIdx.y;
  const int which = chunk >= p.side[0].chunks ? 1 : 0;
  if (which) chunk -= p.side[0].chunks;
  const HeadSide& sd = p.side[which];
  const LanePlan<G> plan(lane, p.D, p.pairs, kInter);
  const float inv_d = 1.f / (float)p.D;
  const int h_begin = chunk * p.heads_per_warp, h_end = min(sd.heads, h_begin + p.heads_per_warp);
  const long long token = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (token >= p.tokens) return;
  long long b, l;
  token_of(p, token, b, l);
  float c[4], s[4], w[8];
  load_turn(p, b * p.table_b + l * p.pairs, plan.pair0, c, s);
  load_weight(sd.w, p.w_dtype, plan, p.D, w);
  const long long xr = b * sd.x_b + l * sd.x_l, yr = b * sd.y_b + l * sd.y_l;
  for (int h0 = h_begin; h0 < h_end; h0 += R * kUnroll) {
    Pieces<DT> raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int h = h0 + u * R + lane / G;
      raw[u] = Pieces<DT>{};
      const long long row = xr + (long long)h * sd.x_h;
      if (h < h_end && plan.on && qchk_span(BS_ROT_IN, row + plan.o0, 4, sd.lim_x) &&
          qchk_span(BS_ROT_IN, row + plan.o1, 4, sd.lim_x))
        raw[u] = load_pieces<DT, kInter>(sd.x, row, plan.o0, plan.o1);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (h0 + u * R >= h_end) break;
      const int h = h0 + u * R + lane / G;
      float f[8], ss = 0.f;
      pieces_to_float<DT>(raw[u], f);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(f[j], f[j], ss);
      const float rstd = rsqrtf(group_sum<G>(ss) * inv_d + p.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = f[j] * rstd * w[j];
      rotate4<kInter, false>(f, c, s);
      const long long row = yr + (long long)h * sd.y_h;
      if (h < h_end && plan.on && qchk_span(BS_ROT_OUT, row + plan.o0, 4, sd.lim_y) &&
          qchk_span(BS_ROT_OUT, row + plan.o1, 4, sd.lim_y))
        store_pieces<DT, kInter>(sd.y, row, plan.o0, plan.o1, f);
    }
  }
}

// Backward.  The CTAs of a side walk over its (token, share of heads) items; every lane sums its 8 columns'
// g * xhat in fp32, the CTA joins its rows in a fixed order and leaves one partial row of dw, and the
// kernel below adds those up, also in a fixed order.  The next rows' loads (of the same token or the warp's next) are
// in flight during these rows' arithmetic.  Measured at 9216 tokens of 96 heads of 128 in bf16: 110 us (6.0 TB/s)
// with three rows ahead and two CTAs on an SM; without loads ahead 129 to 154, with more CTAs and fewer registers
// 145 to 169 (spills).
__host__ __device__ constexpr int bwd_unroll(int dtype) { return dtype == QLIN_F32 ? 2 : 3; }
constexpr int kBwdCtas = 2;  // resident on an SM: 128 registers a thread
template <int DT, int G, bool kInter>
__global__ void __launch_bounds__(256, kBwdCtas) qk_norm_rotary_bwd_kernel(const __grid_constant__ HeadParams p) {
  constexpr int R = 32 / G;
  constexpr int kUnroll = bwd_unroll(DT);
  __shared__ float part[8 * R][G * 8];
  griddep_launch();
  griddep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int which = blockIdx.x >= (unsigned)p.ctas[0] ? 1 : 0;
  const int cta = which ? blockIdx.x - p.ctas[0] : blockIdx.x;
  const HeadSide& sd = p.side[which];
  const LanePlan<G> plan(lane, p.D, p.pairs, kInter);
  float w[8], dw[8];
  load_weight(sd.w, p.w_dtype, plan, p.D, w);
#pragma unroll
  for (int j = 0; j < 8; ++j) dw[j] = 0.f;
  const float inv_d = 1.f / (float)p.D;
  const long long items = p.tokens * sd.chunks, stride = (long long)p.ctas[which] * 8;
  long long item = (long long)cta * 8 + warp;
  // The rows that are loaded ahead: of the same token, or the first ones of the warp's next.
  long long xr = 0, yr = 0, gr = 0;
  int h0 = 0, h_end = 0;
  float c_next[4], s_next[4];
  Pieces<DT> rx[kUnroll], rg[kUnroll];
  auto begin_item = [&]() {
    const long long token = sd.chunks == 1 ? item : item / sd.chunks;
    const int chunk = (int)(item - token * sd.chunks);
    long long b, l;
    token_of(p, token, b, l);
    load_turn(p, b * p.table_b + l * p.pairs, plan.pair0, c_next, s_next);
    xr = b * sd.x_b + l * sd.x_l;
    yr = b * sd.y_b + l * sd.y_l;
    gr = b * sd.dy_b + l * sd.dy_l;
    h0 = chunk * p.heads_per_warp;
    h_end = min(sd.heads, h0 + p.heads_per_warp);
  };
  auto load = [&]() {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int h = h0 + u * R + lane / G;
      rx[u] = Pieces<DT>{};
      rg[u] = Pieces<DT>{};
      const long long row = xr + (long long)h * sd.x_h, grow = gr + (long long)h * sd.dy_h;
      if (h < h_end && plan.on && qchk_span(BS_ROT_IN, row + plan.o0, 4, sd.lim_x) &&
          qchk_span(BS_ROT_IN, row + plan.o1, 4, sd.lim_x) && qchk_span(BS_ROT_IN, grow + plan.o0, 4, sd.lim_dy) &&
          qchk_span(BS_ROT_IN, grow + plan.o1, 4, sd.lim_dy)) {
        rx[u] = load_pieces<DT, kInter>(sd.x, row, plan.o0, plan.o1);
        rg[u] = load_pieces<DT, kInter>(sd.dy, grow, plan.o0, plan.o1);
      }
    }
  };
  if (item < items) {
    begin_item();
    load();
  }
  while (item < items) {
    Pieces<DT> cx[kUnroll], cg[kUnroll];
    float c[4], s[4];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      cx[u] = rx[u];
      cg[u] = rg[u];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = c_next[i];
      s[i] = s_next[i];
    }
    const long long to = yr;
    const int h_now = h0, h_stop = h_end;
    h0 += R * kUnroll;
    if (h0 >= h_end) {
      item += stride;
      if (item < items) begin_item();
    }
    if (item < items) load();
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (h_now + u * R >= h_stop) break;
      const int h = h_now + u * R + lane / G;
      float x[8], g[8], ss = 0.f, dot = 0.f;
      pieces_to_float<DT>(cx[u], x);
      pieces_to_float<DT>(cg[u], g);
      rotate4<kInter, true>(g, c, s);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ss = fmaf(x[j], x[j], ss);
        dot = fmaf(g[j] * w[j], x[j], dot);
      }
      ss = group_sum<G>(ss);
      dot = group_sum<G>(dot);
      const float rstd = rsqrtf(ss * inv_d + p.eps);
      const float pull = rstd * rstd * (dot * inv_d);
      if (h < h_stop) {
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          dw[j] = fmaf(g[j], x[j] * rstd, dw[j]);
          o[j] = rstd * (g[j] * w[j] - x[j] * pull);
        }
        const long long row = to + (long long)h * sd.y_h;
        if (plan.on && qchk_span(BS_ROT_OUT, row + plan.o0, 4, sd.lim_y) &&
            qchk_span(BS_ROT_OUT, row + plan.o1, 4, sd.lim_y))
          store_pieces<DT, kInter>(sd.y, row, plan.o0, plan.o1, o);
      }
    }
  }
  if (sd.dw == nullptr && sd.dw_out == nullptr) return;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (plan.on) part[warp * R + lane / G][(j < 4 ? plan.o0 : plan.o1 - 4) + j] = dw[j];
  __syncthreads();
  for (int i = threadIdx.x; i < p.D; i += 256) {
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 8 * R; ++r) sum += part[r][i];
    put_dw(p, which, cta, i, sum);
  }
}

struct DwParams {
  const float* part[2];
  int ctas[2];
  void* out[2];
  int D, w_dtype;
};

// dw = the sum of the partial rows: 32 columns to a CTA, 32 rows at a time, one rounding to the weight's type.
__global__ void __launch_bounds__(1024) dw_sum_kernel(const DwParams p) {
  __shared__ float part[32][33];
  griddep_launch();
  griddep_wait();
  const int which = blockIdx.y;
  const int i = blockIdx.x * 32 + threadIdx.x;
  if (p.out[which] == nullptr) return;
  float sum = 0.f;
  if (i < p.D)
    for (int r = threadIdx.y; r < p.ctas[which]; r += 32)
      if (qchk(BS_ROT_IN, (long long)r * p.D + i, (long long)p.ctas[which] * p.D))
        sum += p.part[which][(long long)r * p.D + i];
  part[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  float v = part[threadIdx.x][threadIdx.y];  // warp y: the 32 partial sums of column y
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int col = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && col < p.D && qchk(BS_ROT_OUT, col, p.D)) {
    if (p.w_dtype == QLIN_F16) head_store<QLIN_F16>(p.out[which], col, v);
    else if (p.w_dtype == QLIN_BF16) head_store<QLIN_BF16>(p.out[which], col, v);
    else head_store<QLIN_F32>(p.out[which], col, v);
  }
}

// Any head size and alignment: one warp to a row, values one by one, the row read twice (the second time
// from the cache).  kBack: the gradients; dw goes to one partial row per CTA as above, summed by each CTA over
// its own rows in shared memory (D <= 1024), every column always by the same thread's warp in row order.
// Bound by instructions and by loads of one value a lane: 4608 tokens of 48 heads of 100 in bf16 take 157 us forward
// (0.6 TB/s) and 405 us backward (0.3 TB/s).
template <int DT, bool kBack>
__global__ void __launch_bounds__(256) qk_norm_rotary_any_kernel(const __grid_constant__ HeadParams p) {
  extern __shared__ float warp_dw[];  // backward: [8][D]
  griddep_launch();
  griddep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int which = blockIdx.x >= (unsigned)p.ctas[0] ? 1 : 0;
  const int cta = which ? blockIdx.x - p.ctas[0] : blockIdx.x;
  const HeadSide& sd = p.side[which];
  if constexpr (kBack)
    for (int i = lane; i < p.D; i += 32) warp_dw[warp * p.D + i] = 0.f;
  __syncwarp();
  const float inv_d = 1.f / (float)p.D;
  const long long rows = p.tokens * sd.heads;
  const int rot = 2 * p.pairs;
  for (long long row = (long long)cta * 8 + warp; row < rows; row += (long long)p.ctas[which] * 8) {
    const long long token = row / sd.heads, h = row - token * sd.heads;
    const long long b = token / p.L, l = token - b * p.L;
    const long long xr = b * sd.x_b + l * sd.x_l + h * sd.x_h, yr = b * sd.y_b + l * sd.y_l + h * sd.y_h;
    const long long gr = b * sd.dy_b + l * sd.dy_l + h * sd.dy_h;
    const long long tr = b * p.table_b + l * p.pairs;
    auto x_at = [&](int i) { return qchk(BS_ROT_IN, xr + i, sd.lim_x) ? head_load<DT>(sd.x, xr + i) : 0.f; };
    auto dy_at = [&](int i) { return qchk(BS_ROT_IN, gr + i, sd.lim_dy) ? head_load<DT>(sd.dy, gr + i) : 0.f; };
    auto put = [&](int i, float v) {
      if (qchk(BS_ROT_OUT, yr + i, sd.lim_y)) head_store<DT>(sd.y, yr + i, v);
    };
    // item i < pairs: a rotated pair; past that: one plain value
    const int items = p.pairs + (p.D - rot);
    auto place = [&](int i, int& a, int& bb) {
      if (i >= p.pairs) a = bb = rot + (i - p.pairs);
      else if (p.interleaved) { a = 2 * i; bb = a + 1; }
      else { a = i; bb = i + p.pairs; }
    };
    auto grads = [&](int i, int a, int bb, float& ga, float& gb) {  // the gradient, rotated back
      ga = dy_at(a);
      gb = a == bb ? 0.f : dy_at(bb);
      if (i < p.pairs && qchk(BS_ROT_IN, tr + i, p.lim_table)) {
        const float2 t = p.table[tr + i];
        const float v = ga * t.x + gb * t.y;
        gb = gb * t.x - ga * t.y;
        ga = v;
      }
    };
    float ss = 0.f, dot = 0.f;
    for (int i = lane; i < items; i += 32) {
      int a, bb;
      place(i, a, bb);
      const float xa = x_at(a), xb = a == bb ? 0.f : x_at(bb);
      ss += xa * xa + xb * xb;
      if constexpr (kBack) {
        float ga, gb;
        grads(i, a, bb, ga, gb);
        dot += ga * weight_at(sd.w, p.w_dtype, a, p.D) * xa + gb * weight_at(sd.w, p.w_dtype, bb, p.D) * xb;
      }
    }
    const float rstd = rsqrtf(group_sum<32>(ss) * inv_d + p.eps);
    if constexpr (kBack) dot = group_sum<32>(dot);
    for (int i = lane; i < items; i += 32) {
      int a, bb;
      place(i, a, bb);
      const float xa = x_at(a), xb = a == bb ? 0.f : x_at(bb);
      const float wa = weight_at(sd.w, p.w_dtype, a, p.D), wb = weight_at(sd.w, p.w_dtype, bb, p.D);
      if constexpr (kBack) {
        float ga, gb;
        grads(i, a, bb, ga, gb);
        const float pull = rstd * rstd * (dot * inv_d);
        warp_dw[warp * p.D + a] += ga * (xa * rstd);
        if (a != bb) warp_dw[warp * p.D + bb] += gb * (xb * rstd);
        put(a, rstd * (ga * wa - xa * pull));
        if (a != bb) put(bb, rstd * (gb * wb - xb * pull));
      } else {
        const float va = xa * rstd * wa, vb = xb * rstd * wb;
        float2 t = make_float2(1.f, 0.f);
        if (i < p.pairs && qchk(BS_ROT_IN, tr + i, p.lim_table)) t = p.table[tr + i];
        put(a, va * t.x - vb * t.y);
        if (a != bb) put(bb, va * t.y + vb * t.x);
      }
    }
  }
  if constexpr (kBack) {
    if (sd.dw == nullptr && sd.dw_out == nullptr) return;
    __syncthreads();
    for (int i = threadIdx.x; i < p.D; i += 256) {
      float sum = 0.f;
      for (int r = 0; r < 8; ++r) sum += warp_dw[r * p.D + i];
      put_dw(p, which, cta, i, sum);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------
static int rot_launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return QLIN_OK;
  set_error("%s: %s", what, cudaGetErrorString(e));
  return QLIN_ECUDA;
}

template <int CAP>
static void launch_table(const void* positions, int pos_dtype, long long tokens, int axes, const int32_t* axes_dim,
                         int pairs, double theta, float* table, cudaStream_t s) {
  RotTableParams<CAP> p;
  p.pos = positions;
  p.tokens = tokens;
  p.axes = axes;
  p.pairs = pairs;
  p.out = reinterpret_cast<float2*>(table);
  int at = 0;
  for (int a = 0; a < axes; ++a) {
    // the axis' frequencies by repeated products of 64 significant bits: after 255 of them 2^-54 of the value
    long double f = 0.159154943091895335768883763372514362L * 18446744073709551616.0L;  // 2^64 / (2 pi)
    const long double step = axes_dim[a] > 0 ? powl((long double)theta, -2.0L / axes_dim[a]) : 1.0L;
    for (int i = 0; i < axes_dim[a] / 2; ++i, ++at, f *= step) {
      p.turn[at] = (unsigned long long)(f + 0.5L);
      p.axis[at] = (unsigned char)a;
    }
  }
  const dim3 block(32, 8), grid((unsigned)std::min<long long>((tokens + 7) / 8, 2ll * sm_count()), (pairs + 31) / 32);
  if (pos_dtype == QLIN_F32) launch_dependent(rotary_table_kernel<CAP, float>, grid, block, 0, s, 0, p);
  else if (pos_dtype == QLIN_I32) launch_dependent(rotary_table_kernel<CAP, int>, grid, block, 0, s, 0, p);
  else launch_dependent(rotary_table_kernel<CAP, long long>, grid, block, 0, s, 0, p);
}

constexpr int kMaxHeadDim = 1024;
// Rows a backward CTA should have at least: each of its partial rows costs D values of traffic again.
constexpr int kBwdRowsPerCta = 32;

// The vector kernels take heads of whole 8-value pieces up to 256, rotated parts of whole pieces, and rows
// that start on the pieces' alignment.
static bool head_rows_aligned(const void* p, long long sb, long long sl, long long sh, int dtype, bool inter) {
  const int esz = dtype == QLIN_F32 ? 4 : 2;
  const uintptr_t al = dtype == QLIN_F32 || inter ? 16 : 8;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(sb * esz) | (uintptr_t)(sl * esz) |
                         (uintptr_t)(sh * esz);
  return bits % al == 0;
}

static int lanes_per_row(int D) {
  int g = 4;
  while (g * 8 < D) g *= 2;
  return g;
}

// Backward: the CTAs of both sides together, each with a partial row of dw: as many as are resident at once, or
// fewer where there are fewer rows.
static long long bwd_ctas(long long rows) {
  return std::max<long long>(2, std::min<long long>((long long)kBwdCtas * sm_count(), rows / kBwdRowsPerCta));
}
// The sides' shares go by their steps (rows_per_step rows of one token each), not by their rows: two heads take a
// warp as long as six.
static void split_bwd(long long rows, int hq, int hk, int rows_per_step, int (&ctas)[2]) {
  const long long want = bwd_ctas(rows);
  const long long steps[2] = {(hq + rows_per_step - 1) / rows_per_step, (hk + rows_per_step - 1) / rows_per_step};
  for (int i = 0; i < 2; ++i)
    ctas[i] = steps[i] == 0 ? 0 : (int)std::max<long long>(1, want * steps[i] / (steps[0] + steps[1]));
}

template <int DT, bool kInter>
static void launch_rows(const HeadParams& p, int g, bool back, dim3 grid, cudaStream_t s) {
  switch (g) {
#define QLIN_ROWS(G)                                                                    \
  case G:                                                                               \
    if (back) launch_dependent(qk_norm_rotary_bwd_kernel<DT, G, kInter>, grid, dim3(256), 0, s, 0, p); \
    else launch_dependent(qk_norm_rotary_kernel<DT, G, kInter>, grid, dim3(256), 0, s, 0, p);          \
    break;
    QLIN_ROWS(4)
    QLIN_ROWS(8)
    QLIN_ROWS(16)
    QLIN_ROWS(32)
#undef QLIN_ROWS
  }
}

template <int DT>
static void launch_dtype(const HeadParams& p, bool vec, bool back, dim3 grid, cudaStream_t s) {
  if (!vec) {
    if (back) launch_dependent(qk_norm_rotary_any_kernel<DT, true>, grid, dim3(256), (size_t)8 * p.D * 4, s, 0, p);
    else launch_dependent(qk_norm_rotary_any_kernel<DT, false>, grid, dim3(256), 0, s, 0, p);
  } else if (p.interleaved) {
    launch_rows<DT, true>(p, lanes_per_row(p.D), back, grid, s);
  } else {
    launch_rows<DT, false>(p, lanes_per_row(p.D), back, grid, s);
  }
}

static long long reach(long long n0, long long s0, long long n1, long long s1, long long n2, long long s2, long long d) {
  return (n0 - 1) * s0 + (n1 - 1) * s1 + (n2 - 1) * s2 + d;
}

// split_bwd gives each side at least one CTA: at most one more than bwd_ctas in all.
static size_t bwd_workspace(long long tokens, int hq, int hk, int D) {
  return (size_t)(bwd_ctas(tokens * (hq + hk)) + 1) * D * 4;
}

struct HeadCall {
  const char* what;
  bool back;
  const void *q, *k, *dq, *dk;
  void *oq, *ok;
  const int64_t *q_strides, *k_strides, *dq_strides, *dk_strides, *oq_strides, *ok_strides;
  void *dqw, *dkw;
};

static int head_norm(const HeadCall& a, int dtype, int64_t batch, int64_t tokens, int hq, int hk, int dim, const void* qw,
                     const void* kw, int w_dtype, const float* table, int64_t table_batch_stride, int pairs,
                     float eps, int interleaved, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (batch < 0 || tokens < 0 || hq < 0 || hk < 0 || dim <= 0 || pairs < 0 || 2 * pairs > dim ||
      tokens > 0x7fffffff || (table_batch_stride != 0 && table_batch_stride < tokens * pairs * 2)) {
    set_error("%s: bad sizes batch=%lld tokens=%lld heads=%d,%d dim=%d pairs=%d", a.what, (long long)batch,
              (long long)tokens, hq, hk, dim, pairs);
    return QLIN_EINVAL;
  }
  const bool floats = (dtype == QLIN_F32 || dtype == QLIN_F16 || dtype == QLIN_BF16) &&
                      (w_dtype == QLIN_F32 || w_dtype == QLIN_F16 || w_dtype == QLIN_BF16);
  if (!floats || dim > kMaxHeadDim || table_batch_stride % 2 != 0 || (reinterpret_cast<uintptr_t>(table) & 7)) {
    set_error("%s: heads of up to %d values in f32, f16 or bf16, an 8-byte aligned table", a.what, kMaxHeadDim);
    return QLIN_EDECLINE;
  }
  const int64_t rows = batch * tokens;
  if (rows == 0 || hq + hk == 0) {
    const int wsz = w_dtype == QLIN_F32 ? 4 : 2;  // no rows: the weights' gradients are zeros
    if (a.dqw != nullptr && cudaMemsetAsync(a.dqw, 0, (size_t)dim * wsz, stream) != cudaSuccess) return rot_launched(a.what);
    if (a.dkw != nullptr && cudaMemsetAsync(a.dkw, 0, (size_t)dim * wsz, stream) != cudaSuccess) return rot_launched(a.what);
    return QLIN_OK;
  }
  if ((hq > 0 && (a.q == nullptr || a.oq == nullptr || (a.back && a.dq == nullptr))) ||
      (hk > 0 && (a.k == nullptr || a.ok == nullptr || (a.back && a.dk == nullptr))) || (pairs > 0 && table == nullptr)) {
    set_error("%s: null pointer", a.what);
    return QLIN_EINVAL;
  }
  HeadParams p{};
  p.table = reinterpret_cast<const float2*>(table);
  p.table_b = table_batch_stride / 2;
  p.tokens = rows;
  p.L = (int)tokens;
  p.D = dim;
  p.pairs = pairs;
  p.interleaved = interleaved ? 1 : 0;
  p.eps = eps;
  p.w_dtype = w_dtype;
  p.lim_table = (batch - 1) * p.table_b + tokens * pairs;
  const void* xs[2] = {a.q, a.k};
  const void* gs[2] = {a.dq, a.dk};
  void* os[2] = {a.oq, a.ok};
  const void* ws[2] = {qw, kw};
  const int64_t* xst[2] = {a.q_strides, a.k_strides};
  const int64_t* gst[2] = {a.dq_strides, a.dk_strides};
  const int64_t* ost[2] = {a.oq_strides, a.ok_strides};
  const int heads[2] = {hq, hk};
  const bool inter = interleaved != 0;
  bool vec = dim % 8 == 0 && dim <= 256 && pairs % 4 == 0 && (reinterpret_cast<uintptr_t>(table) & 15) == 0 &&
             table_batch_stride % 4 == 0;
  for (int i = 0; i < 2; ++i) {
    HeadSide& sd = p.side[i];
    sd.heads = heads[i];
    if (heads[i] == 0) continue;
    sd.x = xs[i];
    sd.dy = gs[i];
    sd.y = os[i];
    sd.w = ws[i];
    vec = vec && reinterpret_cast<uintptr_t>(sd.w) % (w_dtype == QLIN_F32 ? 16 : 8) == 0;
    sd.x_b = xst[i][0]; sd.x_l = xst[i][1]; sd.x_h = xst[i][2];
    sd.y_b = ost[i][0]; sd.y_l = ost[i][1]; sd.y_h = ost[i][2];
    sd.lim_x = reach(batch, sd.x_b, tokens, sd.x_l, heads[i], sd.x_h, dim);
    sd.lim_y = reach(batch, sd.y_b, tokens, sd.y_l, heads[i], sd.y_h, dim);
    vec = vec && head_rows_aligned(sd.x, sd.x_b, sd.x_l, sd.x_h, dtype, inter) &&
          head_rows_aligned(sd.y, sd.y_b, sd.y_l, sd.y_h, dtype, inter);
    if (a.back) {
      sd.dy_b = gst[i][0]; sd.dy_l = gst[i][1]; sd.dy_h = gst[i][2];
      sd.lim_dy = reach(batch, sd.dy_b, tokens, sd.dy_l, heads[i], sd.dy_h, dim);
      vec = vec && head_rows_aligned(sd.dy, sd.dy_b, sd.dy_l, sd.dy_h, dtype, inter);
    }
  }
  // A warp's share of a token's heads: all of q or of k where there are tokens enough to fill the machine
  // (about 32 warps on each SM), else as few as one set of unrolled rows.
  const int step = std::max(1, 32 / lanes_per_row(dim)) * (a.back ? bwd_unroll(dtype) : 2);
  int per_warp = std::max(hq, hk);
  const long long warps = 32ll * sm_count();
  const int fewest = (std::max(hq, hk) + 16383) / 16384;  // the shares are a grid dimension
  while (per_warp > step && per_warp > 2 * fewest && rows * ((hq + per_warp - 1) / per_warp + (hk + per_warp - 1) / per_warp) < warps)
    per_warp = std::max(step, (per_warp + 1) / 2);
  p.heads_per_warp = per_warp;
  for (int i = 0; i < 2; ++i) p.side[i].chunks = (heads[i] + per_warp - 1) / per_warp;
  dim3 grid(1);
  if (a.back) {
    const size_t need = bwd_workspace(rows, hq, hk, dim);
    if (workspace == nullptr || workspace_bytes < need) {
      set_error("%s: workspace too small: need %zu bytes", a.what, need);
      return QLIN_EINVAL;
    }
    split_bwd(rows * (hq + hk), hq, hk, vec ? std::max(1, 32 / lanes_per_row(dim)) * bwd_unroll(dtype) : 1, p.ctas);
    if (p.ctas[0] <= 1 && p.ctas[1] <= 1) {  // few rows: no partial sums, one launch
      p.side[0].dw_out = hq > 0 ? a.dqw : nullptr;
      p.side[1].dw_out = hk > 0 ? a.dkw : nullptr;
    } else {
      if (a.dqw != nullptr) p.side[0].dw = reinterpret_cast<float*>(workspace);
      if (a.dkw != nullptr) p.side[1].dw = reinterpret_cast<float*>(workspace) + (size_t)p.ctas[0] * dim;
    }
    grid = dim3((unsigned)(p.ctas[0] + p.ctas[1]));
  } else if (vec) {
    if ((rows + 7) / 8 > 0x7fffffff) {
      set_error("%s: too many tokens", a.what);
      return QLIN_EINVAL;
    }
    grid = dim3((unsigned)((rows + 7) / 8), (unsigned)(p.side[0].chunks + p.side[1].chunks));
  } else {
    for (int i = 0; i < 2; ++i)
      p.ctas[i] = (int)std::min<long long>(8ll * sm_count(), (rows * heads[i] + 7) / 8);
    grid = dim3((unsigned)(p.ctas[0] + p.ctas[1]));
  }
  if (dtype == QLIN_F16) launch_dtype<QLIN_F16>(p, vec, a.back, grid, stream);
  else if (dtype == QLIN_BF16) launch_dtype<QLIN_BF16>(p, vec, a.back, grid, stream);
  else launch_dtype<QLIN_F32>(p, vec, a.back, grid, stream);
  int rc = rot_launched(a.what);
  if (rc || !a.back || (a.dqw == nullptr && a.dkw == nullptr)) return rc;
  // What is left: a side's partial rows to add up, or a side without heads, whose gradient is zeros.
  const bool direct = p.ctas[0] <= 1 && p.ctas[1] <= 1;
  if (direct && (hq > 0 || a.dqw == nullptr) && (hk > 0 || a.dkw == nullptr)) return rc;
  DwParams d{};
  d.part[0] = p.side[0].dw;
  d.part[1] = p.side[1].dw;
  d.ctas[0] = p.ctas[0];
  d.ctas[1] = p.ctas[1];
  d.out[0] = direct && hq > 0 ? nullptr : a.dqw;
  d.out[1] = direct && hk > 0 ? nullptr : a.dkw;
  d.D = dim;
  d.w_dtype = w_dtype;
  launch_dependent(dw_sum_kernel, dim3((dim + 31) / 32, 2), dim3(32, 32), 0, stream, 0, d);
  return rot_launched(a.what);
}

// This translation unit's bounds record (QLIN_CHECKS build).
QLIN_BOUNDS_READER(bounds_read_rotary)

}  // namespace qlin

using namespace qlin;

extern "C" {

int qlin_rotary_table(const void* positions, int pos_dtype, int64_t tokens, int axes, const int32_t* axes_dim,
                      double theta, float* table, void* stream) {
  if (tokens < 0 || axes <= 0 || axes_dim == nullptr || !(theta >= 1.0) || !std::isfinite(theta)) {
    set_error("qlin_rotary_table: bad sizes tokens=%lld axes=%d theta=%g", (long long)tokens, axes, theta);
    return QLIN_EINVAL;
  }
  if (axes > kMaxPairs) {
    set_error("qlin_rotary_table: at most %d axes", kMaxPairs);
    return QLIN_EDECLINE;
  }
  int pairs = 0;
  for (int a = 0; a < axes; ++a) {
    if (axes_dim[a] < 0 || axes_dim[a] % 2 != 0) {
      set_error("qlin_rotary_table: axis %d has %d dimensions (an even number is needed)", a, (int)axes_dim[a]);
      return QLIN_EINVAL;
    }
    if (axes_dim[a] / 2 > kMaxPairs - pairs) {
      set_error("qlin_rotary_table: at most %d rotated pairs", kMaxPairs);
      return QLIN_EDECLINE;
    }
    pairs += axes_dim[a] / 2;
  }
  if (pos_dtype != QLIN_F32 && pos_dtype != QLIN_I32 && pos_dtype != QLIN_I64) {
    set_error("qlin_rotary_table: positions are f32, i32 or i64");
    return QLIN_EDECLINE;
  }
  if (tokens == 0 || pairs == 0) return QLIN_OK;
  if (positions == nullptr || table == nullptr || (reinterpret_cast<uintptr_t>(table) & 7)) {
    set_error("qlin_rotary_table: null or misaligned pointer");
    return QLIN_EINVAL;
  }
  // Launch parameters cost their size: a quarter of the largest table's for the usual head of up to 128 values.
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (pairs <= 64) launch_table<64>(positions, pos_dtype, tokens, axes, axes_dim, pairs, theta, table, s);
  else launch_table<kMaxPairs>(positions, pos_dtype, tokens, axes, axes_dim, pairs, theta, table, s);
  return rot_launched("qlin_rotary_table");
}

int qlin_qk_norm_rotary(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, int dtype,
                        int64_t batch, int64_t tokens, int q_heads, int k_heads, int head_dim, const void* q_weight,
                        const void* k_weight, int weight_dtype, const float* table, int64_t table_batch_stride,
                        int pairs, float eps, int interleaved, void* q_out, const int64_t* q_out_strides, void* k_out,
                        const int64_t* k_out_strides, void* stream) {
  HeadCall a{};
  a.what = "qlin_qk_norm_rotary";
  a.q = q;
  a.k = k;
  a.q_strides = q_strides;
  a.k_strides = k_strides;
  a.oq = q_out;
  a.ok = k_out;
  a.oq_strides = q_out_strides;
  a.ok_strides = k_out_strides;
  if ((q_heads > 0 && (q_strides == nullptr || q_out_strides == nullptr)) ||
      (k_heads > 0 && (k_strides == nullptr || k_out_strides == nullptr))) {
    set_error("%s: null strides", a.what);
    return QLIN_EINVAL;
  }
  return head_norm(a, dtype, batch, tokens, q_heads, k_heads, head_dim, q_weight, k_weight, weight_dtype, table,
                   table_batch_stride, pairs, eps, interleaved, nullptr, 0, reinterpret_cast<cudaStream_t>(stream));
}

size_t qlin_qk_norm_rotary_backward_workspace(int64_t batch, int64_t tokens, int q_heads, int k_heads, int head_dim) {
  if (batch <= 0 || tokens <= 0 || q_heads < 0 || k_heads < 0 || q_heads + k_heads == 0 || head_dim <= 0) return 0;
  return bwd_workspace(batch * tokens, q_heads, k_heads, head_dim);
}

int qlin_qk_norm_rotary_backward(const void* dq, const int64_t* dq_strides, const void* dk, const int64_t* dk_strides,
                                 const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                 int dtype, int64_t batch, int64_t tokens, int q_heads, int k_heads, int head_dim,
                                 const void* q_weight, const void* k_weight, int weight_dtype, const float* table,
                                 int64_t table_batch_stride, int pairs, float eps, int interleaved, void* q_grad,
                                 const int64_t* q_grad_strides, void* k_grad, const int64_t* k_grad_strides,
                                 void* q_weight_grad, void* k_weight_grad, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  HeadCall a{};
  a.what = "qlin_qk_norm_rotary_backward";
  a.back = true;
  a.q = q;
  a.k = k;
  a.dq = dq;
  a.dk = dk;
  a.q_strides = q_strides;
  a.k_strides = k_strides;
  a.dq_strides = dq_strides;
  a.dk_strides = dk_strides;
  a.oq = q_grad;
  a.ok = k_grad;
  a.oq_strides = q_grad_strides;
  a.ok_strides = k_grad_strides;
  a.dqw = q_weight_grad;
  a.dkw = k_weight_grad;
  if ((q_heads > 0 && (q_strides == nullptr || dq_strides == nullptr || q_grad_strides == nullptr)) ||
      (k_heads > 0 && (k_strides == nullptr || dk_strides == nullptr || k_grad_strides == nullptr))) {
    set_error("%s: null strides", a.what);
    return QLIN_EINVAL;
  }
  return head_norm(a, dtype, batch, tokens, q_heads, k_heads, head_dim, q_weight, k_weight, weight_dtype, table,
                   table_batch_stride, pairs, eps, interleaved, workspace, workspace_bytes,
                   reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
