// Shared by the selective state scan's kernels (whole sequences, forward and backward, and
// single tokens): parameters, loads and stores of either type, sums over a channel's lanes.
#pragma once

#include <cuda_bf16.h>

#include "semx_common.cuh"
#include "semx_math.cuh"
#include "semx_seq.cuh"

namespace semx_scan {

using semx::find_piece;
using semx::find_slot;
using semx::Piece;
using semx::piece_base;
using semx::rows_end;
using semx::seq_start;

constexpr int kThreads = 128;
constexpr int kMaxN = 128;
constexpr int kBlock = 8;  // steps between the states that a training forward keeps
constexpr float kLog2e = 1.4426950408889634f;

struct ScanParams {
  semx::SeqMap m;
  int C, N, G, cpg;      // channels, modes, groups, channels per group
  int ctiles, tpg;       // channel tiles, and tiles per group
  int bf16, dt_bf16, softplus;
  int vec2;              // every row operand allows accesses of two neighbouring channels
  int64_t ldx, lddt, ldz, ldb, ldc;
  const void* x;
  const void* dt;
  const float* A;
  const void* B;
  const void* Cm;
  const float* D;
  const void* z;
  const float* dt_bias;
  void* y;
  float* state;
  void* v;
  float* ckpt;
  float* entry;  // (pieces, C, N) state in front of each piece (backward: gradient behind it)
  float* dsum;   // (pieces, C) sum of the piece's steps
  const void* dy;
  void* dx;
  void* ddt;
  void* dz;
  float* pBC;    // backward: (channel tiles, T, 2 N) partial dB | dC
  float* part;   // backward: (pieces, C (N + 2)) partial dA | dD | ddt_bias
};

int scan_validate(const SemxStateScanArgs* a, bool bwd, ScanParams* p);
size_t scan_bwd_workspace(ScanParams& p);

__device__ __forceinline__ uint32_t load_raw(const void* base, int64_t i, int bf16) {
  return bf16 ? (uint32_t) reinterpret_cast<const unsigned short*>(base)[i] : reinterpret_cast<const uint32_t*>(base)[i];
}
__device__ __forceinline__ float as_float(uint32_t raw, int bf16) { return __uint_as_float(bf16 ? raw << 16 : raw); }
__device__ __forceinline__ float load(const void* base, int64_t i, int bf16) { return as_float(load_raw(base, i, bf16), bf16); }
__device__ __forceinline__ void store(void* base, int64_t i, int bf16, float v) {
  if (bf16) reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16(v);
  else reinterpret_cast<float*>(base)[i] = v;
}

// Two neighbouring channels of a row as they are stored (bf16: x alone).
__device__ __forceinline__ uint2 load_pair(const void* base, int64_t i, int bf16, bool vec, bool two) {
  uint2 r = make_uint2(0u, 0u);
  if (bf16) {
    const unsigned short* b = reinterpret_cast<const unsigned short*>(base) + i;
    if (vec) r.x = *reinterpret_cast<const uint32_t*>(b);
    else r.x = (uint32_t)b[0] | (two ? (uint32_t)b[1] << 16 : 0u);
  } else {
    const uint32_t* b = reinterpret_cast<const uint32_t*>(base) + i;
    if (vec) r = *reinterpret_cast<const uint2*>(b);
    else r = make_uint2(b[0], two ? b[1] : 0u);
  }
  return r;
}
__device__ __forceinline__ float2 pair_floats(uint2 r, int bf16) {
  return bf16 ? make_float2(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u))
              : make_float2(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ __forceinline__ void store_pair(void* base, int64_t i, int bf16, bool vec, bool two, float a, float b) {
  if (bf16) {
    __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(base) + i;
    if (vec) {
      *reinterpret_cast<__nv_bfloat162*>(o) = __floats2bfloat162_rn(a, b);
    } else {
      o[0] = __float2bfloat16(a);
      if (two) o[1] = __float2bfloat16(b);
    }
  } else {
    float* o = reinterpret_cast<float*>(base) + i;
    if (vec) {
      *reinterpret_cast<float2*>(o) = make_float2(a, b);
    } else {
      o[0] = a;
      if (two) o[1] = b;
    }
  }
}

// Pairs of fp32 values in one register pair: one instruction works on both.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack2(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(f2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Poles exp(d A) of two modes from d (in both halves) and A log2(e). The special-function
// exponential of small negative arguments is measured 2e-8 low on average (rms 3.5e-8); a
// state multiplies hundreds of poles, so that average is what reaches the results. kPoleBias
// moves the argument by as much, inside the multiply-add that forms it.
constexpr float kPoleBias = 3.0e-8f;
__device__ __forceinline__ f2 poles2(f2 dd, f2 A2, f2 bias) {
  const float2 v = unpack2(fma2(dd, A2, bias));
  return pack2(semx::ex2_approx(v.x), semx::ex2_approx(v.y));
}

__device__ __forceinline__ float sigmoid(float v) { return semx::rcp_approx(1.f + semx::ex2_approx(-kLog2e * v)); }

// log(1 + exp(v)) = max(v, 0) + log1p(e), e = exp(-|v|): log1p(e) / e on [0, 1] is a degree 9
// Chebyshev interpolant (5e-9 off, 1e-7 with its roundings); e is corrected for the rounding
// of its argument, which small steps (v near -7) would show in full. Above 20 the
// logarithm is below half a step of v.
__device__ __forceinline__ float softplus(float v) {
  const float t = -fabsf(v), p = t * kLog2e;
  const float lost = fmaf(t, kLog2e, -p) + t * 1.925963033500e-8f;  // log2(e) - float(log2(e))
  float e = semx::ex2_approx(p);
  e = fmaf(e, lost * 0.6931471805599453f, e);
  float s = -0.0031760570127512695f;
  s = fmaf(s, e, 0.019542528316378593f);
  s = fmaf(s, e, -0.05637361481785774f);
  s = fmaf(s, e, 0.10543623566627502f);
  s = fmaf(s, e, -0.1526966691017151f);
  s = fmaf(s, e, 0.1966327428817749f);
  s = fmaf(s, e, -0.24951615929603577f);
  s = fmaf(s, e, 0.33329710364341736f);
  s = fmaf(s, e, -0.49999892711639404f);
  s = fmaf(s, e, 1.0f);
  return fmaf(s, e, fmaxf(v, 0.f));
}

// Lanes per channel for N modes, MPT per thread.
inline int lanes_for(int N, int mpt) {
  int g = 1;
  while (g * mpt < N) g *= 2;
  return g;
}

// v summed over GL neighbouring lanes step by step: of the R = min(GL, 4) values, lane m
// returns the total of v[m mod R].
template <int GL, int R>
__device__ __forceinline__ float lanes_scatter_sum(const float (&v)[R], int lane) {
  float s;
  if constexpr (R == 1) {
    s = v[0];
  } else if constexpr (R == 2) {
    const bool hi = lane & 1;
    s = (hi ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[1], 1);
  } else {
    const bool h2 = lane & 2, h1 = lane & 1;
    const float a = (h2 ? v[2] : v[0]) + __shfl_xor_sync(0xffffffffu, h2 ? v[0] : v[2], 2);
    const float b = (h2 ? v[3] : v[1]) + __shfl_xor_sync(0xffffffffu, h2 ? v[1] : v[3], 2);
    s = (h1 ? b : a) + __shfl_xor_sync(0xffffffffu, h1 ? a : b, 1);
  }
#pragma unroll
  for (int m = 4; m < GL; m *= 2) s += __shfl_xor_sync(0xffffffffu, s, m);
  return s;
}

}  // namespace semx_scan
