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
using semx::for_unused_rows;
using semx::Piece;
using semx::piece_base;
using semx::rows_begin;
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
  int access;            // enum Access that all row operands allow
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
  float* v;  // in front of the gate, fp32: dz is made from it, and a rounding to bf16 showed (2.34e-3 off, now 1.66e-3)
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

// How a kernel reads and writes rows: kAny takes any type, stride, alignment and width, one
// element at a time; kBf16 and kFp32 take four neighbours in one access (every operand of
// that type, rows and groups that start on four elements: ScanParams::access).
enum Access { kAny = 0, kBf16 = 1, kFp32 = 2 };
// Access of an fp32 tensor beside rows of access ACC.
constexpr int fp32_beside(int acc) { return acc == kAny ? kAny : kFp32; }

template <int ACC>
struct RawQuad {
  typedef uint4 type;
};
template <>
struct RawQuad<kBf16> {
  typedef uint2 type;
};

// Elements i .. i + 3 as they are stored (kAny: the first n of them).
template <int ACC>
__device__ __forceinline__ typename RawQuad<ACC>::type load_quad(const void* base, int64_t i, int bf16, int n) {
  if constexpr (ACC == kBf16) {
    return *reinterpret_cast<const uint2*>(reinterpret_cast<const unsigned short*>(base) + i);
  } else if constexpr (ACC == kFp32) {
    return *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(base) + i);
  } else {
    uint4 r = make_uint4(0u, 0u, 0u, 0u);
    if (n > 0) r.x = load_raw(base, i, bf16);
    if (n > 1) r.y = load_raw(base, i + 1, bf16);
    if (n > 2) r.z = load_raw(base, i + 2, bf16);
    if (n > 3) r.w = load_raw(base, i + 3, bf16);
    return r;
  }
}
template <int ACC>
__device__ __forceinline__ float4 quad_floats(const typename RawQuad<ACC>::type& r, int bf16) {
  if constexpr (ACC == kBf16) {
    return make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16),
                       __uint_as_float(r.y & 0xffff0000u));
  } else if constexpr (ACC == kFp32) {
    return make_float4(__uint_as_float(r.x), __uint_as_float(r.y), __uint_as_float(r.z), __uint_as_float(r.w));
  } else {
    return make_float4(as_float(r.x, bf16), as_float(r.y, bf16), as_float(r.z, bf16), as_float(r.w, bf16));
  }
}
template <int ACC>
__device__ __forceinline__ void store_quad(void* base, int64_t i, int bf16, int n, float4 v) {
  if constexpr (ACC == kBf16) {
    uint2 q;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
    h[0] = __floats2bfloat162_rn(v.x, v.y);
    h[1] = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(base) + i) = q;
  } else if constexpr (ACC == kFp32) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + i) = v;
  } else {
    if (n > 0) store(base, i, bf16, v.x);
    if (n > 1) store(base, i + 1, bf16, v.y);
    if (n > 2) store(base, i + 2, bf16, v.z);
    if (n > 3) store(base, i + 3, bf16, v.w);
  }
}
// Four elements from base[i] on (kBf16, kFp32) into shared memory, zeros where there are none to
// copy; on their way until copies_done(). Only the thread that asked for them reads them.
template <int ACC>
__device__ __forceinline__ void copy_quad(typename RawQuad<ACC>::type* to, const void* base, int64_t i, bool any) {
  const unsigned at = (unsigned)__cvta_generic_to_shared(to);
  const char* from = reinterpret_cast<const char*>(base) + (any ? i * (ACC == kBf16 ? 2 : 4) : 0);
  if constexpr (ACC == kBf16)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(at), "l"(from), "r"(any ? 8 : 0) : "memory");
  else
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(from), "r"(any ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// The first n of four parameters (0 for the rest and without a parameter).
__device__ __forceinline__ float4 load_params(const float* base, int64_t i, int n) {
  if (base == nullptr) return make_float4(0.f, 0.f, 0.f, 0.f);
  return make_float4(n > 0 ? base[i] : 0.f, n > 1 ? base[i + 1] : 0.f, n > 2 ? base[i + 2] : 0.f, n > 3 ? base[i + 3] : 0.f);
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

// Pole exp(d A) from d and A log2(e). The special-function exponential of small negative
// arguments is measured 2e-8 low on average (rms 3.5e-8); a state multiplies hundreds of
// poles, so that average is what reaches the results. kPoleBias moves the argument by as
// much, inside the multiply-add that forms it.
constexpr float kPoleBias = 3.0e-8f;
// A log2(e). An A of -inf becomes the lowest finite value: the rows that fill up a tile have
// d = 0, and 0 times -inf would put a NaN into the state (a step with d > 0 still forgets all).
__device__ __forceinline__ float log2_rate(float A) {
  constexpr float kLowest = -3.4028234663852886e38f;
  const float a = A * kLog2e;
  return a < kLowest ? kLowest : a;
}
__device__ __forceinline__ float pole(float d, float A2) { return semx::ex2_approx(fmaf(d, A2, kPoleBias)); }

__device__ __forceinline__ float sigmoid(float v) { return semx::rcp_approx(1.f + semx::ex2_approx(-kLog2e * v)); }

// log(1 + exp(v)) = max(v, 0) + log1p(e), e = exp(-|v|): log1p(e) / e on [0, 1] is a degree 9
// Chebyshev interpolant (5e-9 off, 1e-7 with its roundings); e is corrected for the rounding
// of its argument, which small steps (v near -7) would show in full. Above 20 the logarithm
// is below half a step of v. e comes back for the derivative.
__device__ __forceinline__ float softplus(float v, float* exp_out = nullptr) {
  // exp(-150) is 0 in fp32; the bound keeps infinities out of the products below.
  const float t = fmaxf(-fabsf(v), -150.f), p = t * kLog2e;
  // What the product lost, and the constant's own tail log2(e) - float(log2(e)).
  const float lost = fmaf(t, 1.925963033500e-8f, fmaf(t, kLog2e, -p));
  float e = semx::ex2_approx(p);
  e = fmaf(e, lost * 0.6931471805599453f, e);
  if (exp_out != nullptr) *exp_out = e;
  float s = fmaf(-0.0031760570127512695f, e, 0.019542528316378593f);
  s = fmaf(s, e, -0.05637361481785774f);
  s = fmaf(s, e, 0.10543623566627502f);
  s = fmaf(s, e, -0.1526966691017151f);
  s = fmaf(s, e, 0.1966327428817749f);
  s = fmaf(s, e, -0.24951615929603577f);
  s = fmaf(s, e, 0.33329710364341736f);
  s = fmaf(s, e, -0.49999892711639404f);
  s = fmaf(s, e, 1.0f);
  return fmaf(s, e, v < 0.f ? 0.f : v);  // a NaN stays
}
__device__ __forceinline__ float4 softplus4(float4 v) {
  return make_float4(softplus(v.x), softplus(v.y), softplus(v.z), softplus(v.w));
}
// softplus' = 1 / (1 + exp(-v)) from e = exp(-|v|).
__device__ __forceinline__ float softplus_slope(float v, float e) {
  const float r = semx::rcp_approx(1.f + e);
  return v < 0.f ? e * r : r;
}

__device__ __forceinline__ float4 gate4(float4 v, float4 z) {
  return make_float4(v.x * (z.x * sigmoid(z.x)), v.y * (z.y * sigmoid(z.y)), v.z * (z.z * sigmoid(z.z)),
                     v.w * (z.w * sigmoid(z.w)));
}

// Rows at which a sequence of a packed batch is cut although the batch as a whole fills the
// GPU: one far longer than the mean (a prompt beside single tokens) would run on alone. The
// others stay whole and cost the two additional launches. 8192 rows of 1024 channels in 64
// sequences: one of 7940 rows and 63 of 4, whole 979 us, cut at 4 times the mean 191 us; all of
// 128 rows, 64 us and 70.
inline int64_t outlier_rows(int64_t mean) {
  const int64_t Q = (4 * mean + 15) / 16 * 16;
  return Q < 128 ? 128 : Q;
}

// CTAs that join pieces: the (channel, mode)s across, a few of the sequences at a time down.
inline dim3 join_grid(const ScanParams& p) {
  const int64_t tiles = semx::cdiv((int64_t)p.C * p.N, kThreads);
  int64_t down = semx::cdiv((int64_t)148 * 16, tiles);
  if (down > p.m.S) down = p.m.S;
  return dim3((unsigned)tiles, (unsigned)(down < 1 ? 1 : down > 65535 ? 65535 : down));
}

// Whether one of the sequences that the CTA walks over (every gridDim.y-th) has more than one
// piece. Called by all threads of the CTA.
__device__ __forceinline__ bool any_split(const semx::SeqMap& m) {
  int found = 0;
  for (int64_t s = blockIdx.y + (int64_t)threadIdx.x * gridDim.y; s < m.S; s += (int64_t)blockDim.x * gridDim.y) {
    const int64_t row0 = seq_start(m, s);
    found |= (m.cu == nullptr ? m.L : seq_start(m, s + 1) - row0) > m.Q;
  }
  return __syncthreads_or(found) != 0;
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
