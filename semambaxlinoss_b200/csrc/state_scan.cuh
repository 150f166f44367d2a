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

// E elements at i, i + stride, ... of steps t, t + TS, ... (0 from step t1 on).
template <int E, int TS>
__device__ __forceinline__ void fetch_pairs(uint32_t (&r)[E], const void* base, int bf16, int64_t i, int64_t stride,
                                            int t, int t1, bool ok) {
  if (bf16) {
    const unsigned short* b = reinterpret_cast<const unsigned short*>(base);
#pragma unroll
    for (int e = 0; e < E; ++e) r[e] = ok && t + e * TS < t1 ? b[i + e * stride] : 0u;
  } else {
    const uint32_t* b = reinterpret_cast<const uint32_t*>(base);
#pragma unroll
    for (int e = 0; e < E; ++e) r[e] = ok && t + e * TS < t1 ? b[i + e * stride] : 0u;
  }
}

__device__ __forceinline__ float sigmoid(float v) { return semx::rcp_approx(1.f + semx::ex2_approx(-kLog2e * v)); }
__device__ __forceinline__ float softplus(float v) { return semx::softplus(v); }

// Lanes per channel for N modes, MPT per thread.
inline int lanes_for(int N, int mpt) {
  int g = 1;
  while (g * mpt < N) g *= 2;
  return g;
}

// v[u] summed over the GL neighbouring lanes; lane m (mod R, R = 1, 2 or 4 values) returns
// the total of v[m mod R].
template <int GL, int R>
__device__ __forceinline__ float lanes_scatter_sum(float (&v)[R], int lane) {
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
