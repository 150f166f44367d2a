// Deterministic reduction of per-sequence partial rows over the sequence axis.
//
// rows (S, K) -> out (K), in two fixed-order stages so the result is bitwise
// reproducible: stage 1 sums kRowsPerGroup consecutive rows per column (one CTA column
// block x row group), stage 2 sums the groups in order and scatters the K columns into up
// to kMaxSegments output arrays (consecutive column ranges; NULL arrays are skipped).
#pragma once

#include "semx_common.cuh"

namespace semx {
namespace {

constexpr int kRowsPerGroup = 32;
constexpr int kMaxSegments = 8;

struct Segments {
  float* out[kMaxSegments];
  int64_t len[kMaxSegments];
  int n;
};

__global__ void colsum_stage1(const float* __restrict__ rows, int64_t S, int64_t K,
                              float* __restrict__ group_sums) {
  const int64_t k = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (k >= K) return;
  const int64_t r0 = (int64_t)blockIdx.y * kRowsPerGroup;
  const int64_t r1 = min(r0 + kRowsPerGroup, S);
  float acc = 0.f;
  for (int64_t r = r0; r < r1; ++r) acc += rows[r * K + k];
  group_sums[(int64_t)blockIdx.y * K + k] = acc;
}

__global__ void colsum_stage2(const float* __restrict__ group_sums, int64_t G, int64_t K,
                              Segments seg) {
  const int64_t k = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (k >= K) return;
  int64_t off = k;
  int which = 0;
  while (which < seg.n && off >= seg.len[which]) {
    off -= seg.len[which];
    ++which;
  }
  if (which >= seg.n || seg.out[which] == nullptr) return;
  float acc = 0.f;
  for (int64_t q = 0; q < G; ++q) acc += group_sums[q * K + k];
  seg.out[which][off] = acc;
}

// One-launch form for tall, narrow partial sums: a CTA takes COLS columns, its 1024 / COLS
// row lanes every (1024 / COLS)-th row each, and the lanes' sums are added in lane order. The
// order is fixed too, but it is another one than colsum's, so the two do not give the same
// bits. 2424 rows of 1280: 16 us in two launches, 8 us in this one.
template <int COLS>
__global__ void __launch_bounds__(1024) colsum_once_kernel(const float* __restrict__ rows, int64_t S, int64_t K,
                                                           Segments seg) {
  constexpr int LANES = 1024 / COLS;
  __shared__ float sums[LANES][COLS + 1];
  const int col = threadIdx.x % COLS, lane = threadIdx.x / COLS;
  const int64_t k = (int64_t)blockIdx.x * COLS + col;
  float acc = 0.f;
  if (k < K)
#pragma unroll 8
    for (int64_t r = lane; r < S; r += LANES) acc += rows[r * K + k];
  sums[lane][col] = acc;
  // Halving in a fixed order: lane l takes lane l + n.
#pragma unroll
  for (int n = LANES / 2; n >= 1; n /= 2) {
    __syncthreads();
    if (lane < n) sums[lane][col] += sums[lane + n][col];
  }
  if (lane != 0 || k >= K) return;
  int64_t off = k;
  int which = 0;
  while (which < seg.n && off >= seg.len[which]) {
    off -= seg.len[which];
    ++which;
  }
  if (which < seg.n && seg.out[which] != nullptr) seg.out[which][off] = sums[0][col];
}

inline int colsum_once(const float* rows, int64_t S, int64_t K, const Segments& seg, cudaStream_t st) {
  if (K <= 0) return SEMX_OK;
  // Few columns: narrower CTAs, so that they still fill the GPU (2424 rows of 1280 columns: 32
  // columns per CTA 22.8 us, 8 columns 10.8 with 4 rows loaded ahead, 8 with 8).
  if (K < 32 * 148) colsum_once_kernel<8><<<(unsigned)cdiv(K, 8), 1024, 0, st>>>(rows, S, K, seg);
  else colsum_once_kernel<32><<<(unsigned)cdiv(K, 32), 1024, 0, st>>>(rows, S, K, seg);
  return check_launch("colsum_once_kernel");
}

inline size_t colsum_group_floats(int64_t S, int64_t K) {
  return (size_t)cdiv(S, kRowsPerGroup) * (size_t)K;
}

// rows: (S, K); group_sums: colsum_group_floats(S, K) floats of scratch.
inline int colsum(const float* rows, int64_t S, int64_t K, float* group_sums, const Segments& seg,
                  cudaStream_t st) {
  if (K <= 0) return SEMX_OK;
  const int64_t G = cdiv(S, kRowsPerGroup);
  if (G > 0) {
    colsum_stage1<<<dim3((unsigned)cdiv(K, 256), (unsigned)G), 256, 0, st>>>(rows, S, K, group_sums);
    int rc = check_launch("colsum_stage1");
    if (rc != SEMX_OK) return rc;
  }
  colsum_stage2<<<(unsigned)cdiv(K, 256), 256, 0, st>>>(group_sums, G, K, seg);
  return check_launch("colsum_stage2");
}

}  // namespace
}  // namespace semx
