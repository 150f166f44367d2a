// Gated projection of a feed-forward block, forward and backward, for sm_100a.
//
//   [u | g] = x W^T + b  (W: H rows of the value, then H rows of the gate);  h = u act(g)
//   du = dh act(g), dg = dh u act'(g);  dx = du Wu + dg Wg,  dW = [du | dg]^T x,  db = column sums
//
// Forward: one kernel does both products, the activation and the last product. A tile is 128 rows of
// x by the same columns of u and g side by side in one accumulator, so the epilogue has both.
// Backward: an elementwise pass makes du and dg from what the forward kept (u and g in fp32: rounded
// to bf16 they would put their rounding into dx and dW on top of that of du and dg), then two
// products run on the same kernel with other operand orders.
// With bf16 operands du and dg are rounded to bf16, because a product of the tensor cores takes both operands of one
// type: dx and dW are 0.0023 off (root mean square) instead of 0.0017. A second part of each would double both products
// (490 of 870 us of a training pass of 8192 x 2048 -> 5504). What is made again (kGate) comes from the forward's
// operands, summed in another order where the forward ran on few rows or began its depth elsewhere: the difference is
// fp32's, under the rounding of du and dg.
//
// Products: tcgen05 on pairs of SMs (a cluster of two CTAs has 256 rows of the result, each CTA's tensor
// memory its 128; each brings its rows of A and half of B's by TMA, and one thread of the pair issues the
// products for both). Persistent: in each CTA one warp loads and sixteen write the accumulators out; two
// accumulators, so that writing a tile overlaps the next one's products.
// fp32 operands are split into three bf16 parts whose sum is the value up to its last bit; six of the nine
// products of parts are taken (the others are below 2^-24 of the result). The tensor cores cut where
// an addition rounds, which shows over thousands of additions: so the large products (first parts) are
// summed in tensor memory over 128 of the depth at a time, and those sums in registers; the small ones
// have an accumulator of their own. bf16 sums over rows (dW) leave tensor memory every 4096 rows; h and dx, whose depth
// is a width, stay there (9e-8 of a sum per 16 of the depth at most, where terms have one sign).
// Few rows (bf16 up to 16, fp32 16 by eights): the weights' bytes are the bound, and warps stream them, bf16
// through the legacy tensor products (a tcgen05 tile would be nearly empty), fp32 through packed multiplies.
//
// Measured (device time): 8192 x 2048 -> 5504 bf16 forward 272 us (1.36 PFLOP/s; the GPU's power limit is what
// bounds it), dW 250, dx 237; 4099 x 2048 -> 5461 131 (1.40); 192 x 4096 -> 11008 43 (4.2 TB/s of weights);
// 129684 x 64 -> 256 fp32, which is its results' bytes: forward 118 (3.7 TB/s; the epilogue's chain of
// tensor memory, activation and exchange), dx 85, dW 76; bf16 forward 49 (without biases 42), its products again for
// du and dg 112 (88).
#include <cuda.h>
#include <cuda_bf16.h>

#include <atomic>
#include <type_traits>

#include "semx_reduce.cuh"
#include "semx_tc.cuh"
#include "state_scan.cuh"

namespace {

using semx::cdiv;
using semx_scan::sigmoid;

constexpr int kM = 128, kK = 64;    // rows of a CTA's tile, depth of a stage (128 bytes of bf16)
constexpr int kEpi = 16;            // warps that write out: four for each quarter of the rows
constexpr int kGemmT = (kEpi + 2) * 32;  // then one that loads and one that issues products
constexpr int kSms = 148, kPairs = kSms / 2;
constexpr long long kPatience = 4000000000ll;  // cycles that a wait takes at most
constexpr int kCols = 16;           // columns that a warp writes at a time
constexpr int kBufRow = kCols + 4;  // floats of a row of its exchange buffer
constexpr int kBuf = 32 * kBufRow + 64;  // floats of the buffer, and of u's and g's biases (32 columns) behind it
constexpr int kParts = 3;           // bf16 parts of an fp32 value
// Stages whose large products one accumulator takes: of fp32; and of bf16 where the depth is the rows, which have no
// end (dW of 131072 x 1024 -> 2752, terms of one sign: in one sum 7.1e-4 too small, of 524288 rows 3.0e-3, where the
// results' own rounding is 1.4e-3; in runs of 64 stages 1.2e-5 for the former. dW of 8192 x 2048 -> 5504
// 246.7 us in one sum, 249.8, 248.9 and 248.5 in runs of 16, 32 and 64; 16384 x 1024 -> 2752 131.8, and 139.6, 136.3, 134.6).
constexpr int kDrain = 2, kRun = 64;

__device__ unsigned int g_gemm_timeouts;

enum Mode { kFwd = 0, kDx = 1, kDw = 2, kGate = 3 };  // kGate (bf16): the forward's products again, for du and dg

struct GemmParams {
  int64_t M, N;           // rows and columns of the result (kFwd: N = H; kDw: M = H, once per half)
  int tiles_m, tiles_n;   // kDw: tiles_m of one half
  int tiles;              // in all
  int depth, khalf;       // stages in all, and of one half of the depth (kDx: u, then g)
  int whole, splits;      // tiles from number `whole` on run in as many slices of the depth
  void* out;              // kFwd: h
  int64_t ldo;
  int out_bf16;
  const void* dh;         // kGate: (M, N) of out's type
  __nv_bfloat16* dz;      // kGate: du and dg (2, M, ldz)
  int64_t ldz;
  float* sums;            // kGate: column sums of each warp's 32 rows (8 tiles_m, 2 N), or NULL
  float* u;               // kFwd: u and g in front of the activation, or NULL
  float* g;
  int64_t ldu;
  const void* bias;       // (2 H) or NULL
  int bias_bf16;
  int gelu;
  float* part;            // sums of the sliced tiles: (slices, tiles - whole, 256, accumulator's columns)
};

// Half of erfc(|g| / sqrt(2)) and e = exp(-g^2 / 2): erfc(z) = t q(t) exp(-z^2) with t = 1 / (1 + z / 2), the
// substitution of the erfc in Press et al., Numerical Recipes; q is a polynomial of degree 8 of our own, fitted to the
// least largest relative error for z up to 9.5 (at most 6.6e-8; further out the exponential is 0). The exponential's
// argument is rounded, so that e is up to 2^-24 g^2 of itself off beside the special function's error: 4.3e-7 for
// |g| < 3, 7.6e-6 in the far tail at 13, whose values are 1e-38.
__device__ __forceinline__ float normal_tail(float g, float* e) {
  const float t = semx::rcp_approx(fmaf(fabsf(g), 0.35355339059327379f, 1.f));
  *e = semx::ex2_approx(-0.72134752044448170f * g * g);
  float q = fmaf(-0.029445456340909004f, t, 0.1418512910604477f);
  q = fmaf(q, t, -0.24269245564937592f);
  q = fmaf(q, t, 0.13798969984054565f);
  q = fmaf(q, t, -0.012589219957590103f);
  q = fmaf(q, t, 0.10103505849838257f);
  q = fmaf(q, t, 0.1216304749250412f);
  q = fmaf(q, t, 0.1411767452955246f);
  q = fmaf(q, t, 0.14104384183883667f);
  return t * q * *e;
}
// (gelu: known to the compiler where many values follow one another. A branch in front of each would keep their
// special functions apart: 129684 x 64 -> 256 bf16 forward 62 us, so 50.)
__device__ __forceinline__ float act_of(float g, bool gelu) {
  if (!gelu) return g * sigmoid(g);
  float e;
  const float tail = normal_tail(g, &e);
  return g * (g < 0.f ? tail : 1.f - tail);
}
// act(g) and act'(g).
__device__ __forceinline__ void act_and_slope(float g, bool gelu, float* act, float* slope) {
  if (gelu) {
    float e;
    const float tail = normal_tail(g, &e), cdf = g < 0.f ? tail : 1.f - tail;
    *act = g * cdf;
    *slope = fmaf(g * 0.3989422804014327f, e, cdf);
  } else {
    const float s = sigmoid(g);
    *act = g * s;
    *slope = s * fmaf(g, 1.f - s, 1.f);
  }
}

// Value n of the parts of v: v rounded to bf16, then what is left, each rounded. What no bf16 holds
// (infinities, NaN) stays in the first; a value that would round to infinity is cut instead.
__device__ __forceinline__ void parts_of(float v, __nv_bfloat16 (&part)[kParts]) {
  part[0] = __float2bfloat16(v);
  float rest = 0.f;
  if (fabsf(v) <= 3.4028234663852886e38f) {
    if (fabsf(v) >= 3.3961775292304608e38f) part[0] = __ushort_as_bfloat16((unsigned short)(__float_as_uint(v) >> 16));
    rest = v - __bfloat162float(part[0]);
  }
  part[1] = __float2bfloat16(rest);
  part[2] = __float2bfloat16(rest - __bfloat162float(part[1]));
}

// -- tensor core plumbing -----------------------------------------------------------------------

// A copy into this CTA's shared memory that reports to `bar`, a barrier of the pair (its address in the
// cluster's window).
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          semx::tc::smem_addr(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
// Address of CTA `rank`'s copy of a shared variable in the cluster's window.
__device__ __forceinline__ uint32_t in_cluster(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(semx::tc::smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void expect_bytes(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(semx::tc::smem_addr(bar)), "r"(bytes) : "memory");
}
// (Relaxed: it says that tensor memory has been read, which has ended by then, and hands on nothing in
// memory. A release waits for the tile's stores: 4 of 19 cycles between two instructions.)
__device__ __forceinline__ void arrive_in_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// Arrives on this barrier of both CTAs once every product issued before has completed.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                   semx::tc::smem_addr(bar)),
               "h"((uint16_t)3)
               : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* slot, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(semx::tc::smem_addr(slot)), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(taddr), "r"(ncols) : "memory");
}
// 16 columns of this thread's lane of tensor memory from t0 on, and 16 from t1 on; one wait for both.
__device__ __forceinline__ void tmem_ld16_twice(uint32_t t0, uint32_t t1, float (&v)[16], float (&w)[16]) {
  uint32_t r[32];
#define SEMX_R8(o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%32];\n"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%33];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : SEMX_R8(0), SEMX_R8(8), SEMX_R8(16), SEMX_R8(24)
      : "r"(t0), "r"(t1)
      : "memory");
#undef SEMX_R8
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    v[i] = __uint_as_float(r[i]);
    w[i] = __uint_as_float(r[16 + i]);
  }
}
// Descriptor of an operand in 128-byte rows with the 128-byte swizzle. K-major: a row is 64 values of
// the depth, 8-row groups 1024 bytes apart. MN-major: a row is 64 neighbouring M or N values at one
// depth, 8-row groups 1024 bytes apart, the next 64 values 64 rows (8192 bytes) on.
template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  const uint64_t lead = MN ? 8192 >> 4 : 1;
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (lead << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}
constexpr uint32_t idesc_bf16(int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4)                    // fp32 accumulator
         | (1u << 7) | (1u << 10)     // bf16 A and B
         | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// One lane of the warp, always the same one.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}\n" : "=r"(p));
  return p != 0;
}
// Waits for a phase of bar, some two seconds at most.
__device__ __forceinline__ bool wait_some(uint64_t* bar, uint32_t parity, volatile int* dead) {
  if (semx::tc::mbar_wait(bar, parity, 16)) return true;
  const long long from = clock64();
  do {
    if (semx::tc::mbar_wait(bar, parity, 64)) return true;
    if (dead != nullptr && *dead) return false;
  } while (clock64() - from < kPatience);
  return false;
}
// The same; false when it gave up or another role has.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, volatile int* dead) {
  if (wait_some(bar, parity, dead)) return true;
  if (*dead) return false;
  if (atomicExch((int*)dead, 1) == 0) atomicAdd(&g_gemm_timeouts, 1u);
  return false;
}

// Shared memory is a ring of slots: one part of a stage's rows of A (128) and of B (half of the tile's).
constexpr int slot_bytes(int bn) { return (kM + bn / 2) * kK * 2; }
constexpr int slots_of(int bn) { return bn == 256 ? 5 : bn == 128 ? 7 : 8; }
constexpr size_t gemm_smem(int bn) {
  return 1024 + (size_t)slots_of(bn) * slot_bytes(bn) + kEpi * kBuf * sizeof(float);
}

// Tile number `index` of the result; slice `split` of `of` of its depth.
struct Tile {
  int m, n, half, index, split, of;
};
__host__ __device__ __forceinline__ int works_of(const GemmParams& p) { return p.whole + (p.tiles - p.whole) * p.splits; }
__device__ __forceinline__ Tile tile_number(const GemmParams& p, int index) {
  Tile t;
  t.index = index;
  t.split = 0;
  t.of = 1;
  t.half = 0;
  int i = index;
  const int per_half = p.tiles_m * p.tiles_n;
  if (i >= per_half) {
    t.half = 1;
    i -= per_half;
  }
  // Eight tiles down, then one across: the operands of the tiles that run together stay in L2.
  const int per = 8 * p.tiles_n, grp = i / per, r = i % per;
  const int down = min(8, p.tiles_m - grp * 8);
  t.m = grp * 8 + r % down;
  t.n = r / down;
  return t;
}
__device__ __forceinline__ Tile tile_at(const GemmParams& p, int w) {
  if (w < p.whole) return tile_number(p, w);
  const int i = (w - p.whole) / p.splits;
  Tile t = tile_number(p, p.whole + i);
  t.split = w - p.whole - i * p.splits;
  t.of = p.splits;
  return t;
}

// 32 rows of 16 values, a lane's row each, to out[row0 ..][col0 ..] through the warp's buffer, so that a
// row's values leave as whole sectors. rows, cols: how many of them exist.
__device__ __forceinline__ void write_block(float* buf, const float (&v)[kCols], void* out, int64_t ld, int64_t row0, int64_t col0,
                                            int rows, int cols, int bf16) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kCols; i += 4)
    *reinterpret_cast<float4*>(&buf[lane * kBufRow + i]) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  __syncwarp();
  if (bf16) {
    __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(out) + row0 * ld + col0;
    if (cols >= kCols && ld % 8 == 0 && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
      const int c = lane % 2 * 8;
#pragma unroll
      for (int it = 0; it < 2; ++it) {
        const int r = it * 16 + lane / 2;
        const float4 a = *reinterpret_cast<const float4*>(&buf[r * kBufRow + c]);
        const float4 b = *reinterpret_cast<const float4*>(&buf[r * kBufRow + c + 4]);
        uint4 q;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
        h[0] = __floats2bfloat162_rn(a.x, a.y);
        h[1] = __floats2bfloat162_rn(a.z, a.w);
        h[2] = __floats2bfloat162_rn(b.x, b.y);
        h[3] = __floats2bfloat162_rn(b.z, b.w);
        if (r < rows) *reinterpret_cast<uint4*>(to + r * ld + c) = q;
      }
    } else {
      const int c = lane % kCols;
      for (int r = lane / kCols; r < rows; r += 2)
        if (c < cols) to[r * ld + c] = __float2bfloat16(buf[r * kBufRow + c]);
    }
  } else {
    float* to = reinterpret_cast<float*>(out) + row0 * ld + col0;
    if (cols >= kCols && ld % 4 == 0 && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
      const int c = lane % 4 * 4;
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const int r = it * 8 + lane / 4;
        const float4 a = *reinterpret_cast<const float4*>(&buf[r * kBufRow + c]);
        if (r < rows) *reinterpret_cast<float4*>(to + r * ld + c) = a;
      }
    } else {
      const int c = lane % kCols;
      for (int r = lane / kCols; r < rows; r += 2)
        if (c < cols) to[r * ld + c] = buf[r * kBufRow + c];
    }
  }
  __syncwarp();
}

// The other way: 32 rows of 16 bf16 values to a lane's row each, zeros where there are none.
__device__ __forceinline__ void read_block(float* buf, float (&v)[kCols], const void* src, int64_t ld, int64_t row0, int64_t col0, int rows,
                                           int cols) {
  const int lane = threadIdx.x & 31;
  const __nv_bfloat16* from = reinterpret_cast<const __nv_bfloat16*>(src) + row0 * ld + col0;
  if (cols >= kCols && ld % 8 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    const int c = lane % 2 * 8;
    uint4 q[2];
#pragma unroll
    for (int it = 0; it < 2; ++it) {
      const int r = it * 16 + lane / 2;
      q[it] = r < rows ? __ldcs(reinterpret_cast<const uint4*>(from + r * ld + c)) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int it = 0; it < 2; ++it) {
      float* to = &buf[(it * 16 + lane / 2) * kBufRow + c];
      *reinterpret_cast<float4*>(to) = semx_scan::quad_floats<semx_scan::kBf16>(make_uint2(q[it].x, q[it].y), 1);
      *reinterpret_cast<float4*>(to + 4) = semx_scan::quad_floats<semx_scan::kBf16>(make_uint2(q[it].z, q[it].w), 1);
    }
  } else {
    const int c = lane % kCols;
    for (int r = lane / kCols; r < 32; r += 2) buf[r * kBufRow + c] = r < rows && c < cols ? __bfloat162float(from[r * ld + c]) : 0.f;
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kCols; i += 4) {
    const float4 q = *reinterpret_cast<const float4*>(&buf[lane * kBufRow + i]);
    v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
  }
  __syncwarp();
}

// 32 rows of 16 values as bf16 to rows of ld, a multiple of 8; columns of a row are written in eights.
// Their column sums to sums[0 .. 15] where wanted.
__device__ __forceinline__ void write_summed(float* buf, const float (&v)[kCols], __nv_bfloat16* to, int64_t ld, int rows, int cols,
                                             float* sums) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kCols; i += 4)
    *reinterpret_cast<float4*>(&buf[lane * kBufRow + i]) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  __syncwarp();
  if (sums != nullptr) {  // (Rows that do not exist hold products with gradients of zero.)
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) s += buf[(2 * r + lane / kCols) * kBufRow + lane % kCols];
    s += __shfl_xor_sync(0xffffffffu, s, kCols);
    if (lane < cols) sums[lane] = s;
  }
  const int c = lane % 2 * 8;
#pragma unroll
  for (int it = 0; it < 2; ++it) {
    const int r = it * 16 + lane / 2;
    const float4 a = *reinterpret_cast<const float4*>(&buf[r * kBufRow + c]);
    const float4 b = *reinterpret_cast<const float4*>(&buf[r * kBufRow + c + 4]);
    uint4 q;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
    h[0] = __floats2bfloat162_rn(a.x, a.y);
    h[1] = __floats2bfloat162_rn(a.z, a.w);
    h[2] = __floats2bfloat162_rn(b.x, b.y);
    h[3] = __floats2bfloat162_rn(b.z, b.w);
    if (r < rows && c < cols) *reinterpret_cast<uint4*>(to + r * ld + c) = q;
  }
  __syncwarp();
}

// Result of one mode. BN: columns of the accumulator (kFwd: BN / 2 of u, then as many of g). PARTS: 1
// (bf16), or 3 (fp32; BN 128).
template <int MODE, int BN, int PARTS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmT, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const GemmParams p) {
  constexpr int ST = slots_of(BN), BYTES = slot_bytes(BN), ABYTES = kM * kK * 2;
  constexpr bool GATED = MODE == kFwd || MODE == kGate;  // u and g side by side
  constexpr bool A_MN = MODE == kDw, B_MN = !GATED;
  constexpr int CN = GATED ? BN / 2 : BN;               // columns of the result in a tile
  constexpr bool DRAINED = PARTS > 1 || MODE == kDw;    // sums leave tensor memory every RUN stages
  constexpr int RUN = PARTS > 1 ? kDrain : kRun;
  constexpr int COLS = (PARTS > 1 ? 4 : 2) * BN;        // of tensor memory: two accumulators, fp32 two more for the small products
  static_assert(COLS <= 512, "tensor memory");
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[ST], empty[ST], acc_full[2], acc_empty[2], small_full[2], small_empty[2], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ int dead;
  uint8_t* slot0 = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  float* bufs = reinterpret_cast<float*>(slot0 + ST * BYTES);
  // (Of the whole warp, and known to be: the loading and the issuing warp run their loops as one.)
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid / 32, 0), lane = tid & 31;
  const uint32_t rank = cluster_rank();
  if (tid == 0) {
    for (int s = 0; s < ST; ++s) {
      semx::tc::mbar_init(&full[s], 1);   // of CTA 0: both CTAs' copies
      semx::tc::mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      semx::tc::mbar_init(&acc_full[b], 1);
      semx::tc::mbar_init(&acc_empty[b], 2 * kEpi);  // of CTA 0: both CTAs' warps
      semx::tc::mbar_init(&small_full[b], 1);
      semx::tc::mbar_init(&small_empty[b], 2 * kEpi);
    }
    semx::tc::mbar_init(&drained, 1);
    dead = 0;
  }
  if (warp == 0) tmem_alloc_pair(&tmem_slot, COLS);
  semx::tc::fence_before_sync();
  __syncthreads();
  cluster_sync();
  semx::tc::fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  const int works = works_of(p), pair0 = blockIdx.x / 2, pairs = gridDim.x / 2;
  auto slice = [&](const Tile& t, int* k0, int* k1) {
    *k0 = (int)((int64_t)p.depth * t.split / t.of);
    *k1 = (int)((int64_t)p.depth * (t.split + 1) / t.of);
  };

  if (warp == kEpi) {
    // The warp runs the loop as one and one lane issues, so that what the copies take is in uniform
    // registers; no divisions in here: a stage is 512 cycles of products.
    const bool issues = elect_one();
    const uint32_t bars = in_cluster(&full[0], 0);
    uint32_t s = 0, phase = 1, issued = 0;
    bool ok = true;
    for (int w = pair0; w < works && ok; w += pairs) {
      const Tile t = tile_at(p, w);
      int k0, k1;
      slice(t, &k0, &k1);
      const int m0 = t.m * 2 * kM + (int)rank * kM, n0 = t.n * BN + (int)rank * (BN / 2);
      int kh = k0 >= p.khalf ? 1 : 0, kk = (k0 - kh * p.khalf) * kK;
      // Where each row of W is read once, tiles start their depth at different places: in step, all rows' addresses
      // would be the same but for the row (192 x 4096 -> 11008: 45.1 and 43.2 us).
      const bool turns = MODE == kFwd && PARTS == 1 && p.tiles_m == 1;
      if (turns) kk = (k0 + w * 5 % (k1 - k0)) * kK;
      for (int k = k0; k < k1 && ok; ++k) {
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          ok = __all_sync(0xffffffffu, wait_phase(&empty[s], phase, &dead));
          if (!ok) break;
          const uint32_t bar = bars + 8 * s;
          uint8_t *sa = slot0 + s * BYTES, *sb = sa + ABYTES;
          if (issues) {
            if (rank == 0) expect_bytes(&full[s], 2 * BYTES);
            if (MODE == kDw) {
#pragma unroll
              for (int b = 0; b < kM / 64; ++b) tma_load(sa + b * 8192, &map_a, m0 + b * 64, kk, t.half, part, bar);
#pragma unroll
              for (int b = 0; b < BN / 128; ++b) tma_load(sb + b * 8192, &map_b, n0 + b * 64, kk, 0, part, bar);
            } else if (MODE == kDx) {
              tma_load(sa, &map_a, kk, m0, kh, part, bar);
#pragma unroll
              for (int b = 0; b < BN / 128; ++b) tma_load(sb + b * 8192, &map_b, n0 + b * 64, kk, kh, part, bar);
            } else {  // CTA 0 brings u's rows of W, CTA 1 g's
              tma_load(sa, &map_a, kk, m0, 0, part, bar);
              tma_load(sb, &map_b, kk, t.n * CN, (int)rank, part, bar);
            }
          }
          __syncwarp();
          ++issued;
          if (++s == ST) s = 0, phase ^= 1;
        }
        kk += kK;
        if (turns && kk == k1 * kK) kk = k0 * kK;
        if (MODE == kDx && kk >= p.khalf * kK) kk = 0, ++kh;
      }
    }
    // After a wait that gave up: the copies on their way land before the CTAs end (CTA 0 sees both CTAs').
    if (!ok && rank == 0)
      for (uint32_t i = issued > ST ? issued - ST : 0; i < issued; ++i) wait_some(&full[i % ST], (i / ST) & 1, nullptr);
  } else if (warp == kEpi + 1) {
    if (rank == 0) {
      constexpr uint32_t idesc = idesc_bf16(2 * kM, BN, A_MN, B_MN);
      constexpr uint32_t a_step = (A_MN ? 2048 : 32), b_step = (B_MN ? 2048 : 32);  // 16 of the depth
      const bool issues = elect_one();
      const uint64_t desc_a = operand_desc<A_MN>(semx::tc::smem_addr(slot0)), desc_b = operand_desc<B_MN>(semx::tc::smem_addr(slot0) + ABYTES);
      uint32_t acc = 0, tiles = 0, s = 0, phase = 0;
      bool ok = true;
      auto multiply = [&](uint32_t d, uint32_t sa, uint32_t sb, bool accumulate) {
        const uint64_t a = desc_a + sa * (BYTES >> 4), b = desc_b + sb * (BYTES >> 4);
        if (issues) {
#pragma unroll
          for (int q = 0; q < 4; ++q) mma_pair(d, a + q * (a_step >> 4), b + q * (b_step >> 4), idesc, accumulate || q > 0);
        }
      };
      auto await = [&](uint64_t* bar, uint32_t parity) {
        ok = __all_sync(0xffffffffu, wait_phase(bar, parity, &dead));
        semx::tc::fence_after_sync();
        return ok;
      };
      auto done = [&](uint64_t* bar) {
        if (issues) commit_pair(bar);
        __syncwarp();
      };
      // The next slot, once its copies are there.
      auto next_slot = [&]() {
        const uint32_t at = s;
        await(&full[at], phase);
        if (++s == ST) s = 0, phase ^= 1;
        return at;
      };
      for (int w = pair0; w < works && ok; w += pairs, ++tiles) {
        const Tile t = tile_at(p, w);
        int k0, k1;
        slice(t, &k0, &k1);
        const uint32_t small = tmem + 2 * BN + (tiles & 1) * BN;
        if (PARTS > 1 && !await(&small_empty[tiles & 1], ((tiles >> 1) & 1) ^ 1)) break;
        const int drain = DRAINED ? RUN : k1 - k0;
        for (int c0 = k0; c0 < k1 && ok; c0 += drain, ++acc) {
          const uint32_t b = acc & 1, d = tmem + b * BN;
          if (!await(&acc_empty[b], ((acc >> 1) & 1) ^ 1)) break;
          const int c1 = min(k1, c0 + drain);
          for (int k = c0; k < c1; ++k) {
            const uint32_t s0 = next_slot();
            if (!ok) break;
            multiply(d, s0, s0, k > c0);
            if (PARTS > 1) {
              const uint32_t s1 = next_slot();
              if (!ok) break;
              multiply(small, s0, s1, k > k0);
              multiply(small, s1, s0, true);
              multiply(small, s1, s1, true);
              const uint32_t s2 = next_slot();
              if (!ok) break;
              multiply(small, s0, s2, true);
              multiply(small, s2, s0, true);
              done(&empty[s0]);
              done(&empty[s1]);
              done(&empty[s2]);
            } else {
              done(&empty[s0]);
            }
          }
          if (ok) done(&acc_full[b]);
        }
        if (PARTS > 1 && ok) done(&small_full[tiles & 1]);
      }
      if (!ok) {  // products on their way end before tensor memory is given back
        done(&drained);
        wait_some(&drained, 0, nullptr);
      }
    }
  } else {
    float* buf = bufs + warp * kBuf;
    const int quarter = warp % 4, side = warp / 4;  // rows; columns (which quarter of u's and g's, or of the tile)
    const uint32_t lanes = (uint32_t)quarter << 21;
    // Columns of the result that a warp has; of 32 the first eight warps have all.
    constexpr int WC = CN > 32 ? CN / 4 : 16;
    const bool idle = side * WC >= CN;
    constexpr int VALUES = GATED ? 2 * WC : WC;  // of the accumulator
    const uint32_t acc_e0 = in_cluster(&acc_empty[0], 0), acc_e1 = in_cluster(&acc_empty[1], 0);
    const uint32_t small_e0 = in_cluster(&small_empty[0], 0), small_e1 = in_cluster(&small_empty[1], 0);
    auto release = [&](uint32_t bar) {
      semx::tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) arrive_in_cluster(bar);
    };
    // Column (of the accumulator) of value i of this warp.
    auto column = [&](int i) { return GATED ? (i / WC) * CN + side * WC + i % WC : side * WC + i; };
    // What becomes of 16 columns from c of the result on: v (and g, kFwd).
    auto write = [&](const Tile& t, int c, float (&v)[kCols], float (&g)[kCols]) {
      const int64_t row0 = ((int64_t)t.m * 2 + rank) * kM + quarter * 32, col0 = (int64_t)t.n * CN + side * WC + c;
      const int rows = (int)max((int64_t)0, min((int64_t)32, p.M - row0)), cols = (int)max((int64_t)0, min((int64_t)kCols, p.N - col0));
      if (MODE == kGate && rows == 0 && p.sums != nullptr && lane < cols) {
        float* to = p.sums + (((int64_t)t.m * 2 + rank) * 4 + quarter) * 2 * p.N + col0 + lane;
        to[0] = to[p.N] = 0.f;
      }
      if (rows == 0 || cols == 0) return;
      if (t.of > 1) {
        float* to = p.part + ((int64_t)t.split * (p.tiles - p.whole) + t.index - p.whole) * (2 * kM * BN);
        const int row = (int)rank * kM + quarter * 32, col = side * WC + c;
        write_block(buf, v, to, BN, row, col, rows, kCols, 0);
        if (GATED) write_block(buf, g, to, BN, row, CN + col, rows, kCols, 0);
        return;
      }
      if constexpr (GATED) {
        if (p.bias != nullptr) {
          const float* at = buf + 32 * kBufRow + c;
#pragma unroll
          for (int i = 0; i < kCols; i += 4) {
            const float4 bu = *reinterpret_cast<const float4*>(at + i), bg = *reinterpret_cast<const float4*>(at + 32 + i);
            v[i] += bu.x; v[i + 1] += bu.y; v[i + 2] += bu.z; v[i + 3] += bu.w;
            g[i] += bg.x; g[i + 1] += bg.y; g[i + 2] += bg.z; g[i + 3] += bg.w;
          }
        }
        if constexpr (MODE == kGate) {
          float d[kCols];
          read_block(buf, d, p.dh, p.N, row0, col0, rows, cols);
          auto slopes = [&](auto gelu) {
#pragma unroll
            for (int i = 0; i < kCols; ++i) {
              float act, slope;
              act_and_slope(g[i], decltype(gelu)::value, &act, &slope);
              g[i] = d[i] * v[i] * slope;
              v[i] = d[i] * act;
            }
          };
          if (p.gelu) slopes(std::true_type());
          else slopes(std::false_type());
          float* to = p.sums == nullptr ? nullptr : p.sums + (((int64_t)t.m * 2 + rank) * 4 + quarter) * 2 * p.N + col0;
          const int64_t at = row0 * p.ldz + col0;
          write_summed(buf, v, p.dz + at, p.ldz, rows, cols, to);
          write_summed(buf, g, p.dz + p.M * p.ldz + at, p.ldz, rows, cols, to == nullptr ? nullptr : to + p.N);
          return;
        }
        if (p.u != nullptr) {
          write_block(buf, v, p.u, p.ldu, row0, col0, rows, cols, 0);
          write_block(buf, g, p.g, p.ldu, row0, col0, rows, cols, 0);
        }
        auto acts = [&](auto gelu) {
#pragma unroll
          for (int i = 0; i < kCols; ++i) v[i] *= act_of(g[i], decltype(gelu)::value);
        };
        if (p.gelu) acts(std::true_type());
        else acts(std::false_type());
        write_block(buf, v, p.out, p.ldo, row0, col0, rows, cols, p.out_bf16);
      } else {
        write_block(buf, v, p.out, p.ldo, (int64_t)t.half * p.M + row0, col0, rows, cols, p.out_bf16);
      }
    };
    // The biases of a tile, a lane per column: fetched while the tile before is written (when
    // the tile begins: 129684 x 64 -> 256 fp32 forward 131 us, so 118).
    static_assert(!GATED || WC <= 32, "biases");
    uint32_t bias_u = 0, bias_g = 0;
    auto fetch_bias = [&](const Tile& t) {
      const int64_t col = (int64_t)t.n * CN + side * WC + lane;
      const bool any = lane < WC && col < p.N;
      bias_u = any ? semx_scan::load_raw(p.bias, col, p.bias_bf16) : 0;
      bias_g = any ? semx_scan::load_raw(p.bias, p.N + col, p.bias_bf16) : 0;
    };
    uint32_t acc = 0, tiles = 0;
    if (GATED && p.bias != nullptr && pair0 < works) fetch_bias(tile_at(p, pair0));
    for (int w = pair0; w < works; w += pairs, ++tiles) {
      const Tile t = tile_at(p, w);
      if (GATED && p.bias != nullptr) {
        __syncwarp();
        buf[32 * kBufRow + lane] = semx_scan::as_float(bias_u, p.bias_bf16);
        buf[32 * kBufRow + 32 + lane] = semx_scan::as_float(bias_g, p.bias_bf16);
        __syncwarp();
        if (w + pairs < works) fetch_bias(tile_at(p, w + pairs));
      }
      if constexpr (!DRAINED) {
        const uint32_t b = acc & 1, d = tmem + b * BN + lanes;
        const bool ok = wait_phase(&acc_full[b], (acc >> 1) & 1, &dead);
        if (!__all_sync(0xffffffffu, ok)) break;
        semx::tc::fence_after_sync();
        if (idle) release(b ? acc_e1 : acc_e0);
#pragma unroll 1
        for (int c = 0; c < WC && !idle; c += GATED ? kCols : 2 * kCols) {
          float v[kCols], g[kCols];  // of u and g, or of 32 neighbours
          tmem_ld16_twice(d + column(c), d + column(GATED ? WC + c : c + kCols), v, g);
          if (c + (GATED ? 1 : 2) * kCols >= WC) release(b ? acc_e1 : acc_e0);
          write(t, c, v, g);
          if (!GATED) write(t, c + kCols, g, v);
        }
        ++acc;
      } else {
        int k0, k1;
        slice(t, &k0, &k1);
        float sum[VALUES];
        bool ok = true;
        auto drain = [&](auto first) {
          const uint32_t b = acc & 1, d = tmem + b * BN + lanes;
          ok = wait_phase(&acc_full[b], (acc >> 1) & 1, &dead);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) return;
          semx::tc::fence_after_sync();
#pragma unroll
          for (int i = 0; i < VALUES; i += 2 * kCols) {
            float v[kCols], y[kCols];
            tmem_ld16_twice(d + column(i), d + column(i + kCols), v, y);
#pragma unroll
            for (int j = 0; j < kCols; ++j) {
              sum[i + j] = decltype(first)::value ? v[j] : sum[i + j] + v[j];
              sum[i + kCols + j] = decltype(first)::value ? y[j] : sum[i + kCols + j] + y[j];
            }
          }
          release(b ? acc_e1 : acc_e0);
          ++acc;
        };
        drain(std::true_type());
        for (int c0 = k0 + RUN; c0 < k1 && ok; c0 += RUN) drain(std::false_type());
        if (!ok) break;
        if constexpr (PARTS > 1) {
          ok = wait_phase(&small_full[tiles & 1], (tiles >> 1) & 1, &dead);
          if (!__all_sync(0xffffffffu, ok)) break;
          semx::tc::fence_after_sync();
#pragma unroll
          for (int i = 0; i < VALUES; i += 2 * kCols) {
            float v[kCols], y[kCols];
            const uint32_t small = tmem + 2 * BN + (tiles & 1) * BN + lanes;
            tmem_ld16_twice(small + column(i), small + column(i + kCols), v, y);
#pragma unroll
            for (int j = 0; j < kCols; ++j) {
              sum[i + j] += v[j];
              sum[i + kCols + j] += y[j];
            }
          }
          release((tiles & 1) ? small_e1 : small_e0);
        }
#pragma unroll
        for (int c = 0; c < WC; c += kCols) {
          float v[kCols], g[kCols];
#pragma unroll
          for (int j = 0; j < kCols; ++j) {
            v[j] = sum[c + j];
            g[j] = GATED ? sum[WC + c + j] : 0.f;
          }
          write(t, c, v, g);
        }
      }
    }
  }
  semx::tc::fence_before_sync();
  __syncthreads();
  cluster_sync();  // neither CTA's barriers and shared memory end before the other is done with them
  semx::tc::fence_after_sync();
  if (warp == 0) tmem_dealloc_pair(tmem, COLS);
}

// Sums of the slices of a tile's depth, in their order, and what the epilogue does with them. A thread has
// four columns of a row of a tile, eight slices on their way at a time. Bound by the slices' bytes, most of them
// still in L2 (192 x 4096 -> 11008 4 us, the three of 8192 x 2048 -> 5504 in training 12).
template <int MODE>
__global__ void __launch_bounds__(256) join_kernel(const GemmParams p, int bn) {
  const int cn = MODE == kFwd ? bn / 2 : bn, across = cn / 4, sliced = p.tiles - p.whole;
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int i = (int)(n / (2 * kM * across)), in = (int)(n % (2 * kM * across)), r = in / across, c = in % across * 4;
  if (i >= sliced) return;
  const Tile t = tile_number(p, p.whole + i);
  const int64_t row = (int64_t)t.m * 2 * kM + r, col = (int64_t)t.n * cn + c;
  const int nn = (int)min((int64_t)4, p.N - col);
  if (row >= p.M || nn <= 0) return;
  float u[4] = {}, g[4] = {};
  const float* from = p.part + ((int64_t)i * (2 * kM) + r) * bn + c;
  const int64_t next = (int64_t)sliced * 2 * kM * bn;
  constexpr int AHEAD = MODE == kFwd ? 4 : 8;
  for (int k0 = 0; k0 < p.splits; k0 += AHEAD) {
    float4 a[AHEAD], b[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      a[k] = b[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k0 + k >= p.splits) continue;
      a[k] = __ldcs(reinterpret_cast<const float4*>(from + (k0 + k) * next));
      if (MODE == kFwd) b[k] = __ldcs(reinterpret_cast<const float4*>(from + (k0 + k) * next + cn));
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      u[0] += a[k].x; u[1] += a[k].y; u[2] += a[k].z; u[3] += a[k].w;
      g[0] += b[k].x; g[1] += b[k].y; g[2] += b[k].z; g[3] += b[k].w;
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k >= nn || MODE != kFwd) break;
    if (p.bias != nullptr) {
      u[k] += semx_scan::load(p.bias, col + k, p.bias_bf16);
      g[k] += semx_scan::load(p.bias, p.N + col + k, p.bias_bf16);
    }
    if (p.u != nullptr) {
      p.u[row * p.ldu + col + k] = u[k];
      p.g[row * p.ldu + col + k] = g[k];
    }
    u[k] *= act_of(g[k], p.gelu);
  }
  const int64_t at = ((int64_t)t.half * p.M + row) * p.ldo + col;
  const float4 v = make_float4(u[0], u[1], u[2], u[3]);
  if (nn == 4 && p.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & (p.out_bf16 ? 7 : 15)) == 0) {
    if (p.out_bf16) semx_scan::store_quad<semx_scan::kBf16>(p.out, at, 1, 4, v);
    else semx_scan::store_quad<semx_scan::kFp32>(p.out, at, 0, 4, v);
  } else {
    semx_scan::store_quad<semx_scan::kAny>(p.out, at, p.out_bf16, nn, v);
  }
}

// -- operands as the products read them -----------------------------------------------------------

// Rows to lay out: src at row stride ld, dst (parts, rows, ldp).
struct LaySource {
  const void* src;
  int64_t ld, rows;
  __nv_bfloat16* dst;
};
// cols values of each row of both into parts of bf16, ldp a multiple of 8; a thread has 8 neighbours. Columns
// behind the last one are left: the tensor map ends in front of them. Bound by HBM (fp32, 10 bytes per value: 22.5 M
// values 35 us, 6.4 TB/s).
__global__ void __launch_bounds__(256) lay_kernel(const LaySource one, const LaySource two, int bf16, int64_t cols, int64_t ldp, int parts) {
  const int64_t per = ldp / 8;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (one.rows + two.rows) * per; i += (int64_t)gridDim.x * 256) {
    const int64_t of_both = i / per, c = i % per * 8;
    const bool second = of_both >= one.rows;
    const void* src = second ? two.src : one.src;
    __nv_bfloat16* dst = second ? two.dst : one.dst;
    const int64_t row = second ? of_both - one.rows : of_both, rows = second ? two.rows : one.rows, ld = second ? two.ld : one.ld;
    float v[8];
    if (bf16) {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = c + k < cols ? semx_scan::load(src, row * ld + c + k, 1) : 0.f;
    } else {
      const float* s = reinterpret_cast<const float*>(src) + row * ld + c;
      if (c + 8 <= cols && (reinterpret_cast<uintptr_t>(s) & 15) == 0) {
        const float4 a = *reinterpret_cast<const float4*>(s), b = *reinterpret_cast<const float4*>(s + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = c + k < cols ? s[k] : 0.f;
      }
    }
    __align__(16) __nv_bfloat16 out[kParts][8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      __nv_bfloat16 q[kParts];
      parts_of(v[k], q);
#pragma unroll
      for (int n = 0; n < kParts; ++n) out[n][k] = q[n];
    }
#pragma unroll
    for (int n = 0; n < kParts; ++n)
      if (n < parts) *reinterpret_cast<uint4*>(dst + (n * rows + row) * ldp + c) = *reinterpret_cast<const uint4*>(out[n]);
  }
}

// du and dg from u, g (fp32, rows of ldu) and dh, as parts (PARTS, 2, rows, ldp). HBM is the bound: 129684 x 256
// fp32 131 us (6.1 TB/s), 8192 x 5504 bf16 107 (5.9). Column sums of 64
// rows each into sums (row blocks, 2 H) where wanted. A thread has 4 columns of every 4th row, two rows
// on their way at a time; CTAs side by side have columns side by side.
constexpr int kDzRows = 64;
template <int PARTS, bool GELU>
__global__ void __launch_bounds__(256, PARTS == 1 ? 4 : 3) gate_grad_kernel(const float* u, const float* g, int64_t ldu, const void* dh,
                                                        int64_t rows, int64_t H, __nv_bfloat16* dz, int64_t ldp,
                                                        float* sums) {
  constexpr bool BF16 = PARTS == 1;
  constexpr int ACC = BF16 ? semx_scan::kBf16 : semx_scan::kFp32, AHEAD = 2;
  __shared__ float red[2][4][256];
  const int lane = threadIdx.x % 64, down = threadIdx.x / 64;
  const unsigned across = (unsigned)((H + 255) / 256);
  const int64_t c0 = (int64_t)(blockIdx.x % across) * 256, block = blockIdx.x / across;
  const int64_t c = c0 + lane * 4, r0 = block * kDzRows;
  const int nn = (int)max((int64_t)0, min((int64_t)4, H - c)), most = (int)min((int64_t)kDzRows, rows - r0);
  const bool wide = H % 4 == 0 && (reinterpret_cast<uintptr_t>(dh) & (BF16 ? 7 : 15)) == 0;
  float su[4] = {}, sg[4] = {};
  if (nn > 0)
    for (int i0 = down; i0 < most; i0 += 4 * AHEAD) {
      float4 u4[AHEAD], g4[AHEAD];
      float d4[AHEAD][4];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int i = i0 + 4 * a;
        u4[a] = g4[a] = make_float4(0.f, 0.f, 0.f, 0.f);
        d4[a][0] = d4[a][1] = d4[a][2] = d4[a][3] = 0.f;
        if (i >= most) continue;
        const int64_t r = r0 + i;
        u4[a] = __ldcs(reinterpret_cast<const float4*>(u + r * ldu + c));
        g4[a] = __ldcs(reinterpret_cast<const float4*>(g + r * ldu + c));
        if (wide) {
          const float4 q = semx_scan::quad_floats<ACC>(semx_scan::load_quad<ACC>(dh, r * H + c, BF16, 4), BF16);
          d4[a][0] = q.x; d4[a][1] = q.y; d4[a][2] = q.z; d4[a][3] = q.w;
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < nn) d4[a][k] = semx_scan::load(dh, r * H + c + k, BF16);
        }
      }
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int i = i0 + 4 * a;
        if (i >= most) continue;
        const int64_t r = r0 + i;
        const float uu[4] = {u4[a].x, u4[a].y, u4[a].z, u4[a].w}, gg[4] = {g4[a].x, g4[a].y, g4[a].z, g4[a].w};
        __align__(8) __nv_bfloat16 pu[PARTS][4], pg[PARTS][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float act, slope;
          act_and_slope(gg[k], GELU, &act, &slope);
          const bool in = k < nn;
          const float du = in ? d4[a][k] * act : 0.f, dg = in ? d4[a][k] * uu[k] * slope : 0.f;
          su[k] += du;
          sg[k] += dg;
          if constexpr (BF16) {
            pu[0][k] = __float2bfloat16(du);
            pg[0][k] = __float2bfloat16(dg);
          } else {
            __nv_bfloat16 q[kParts];
            parts_of(du, q);
            for (int n = 0; n < kParts; ++n) pu[n][k] = q[n];
            parts_of(dg, q);
            for (int n = 0; n < kParts; ++n) pg[n][k] = q[n];
          }
        }
#pragma unroll
        for (int n = 0; n < PARTS; ++n) {
          *reinterpret_cast<uint2*>(dz + ((2 * n) * rows + r) * ldp + c) = *reinterpret_cast<const uint2*>(pu[n]);
          *reinterpret_cast<uint2*>(dz + ((2 * n + 1) * rows + r) * ldp + c) = *reinterpret_cast<const uint2*>(pg[n]);
        }
      }
    }
  if (sums == nullptr) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    red[0][down][lane * 4 + k] = su[k];
    red[1][down][lane * 4 + k] = sg[k];
  }
  __syncthreads();
  const int64_t cc = c0 + threadIdx.x;
  if (cc < H) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
      sums[block * 2 * H + n * H + cc] =
          red[n][0][threadIdx.x] + red[n][1][threadIdx.x] + red[n][2][threadIdx.x] + red[n][3][threadIdx.x];
  }
}

// -- few rows ---------------------------------------------------------------------------------

// Up to R rows of x. A warp has two columns (four rows of W); x lies in shared memory in fp32, kDepth
// values of each row at a time. Its lanes take 8 neighbouring weights of every 256. Bound by W's bytes for one or two
// rows, then by reading x from shared memory (fp32 2048 -> 5504: 1 row 15.2 us, 5.9 TB/s; 2 rows 16.3, 4 19.4, 8 33).
constexpr int kDepth = 2048, kFewT = 256, kFewBf16 = 16;
// Rows of fp32 that run so, eight at a time (16 x 2048 -> 5504: 67 us, tiles and the parts of W 89); of bf16 that
// the kernel below does not take.
constexpr int kFew = 8, kFewFp32 = 16;
// Place of value k in a row in shared memory: of every 256, the first halves of the lanes' eights, then
// the second ones, so that lanes side by side read side by side.
__device__ __forceinline__ int spread(int k) { return (k & ~255) | (k & 4) << 5 | (k & 248) >> 1 | (k & 3); }
template <int R, bool BF16, bool VEC>
__global__ void __launch_bounds__(kFewT, R > 4 ? 2 : 3) few_rows_kernel(const void* x, int64_t ldx, const void* w, int64_t D, int64_t H, int rows,
                                                         const GemmParams p) {
  extern __shared__ __align__(16) float xs[];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  const bool wide = ldx % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & (BF16 ? 7 : 15)) == 0;
  const int64_t h0 = ((int64_t)blockIdx.x * (kFewT / 32) + warp) * 2;
  semx_scan::f2 acc[4][R];
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[q][r] = semx_scan::pack2(0.f, 0.f);
  int64_t at[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) at[q] = (min(h0 + (q & 1), H - 1) + (q >> 1) * H) * D;
  for (int64_t d0 = 0; d0 < D; d0 += kDepth) {
    const int n = (int)min((int64_t)kDepth, D - d0), n8 = (n + 7) / 8 * 8;
    if (d0 > 0) __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t from = min(r, rows - 1) * ldx + d0;  // (rows that do not exist: the last one, and not written)
      for (int k = tid * 4; k < n8; k += kFewT * 4) {
        float4 v;
        if (k + 4 <= n && wide) {
          v = BF16 ? semx_scan::quad_floats<semx_scan::kBf16>(semx_scan::load_quad<semx_scan::kBf16>(x, from + k, 1, 4), 1)
                   : semx_scan::quad_floats<semx_scan::kFp32>(semx_scan::load_quad<semx_scan::kFp32>(x, from + k, 0, 4), 0);
        } else {
          v = semx_scan::quad_floats<semx_scan::kAny>(semx_scan::load_quad<semx_scan::kAny>(x, from + k, BF16, n - k), BF16);
        }
        *reinterpret_cast<float4*>(&xs[r * kDepth + spread(k)]) = v;
      }
    }
    __syncthreads();
    if (h0 < H)
#pragma unroll 1
      for (int k = lane * 8; k < n; k += 256) {
        semx_scan::f2 wv[4][4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t i = at[q] + d0 + k;
          float f[8];
          if constexpr (VEC && BF16) {
            const uint4 v = __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(w) + i));
            const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              f[2 * j] = __uint_as_float(e[j] << 16);
              f[2 * j + 1] = __uint_as_float(e[j] & 0xffff0000u);
            }
          } else if constexpr (VEC) {
            const float4 a = __ldcs(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(w) + i));
            const float4 b = __ldcs(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(w) + i + 4));
            f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
            f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = k + j < n ? semx_scan::load(w, i + j, BF16) : 0.f;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) wv[q][j] = semx_scan::pack2(f[2 * j], f[2 * j + 1]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float4 a = *reinterpret_cast<const float4*>(&xs[r * kDepth + spread(k)]);
          const float4 b = *reinterpret_cast<const float4*>(&xs[r * kDepth + spread(k) + 128]);
          const semx_scan::f2 xv[4] = {semx_scan::pack2(a.x, a.y), semx_scan::pack2(a.z, a.w), semx_scan::pack2(b.x, b.y),
                                       semx_scan::pack2(b.z, b.w)};
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[q][r] = semx_scan::fma2(wv[q][j], xv[j], acc[q][r]);
        }
      }
  }
  if (h0 >= H) return;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float2 s = semx_scan::unpack2(acc[q][r]);
      v[q] = s.x + s.y;
#pragma unroll
      for (int m = 16; m >= 1; m /= 2) v[q] += __shfl_xor_sync(0xffffffffu, v[q], m);
    }
    if (lane < 2 && r < rows && h0 + lane < H) {
      const int64_t h = h0 + lane;
      float u = lane ? v[1] : v[0], g = lane ? v[3] : v[2];
      if (p.bias != nullptr) {
        u += semx_scan::load(p.bias, h, p.bias_bf16);
        g += semx_scan::load(p.bias, H + h, p.bias_bf16);
      }
      if (p.u != nullptr) {
        p.u[r * p.ldu + h] = u;
        p.g[r * p.ldu + h] = g;
      }
      semx_scan::store(p.out, r * p.ldo + h, BF16, u * act_of(g, p.gelu));
    }
  }
}

// bf16 rows, up to 8 NT of them: products of 16 rows of W (eight of u, the same eight of g) by 16 of the depth
// by 8 rows of x. The depth may be taken in any order, so a lane's eight neighbouring weights (16 bytes) are
// its values of two products, and nothing of W passes through shared memory: each warp streams its rows.
// (tcgen05 would have tiles of 128 rows of x, nearly all of them empty.) Some warps share the depth of
// eight columns; their sums meet in shared memory.
// Bound by W's bytes: 1 row of 2048 -> 5504 9.2 us (4.9 TB/s), 8 of 4096 -> 11008 30.7 (5.9).
// Warps that share the depth (8 rows of 4096 -> 11008, four and eight: 31.8 and 30.7 us, 1 of 2048 -> 5504 11.6
// and 9.3; 16 rows 45.5 and 42.9, but 2048 -> 5504 11.8 and 15.6).
constexpr int few_warps(int nt) { return nt == 1 ? 8 : 4; }
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int NT>
__global__ void __launch_bounds__(few_warps(NT) * 32) few_rows_bf16_kernel(const __nv_bfloat16* x, int64_t ldx, const __nv_bfloat16* w, int64_t D,
                                                                       int64_t H, int rows, const GemmParams p) {
  constexpr int kFewWarps = few_warps(NT);
  __shared__ float sums[kFewWarps][NT * 8][17];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, q = lane / 4, t = lane % 4;
  const int64_t h0 = (int64_t)blockIdx.x * 8;
  // Lane (q, t): row q of u's and of g's eight, values 8 t .. 8 t + 7 of every 32 of the depth; of x row q.
  const __nv_bfloat16* wu = w + min(h0 + q, H - 1) * D + 8 * t;
  const __nv_bfloat16* wg = wu + H * D;
  const __nv_bfloat16* xr[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) xr[n] = x + min(n * 8 + q, rows - 1) * ldx + 8 * t;
  float c[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
  // D is a multiple of 8: a lane's eight values exist or do not.
  constexpr int AHEAD = 4;
  const int blocks = (int)((D + 31) / 32);  // of 32 of the depth; warp k has every kFewWarps-th run of AHEAD
  for (int b0 = warp * AHEAD; b0 < blocks; b0 += kFewWarps * AHEAD) {
    uint4 u[AHEAD], g[AHEAD], v[AHEAD][NT];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int64_t k = (int64_t)(b0 + a) * 32;
      const bool in = k + 8 * t < D;
      u[a] = in ? __ldcs(reinterpret_cast<const uint4*>(wu + k)) : make_uint4(0u, 0u, 0u, 0u);
      g[a] = in ? __ldcs(reinterpret_cast<const uint4*>(wg + k)) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int n = 0; n < NT; ++n) v[a][n] = in ? *reinterpret_cast<const uint4*>(xr[n] + k) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma_16x8x16(c[n], u[a].x, g[a].x, u[a].y, g[a].y, v[a][n].x, v[a][n].y);
        mma_16x8x16(c[n], u[a].z, g[a].z, u[a].w, g[a].w, v[a][n].z, v[a][n].w);
      }
  }
  // c[0], c[1]: u of column q for rows 2 t and 2 t + 1 of x; c[2], c[3]: g.
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      sums[warp][n * 8 + 2 * t + k][q] = c[n][k];
      sums[warp][n * 8 + 2 * t + k][8 + q] = c[n][2 + k];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 64; i += kFewWarps * 32) {
    const int r = i / 8, k = i % 8;
    const int64_t h = h0 + k;
    if (r >= rows || h >= H) continue;
    float uu = 0.f, gg = 0.f;
#pragma unroll
    for (int a = 0; a < kFewWarps; ++a) {
      uu += sums[a][r][k];
      gg += sums[a][r][8 + k];
    }
    if (p.bias != nullptr) {
      uu += semx_scan::load(p.bias, h, p.bias_bf16);
      gg += semx_scan::load(p.bias, H + h, p.bias_bf16);
    }
    if (p.u != nullptr) {
      p.u[r * p.ldu + h] = uu;
      p.g[r * p.ldu + h] = gg;
    }
    semx_scan::store(p.out, r * p.ldo + h, 1, uu * act_of(gg, p.gelu));
  }
}

// Whether the backward makes u and g again.
bool makes_again(const SemxGatedLinearArgs* a) { return a->bf16 && a->D <= 512; }

// -- host ---------------------------------------------------------------------------------------

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static std::atomic<void*> found{nullptr};
  void* f = found.load(std::memory_order_acquire);
  if (f == nullptr) {
    cudaDriverEntryPointQueryResult how;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &how) != cudaSuccess ||
        how != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    found.store(f, std::memory_order_release);
  }
  return reinterpret_cast<EncodeFn>(f);
}

// An operand in memory: (parts, halves, rows, cols) bf16 with 16-byte aligned rows.
struct Operand {
  const void* base;
  int64_t cols, rows, halves, parts;
  int64_t ld, half_stride, part_stride;  // elements
};

// box_rows: rows of a copy (64 columns each).
int make_map(CUtensorMap* map, const Operand& o, int box_rows) {
  EncodeFn encode = encode_fn();
  SEMX_REQUIRE(encode != nullptr, SEMX_ERR_UNSUPPORTED, "gated_linear: the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t dims[4] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)o.halves, (cuuint64_t)o.parts};
  const cuuint64_t strides[3] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(o.halves > 1 ? o.half_stride : o.ld) * 2,
                                 (cuuint64_t)(o.parts > 1 ? o.part_stride : o.ld) * 2};
  const cuuint32_t box[4] = {kK, (cuuint32_t)box_rows, 1, 1}, steps[4] = {1, 1, 1, 1};
  const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(o.base), dims, strides, box, steps,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  SEMX_REQUIRE(rc == CUDA_SUCCESS, SEMX_ERR_SHAPE, "gated_linear: cuTensorMapEncodeTiled refused %lld x %lld, stride %lld (%d)",
               (long long)o.rows, (long long)o.cols, (long long)o.ld, (int)rc);
  return SEMX_OK;
}

int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// What one product needs: tile width, slices of the depth, bytes of their sums.
struct Plan {
  int bn;
  GemmParams p;
  size_t part_bytes;
};

// Of a tile, in columns: what it costs beside them. Narrow tiles bring more of A per product (8192 x 5504 x
// 2048, 4 rounds of 256 columns or 7 of 128: 358 and 422 us).
constexpr int kTileCost = 96;

// M, N: the result; K: the depth of one half.
Plan plan_gemm(int mode, int64_t M, int64_t N, int64_t K, int parts) {
  Plan q = {};
  GemmParams& p = q.p;
  p.M = M;
  p.N = N;
  p.khalf = (int)cdiv(K, (int64_t)kK);
  p.depth = p.khalf * (mode == kDx ? 2 : 1);
  const bool gated = mode == kFwd || mode == kGate;
  const int64_t wide = gated ? 2 * N : N;
  const int64_t down = cdiv(M, (int64_t)2 * kM) * (mode == kDw ? 2 : 1);
  // The tile width that takes the least time in rounds of all pairs of SMs. (The operands read along the result need 128.)
  int64_t least = 0;
  for (int bn = 256; bn >= (mode == kFwd ? 64 : 128); bn /= 2) {
    if (parts > 1 && bn != 128) continue;
    const int64_t cost = cdiv(down * cdiv(wide, (int64_t)bn), (int64_t)kPairs) * (bn + kTileCost);
    if (q.bn == 0 || cost < least) q.bn = bn, least = cost;
  }
  p.tiles_m = (int)cdiv(M, (int64_t)2 * kM);
  p.tiles_n = (int)cdiv(wide, (int64_t)q.bn);
  p.tiles = p.tiles_m * p.tiles_n * (mode == kDw ? 2 : 1);
  // The last round's tiles run in slices of the depth where they leave half of the SMs idle or more, of 8
  // stages (fp32: 4, each of them six products) at least; behind whole rounds only where that saves more
  // than the kernel that adds the slices takes (192 x 4096 -> 11008, 172 tiles of 128 columns: 51 us, sliced 45 and 4.5 of
  // adding).
  const int last = p.tiles % kPairs;
  const int64_t stages = parts > 1 ? 4 : 8;
  int64_t s = last > 0 ? kPairs / last : 1;
  if (s > p.depth / stages) s = p.depth / stages;
  if (s < 1) s = 1;
  const bool pays = p.tiles < kPairs || p.depth - p.depth / s >= 4 * stages;
  p.splits = pays && mode != kGate ? (int)s : 1;
  p.whole = p.splits > 1 ? p.tiles - last : p.tiles;
  q.part_bytes = up256((size_t)p.splits * (p.tiles - p.whole) * 2 * kM * q.bn * sizeof(float));
  return q;
}

template <int MODE, int BN, int PARTS>
int launch_tiles(const Plan& q, const CUtensorMap& a, const CUtensorMap& b, int dev, cudaStream_t st) {
  // The limit stays with the kernel on a device: raised once (a bit for each of 64 devices).
  static std::atomic<uint64_t> raised{0};
  const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
  if ((raised.load(std::memory_order_relaxed) & bit) == 0) {
    if (!semx::allow_smem(gemm_kernel<MODE, BN, PARTS>, gemm_smem(BN))) return SEMX_ERR_LAUNCH;
    raised.fetch_or(bit, std::memory_order_relaxed);
  }
  const int works = works_of(q.p);
  gemm_kernel<MODE, BN, PARTS><<<2 * (works < kPairs ? works : kPairs), kGemmT, gemm_smem(BN), st>>>(a, b, q.p);
  return semx::check_launch("gated_linear gemm_kernel");
}

template <int MODE>
int launch_gemm(const Plan& q, const Operand& A, const Operand& B, cudaStream_t st) {
  // The driver's call wants a context of this thread, which a new thread (autograd's, say) has only after a
  // call of the runtime.
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess)
    return semx::fail(SEMX_ERR_DEVICE, "gated_linear: %s", cudaGetErrorString(cudaGetLastError()));
  CUtensorMap a, b;
  int rc = make_map(&a, A, MODE == kDw ? 64 : kM);
  if (rc != SEMX_OK) return rc;
  rc = make_map(&b, B, MODE == kFwd || MODE == kGate ? q.bn / 2 : 64);
  if (rc != SEMX_OK) return rc;
  if (A.parts > 1) {
    if constexpr (MODE != kGate) rc = launch_tiles<MODE, 128, kParts>(q, a, b, dev, st);
    else rc = semx::fail(SEMX_ERR_UNSUPPORTED, "gated_linear: fp32 keeps u and g");
  } else if (q.bn == 256) {
    rc = launch_tiles<MODE, 256, 1>(q, a, b, dev, st);
  } else if (q.bn == 128) {
    rc = launch_tiles<MODE, 128, 1>(q, a, b, dev, st);
  } else {
    if constexpr (MODE == kFwd) rc = launch_tiles<MODE, 64, 1>(q, a, b, dev, st);
    else rc = semx::fail(SEMX_ERR_UNSUPPORTED, "gated_linear: tile of %d", q.bn);
  }
  if (rc != SEMX_OK || q.p.whole == q.p.tiles || MODE == kGate) return rc;
  const int64_t quads = (int64_t)(q.p.tiles - q.p.whole) * 2 * kM * (MODE == kFwd ? q.bn / 2 : q.bn) / 4;
  if constexpr (MODE != kGate) join_kernel<MODE><<<(unsigned)cdiv(quads, (int64_t)256), 256, 0, st>>>(q.p, q.bn);
  return semx::check_launch("gated_linear join_kernel");
}

int gl_check_sizes(const SemxGatedLinearArgs* a) {
  const int64_t top = (int64_t)1 << 31;
  SEMX_REQUIRE(a->rows >= 0 && a->rows < top && a->D >= 1 && a->D < (1 << 23) && a->H >= 1 && a->H < (1 << 23),
               SEMX_ERR_SHAPE, "gated_linear: rows=%lld, D=%lld, H=%lld", (long long)a->rows, (long long)a->D, (long long)a->H);
  SEMX_REQUIRE(a->ldx >= a->D && a->ldx < top, SEMX_ERR_SHAPE, "gated_linear: row stride %lld for %lld columns",
               (long long)a->ldx, (long long)a->D);
  SEMX_REQUIRE(a->act == 0 || a->act == 1, SEMX_ERR_UNSUPPORTED, "gated_linear: activation %d", a->act);
  // Tiles and their numbers fit 31 bits.
  SEMX_REQUIRE(cdiv(a->rows, (int64_t)64) * cdiv(a->H > a->D ? a->H : a->D, (int64_t)32) < ((int64_t)1 << 30) &&
                   cdiv(a->D, (int64_t)64) * cdiv(a->H, (int64_t)32) < ((int64_t)1 << 30) &&
                   cdiv(a->rows, (int64_t)kK) * 6 < top,
               SEMX_ERR_SHAPE, "gated_linear: rows=%lld, D=%lld, H=%lld", (long long)a->rows, (long long)a->D, (long long)a->H);
  return SEMX_OK;
}
int gl_check(const SemxGatedLinearArgs* a, bool bwd) {
  const int rc = gl_check_sizes(a);
  if (rc != SEMX_OK) return rc;
  if (a->rows == 0 && !bwd) return SEMX_OK;
  SEMX_REQUIRE(a->w && (a->rows == 0 || a->x), SEMX_ERR_NULL, "gated_linear: x / w is NULL");
  if (!bwd) SEMX_REQUIRE(a->h, SEMX_ERR_NULL, "gated_linear: h is NULL");
  else SEMX_REQUIRE(a->rows == 0 || (a->dh && (makes_again(a) || a->saved)), SEMX_ERR_NULL, "gated_linear bwd: dh / saved is NULL");
  SEMX_REQUIRE(semx::all_aligned({a->x, a->w, a->h, a->dh, a->dx, a->dw}, a->bf16 ? 2 : 4) &&
                   semx::aligned(a->bias, a->bias_bf16 ? 2 : 4) && semx::aligned(a->db, 4) &&
                   semx::all_aligned({a->saved, a->workspace}, 16),
               SEMX_ERR_ALIGN, "gated_linear: a pointer is not on an element");
  return SEMX_OK;
}

// Whether TMA reads rows of n bf16 at stride ld from base. (A size query may leave a base open: it could be anywhere.)
bool on_16(const void* base) { return base != nullptr && semx::aligned(base, 16); }
bool in_place(const void* base, int64_t ld, int bf16) { return bf16 && ld % 8 == 0 && on_16(base); }

template <int NT>
int launch_few_bf16(const SemxGatedLinearArgs* a, const GemmParams& p, cudaStream_t st) {
  few_rows_bf16_kernel<NT><<<(unsigned)cdiv(a->H, (int64_t)8), few_warps(NT) * 32, 0, st>>>(
      reinterpret_cast<const __nv_bfloat16*>(a->x), a->ldx, reinterpret_cast<const __nv_bfloat16*>(a->w), a->D, a->H, (int)a->rows, p);
  return semx::check_launch("gated_linear few_rows_bf16_kernel");
}

// Workspace of one call: parts of x, of W, of du | dg, sums of slices, column sums.
struct Layout {
  int parts;
  bool few, few_bf16, lay_x, lay_w;
  int64_t sum_rows;
  size_t x, w, dz, part, sums, total;
  bool again;  // backward: u and g are made again
  Plan fwd, dx, dw;
};

Layout layout_of(const SemxGatedLinearArgs* a, bool bwd) {
  Layout l = {};
  l.parts = a->bf16 ? 1 : kParts;
  // (Rows that the wide loads take.)
  l.few_bf16 = !bwd && a->bf16 && a->rows <= kFewBf16 && a->D % 8 == 0 && (a->ldx % 8 == 0 || a->rows == 1) &&
               on_16(a->x) && on_16(a->w);
  l.few = !bwd && a->rows <= (a->bf16 ? kFew : kFewFp32) && !l.few_bf16;
  if (a->rows == 0 || l.few || l.few_bf16) return l;
  // Laid out anew where TMA cannot read them, which depends on the addresses too: hence workspace_bytes.
  l.lay_x = !in_place(a->x, a->ldx, a->bf16);
  l.lay_w = !in_place(a->w, a->D, a->bf16);
  const int64_t Dp = up8(a->D), Hp = up8(a->H);
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t was = at;
    at += up256(bytes);
    return was;
  };
  l.again = bwd && makes_again(a);
  const bool need_x = !bwd || l.again || a->dw != nullptr, need_w = !bwd || l.again || a->dx != nullptr;
  l.x = take(l.lay_x && need_x ? (size_t)l.parts * a->rows * Dp * 2 : 0);
  l.w = take(l.lay_w && need_w ? (size_t)l.parts * 2 * a->H * Dp * 2 : 0);
  if (!bwd) {
    l.fwd = plan_gemm(kFwd, a->rows, a->H, a->D, l.parts);
    l.part = take(l.fwd.part_bytes);
  } else {
    l.dz = take((size_t)l.parts * 2 * a->rows * Hp * 2);
    l.dx = plan_gemm(kDx, a->rows, a->D, a->H, l.parts);
    l.dw = plan_gemm(kDw, a->H, a->D, a->rows, l.parts);
    if (l.again) l.fwd = plan_gemm(kGate, a->rows, a->H, a->D, l.parts);
    const size_t p1 = a->dx != nullptr ? l.dx.part_bytes : 0, p2 = a->dw != nullptr ? l.dw.part_bytes : 0;
    l.part = take(p1 > p2 ? p1 : p2);
    l.sum_rows = l.again ? 8 * l.fwd.p.tiles_m : cdiv(a->rows, (int64_t)kDzRows);
    l.sums = take(a->db != nullptr ? (size_t)l.sum_rows * 2 * a->H * sizeof(float) : 0);
  }
  l.total = at;
  return l;
}

int gl_check_workspace(const SemxGatedLinearArgs* a, const Layout& l) {
  SEMX_REQUIRE(l.total == 0 || (a->workspace != nullptr && a->workspace_bytes >= (int64_t)l.total), SEMX_ERR_WORKSPACE,
               "gated_linear: a workspace of %lld bytes where the call needs %zu", (long long)(a->workspace ? a->workspace_bytes : 0),
               l.total);
  return SEMX_OK;
}

template <int R>
int launch_few(const SemxGatedLinearArgs* a, const GemmParams& p, cudaStream_t st) {
  const size_t smem = (size_t)R * kDepth * sizeof(float);
  const unsigned grid = (unsigned)cdiv(a->H, (int64_t)(kFewT / 32) * 2);
  const int rows = (int)a->rows;
  const bool vec = a->D % 8 == 0 && semx::aligned(a->w, 16);
#define SEMX_FEW(B, V)                                                                                      \
  do {                                                                                                      \
    if (!semx::allow_smem(few_rows_kernel<R, B, V>, smem)) return SEMX_ERR_LAUNCH;                          \
    few_rows_kernel<R, B, V><<<grid, kFewT, smem, st>>>(a->x, a->ldx, a->w, a->D, a->H, rows, p);           \
  } while (0)
  if (a->bf16) {
    if (vec) SEMX_FEW(true, true);
    else SEMX_FEW(true, false);
  } else {
    if (vec) SEMX_FEW(false, true);
    else SEMX_FEW(false, false);
  }
#undef SEMX_FEW
  return semx::check_launch("gated_linear few_rows_kernel");
}

// x and W as the products read them.
int lay_operands(const SemxGatedLinearArgs* a, const Layout& l, bool need_x, bool need_w, char* ws, cudaStream_t st, Operand* x,
                 Operand* w) {
  const int64_t Dp = up8(a->D);
  *x = Operand{a->x, a->D, a->rows, 1, 1, a->ldx, 0, 0};
  *w = Operand{a->w, a->D, a->H, 2, 1, a->D, a->H * a->D, 0};
  LaySource one = {}, two = {};
  if (need_x && l.lay_x) {
    one = LaySource{a->x, a->ldx, a->rows, reinterpret_cast<__nv_bfloat16*>(ws + l.x)};
    *x = Operand{ws + l.x, a->D, a->rows, 1, l.parts, Dp, 0, a->rows * Dp};
  }
  if (need_w && l.lay_w) {
    two = LaySource{a->w, a->D, 2 * a->H, reinterpret_cast<__nv_bfloat16*>(ws + l.w)};
    *w = Operand{ws + l.w, a->D, a->H, 2, l.parts, Dp, a->H * Dp, 2 * a->H * Dp};
  }
  if (one.rows + two.rows == 0) return SEMX_OK;
  const int64_t n = cdiv((one.rows + two.rows) * (Dp / 8), (int64_t)256);
  lay_kernel<<<(unsigned)(n < kSms * 16 ? n : kSms * 16), 256, 0, st>>>(one, two, a->bf16, a->D, Dp, l.parts);
  return semx::check_launch("gated_linear lay_kernel");
}

}  // namespace

namespace semx {
int gemm_timeouts(uint32_t* count) {
  unsigned v = 0;
  const cudaError_t e = cudaMemcpyFromSymbol(&v, g_gemm_timeouts, sizeof(v));
  if (e != cudaSuccess) return fail(SEMX_ERR_LAUNCH, "gemm_timeouts: %s", cudaGetErrorString(e));
  *count = v;
  return SEMX_OK;
}
}  // namespace semx

extern "C" {

size_t semx_gated_linear_args_size(void) { return sizeof(SemxGatedLinearArgs); }

size_t semx_gated_linear_saved_bytes(const SemxGatedLinearArgs* a) {
  if (a == nullptr || a->rows < 0 || a->H < 0) return 0;
  // Narrow bf16 rows: the backward makes u and g again in less time than it takes to write and read them
  // (training passes, kept and made again: 129684 x 64 -> 256 241 and 199 us, 16384 x 512 -> 1408 226 and 213,
  // 8192 x 1024 -> 2752 299 and 314). In fp32, six times the products and three parts to write, it does not
  // (129684 x 64 -> 256 462 and 549).
  if (makes_again(a)) return 0;
  return (size_t)2 * a->rows * up8(a->H) * sizeof(float);
}

size_t semx_gated_linear_workspace_bytes(const SemxGatedLinearArgs* a, int32_t backward) {
  if (a == nullptr || gl_check_sizes(a) != SEMX_OK) return 0;
  return layout_of(a, backward != 0).total;
}

int semx_gated_linear_fwd(const SemxGatedLinearArgs* a, semx_stream_t stream) {
  SEMX_CHECK_ARGS(a, SemxGatedLinearArgs);
  int rc = gl_check(a, false);
  if (rc != SEMX_OK || a->rows == 0) return rc;
  const Layout l = layout_of(a, false);
  rc = gl_check_workspace(a, l);
  if (rc != SEMX_OK) return rc;
  semx::DeviceScope scope;
  rc = scope.bind({a->h});
  if (rc != SEMX_OK) return rc;
  cudaStream_t st = semx::as_stream(stream);
  Plan q = l.fwd;
  q.p.out = a->h;
  q.p.ldo = a->H;
  q.p.out_bf16 = a->bf16;
  q.p.ldu = up8(a->H);
  q.p.u = a->saved;
  q.p.g = a->saved == nullptr ? nullptr : a->saved + a->rows * q.p.ldu;
  q.p.bias = a->bias;
  q.p.bias_bf16 = a->bias_bf16;
  q.p.gelu = a->act;
  if (l.few_bf16) {
    const int tiles = (int)cdiv(a->rows, (int64_t)8);
    if (tiles == 1) return launch_few_bf16<1>(a, q.p, st);
    return launch_few_bf16<2>(a, q.p, st);
  }
  if (l.few) {
    SemxGatedLinearArgs part = *a;
    for (int64_t r = 0; r < a->rows; r += kFew) {
      const int64_t e = a->bf16 ? 2 : 4;
      part.rows = a->rows - r < kFew ? a->rows - r : kFew;
      part.x = reinterpret_cast<const char*>(a->x) + r * a->ldx * e;
      GemmParams p = q.p;
      p.out = reinterpret_cast<char*>(a->h) + r * a->H * e;
      if (p.u != nullptr) p.u += r * p.ldu, p.g += r * p.ldu;
      rc = part.rows == 1 ? launch_few<1>(&part, p, st)
           : part.rows == 2 ? launch_few<2>(&part, p, st)
           : part.rows <= 4 ? launch_few<4>(&part, p, st) : launch_few<8>(&part, p, st);
      if (rc != SEMX_OK) return rc;
    }
    return SEMX_OK;
  }
  char* ws = reinterpret_cast<char*>(a->workspace);
  q.p.part = reinterpret_cast<float*>(ws + l.part);
  Operand x, w;
  rc = lay_operands(a, l, true, true, ws, st, &x, &w);
  if (rc != SEMX_OK) return rc;
  return launch_gemm<kFwd>(q, x, w, st);
}

int semx_gated_linear_bwd(const SemxGatedLinearArgs* a, semx_stream_t stream) {
  SEMX_CHECK_ARGS(a, SemxGatedLinearArgs);
  int rc = gl_check(a, true);
  if (rc != SEMX_OK) return rc;
  const bool need_x = a->dw != nullptr, need_w = a->dx != nullptr;
  if (!need_x && !need_w && a->db == nullptr) return SEMX_OK;
  const Layout l = layout_of(a, true);
  rc = gl_check_workspace(a, l);
  if (rc != SEMX_OK) return rc;
  semx::DeviceScope scope;
  rc = scope.bind({a->dw, a->dx, a->db});
  if (rc != SEMX_OK) return rc;
  cudaStream_t st = semx::as_stream(stream);
  if (a->rows == 0) {
    cudaError_t e = cudaSuccess;
    if (a->dw != nullptr) e = cudaMemsetAsync(a->dw, 0, (size_t)2 * a->H * a->D * (a->bf16 ? 2 : 4), st);
    if (e == cudaSuccess && a->db != nullptr) e = cudaMemsetAsync(a->db, 0, (size_t)2 * a->H * sizeof(float), st);
    SEMX_REQUIRE(e == cudaSuccess, SEMX_ERR_LAUNCH, "gated_linear bwd: cudaMemsetAsync: %s", cudaGetErrorString(e));
    return SEMX_OK;
  }
  char* ws = reinterpret_cast<char*>(a->workspace);
  const int64_t Hp = up8(a->H);
  float* sums = a->db != nullptr ? reinterpret_cast<float*>(ws + l.sums) : nullptr;
  __nv_bfloat16* dz = reinterpret_cast<__nv_bfloat16*>(ws + l.dz);
  Operand x, w;
  rc = lay_operands(a, l, need_x || l.again, need_w || l.again, ws, st, &x, &w);
  if (rc != SEMX_OK) return rc;
  if (l.again) {
    Plan q = l.fwd;
    q.p.dh = a->dh;
    q.p.dz = dz;
    q.p.ldz = Hp;
    q.p.sums = sums;
    q.p.bias = a->bias;
    q.p.bias_bf16 = a->bias_bf16;
    q.p.gelu = a->act;
    rc = launch_gemm<kGate>(q, x, w, st);
  } else {
    const float *u = a->saved, *g = a->saved + a->rows * Hp;
    const unsigned grid = (unsigned)(cdiv(a->rows, (int64_t)kDzRows) * cdiv(a->H, (int64_t)256));
    auto* kernel = a->bf16 ? (a->act ? gate_grad_kernel<1, true> : gate_grad_kernel<1, false>)
                           : (a->act ? gate_grad_kernel<kParts, true> : gate_grad_kernel<kParts, false>);
    kernel<<<grid, 256, 0, st>>>(u, g, Hp, a->dh, a->rows, a->H, dz, Hp, sums);
    rc = semx::check_launch("gated_linear gate_grad_kernel");
  }
  if (rc != SEMX_OK) return rc;
  const Operand d = {dz, a->H, a->rows, 2, l.parts, Hp, a->rows * Hp, 2 * a->rows * Hp};
  if (need_w) {
    Plan q = l.dx;
    q.p.out = a->dx;
    q.p.ldo = a->D;
    q.p.out_bf16 = a->bf16;
    q.p.part = reinterpret_cast<float*>(ws + l.part);
    rc = launch_gemm<kDx>(q, d, w, st);
    if (rc != SEMX_OK) return rc;
  }
  if (need_x) {
    Plan q = l.dw;
    q.p.out = a->dw;
    q.p.ldo = a->D;
    q.p.out_bf16 = a->bf16;
    q.p.part = reinterpret_cast<float*>(ws + l.part);
    rc = launch_gemm<kDw>(q, d, x, st);
    if (rc != SEMX_OK) return rc;
  }
  if (a->db == nullptr) return SEMX_OK;
  semx::Segments seg = {};
  seg.n = 1;
  seg.out[0] = a->db;
  seg.len[0] = 2 * a->H;
  return semx::colsum_once(sums, l.sum_rows, 2 * a->H, seg, st);
}

}  // extern "C"
