// Layer normalisation over the last dimension, with the residual added first when one is
// given, forward and backward, for sm_100a.
//
//   s = x + r (rounded to the type it is stored in), mean = sum(s) / d,
//   rstd = 1 / sqrt(sum((s - mean)^2) / d + eps), xhat = (s - mean) rstd,
//   y = xhat w + b
//   g = dy w, ds += rstd (g - mean(g) - xhat mean(g xhat)); dx = dr = ds,
//   dw = sum_rows dy xhat, db = sum_rows dy
//
// Bound: HBM. Forward reads x (and r) once and writes y (and s) once; backward reads s, dy
// (and the gradient of s) once and writes dx (and dr) once. A row therefore stays in the
// registers of its TPR threads (8 V elements each) between the statistics and the result,
// and a CTA walks over many rows so that the sums dw, db stay in registers too, and w and b
// where a row is narrow (keeps_params).
// The statistics are two-step (mean, then squares about it): a warp does both by shuffles,
// and the warps of a wide row join their (mean, squares) pairs with the exact update for
// the mean of two samples, so a wide row costs one barrier. All arithmetic is fp32.
// dw and db: each thread adds its columns over the CTA's rows, the row slots of a CTA are
// joined in slot order in shared memory, and the CTAs' rows by the fixed-order column sum,
// so the result does not depend on the order in which CTAs run.
#include <cuda_bf16.h>

#include "semx_common.cuh"
#include "semx_reduce.cuh"

namespace {

constexpr int kMaxD = 32768;

struct LnParams {
  int64_t n;
  int d;
  float eps;
  int x_bf16, r_bf16, y_bf16, s_bf16;
  const void* x;
  const void* r;  // residual or NULL
  const float* w;  // or NULL: 1
  const float* b;  // or NULL: 0
  void* y;
  void* s;  // the sum: forward output, NULL without a residual
  float* mean;
  float* rstd;
  // backward: x is the normalised tensor (type s_bf16)
  const void* dy;
  const void* ds;
  void* dx;
  void* dr;
  float* part;  // (CTAs, 2 d): dw | db
};

// Element i of thread t of a row: VEC takes groups of 8 neighbours (16-byte accesses of
// bf16), otherwise neighbouring threads take neighbouring elements.
template <int TPR, bool VEC>
__device__ __forceinline__ int col(int t, int i) {
  return VEC ? ((i >> 3) * TPR + t) * 8 + (i & 7) : i * TPR + t;
}

// A thread's part of a row as it is stored: loaded a row ahead, converted when it is used.
template <int V>
struct RawRow {
  uint4 q[2 * V];
};

template <int TPR, int V, bool VEC>
__device__ __forceinline__ void load_row(const void* base, int64_t off, int bf16, int t, int d, RawRow<V>& r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r.q);
  if (VEC) {
    if (bf16) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int c = col<TPR, VEC>(t, 8 * k);
        r.q[k] = make_uint4(0, 0, 0, 0);
        if (c < d) r.q[k] = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(base) + off + c);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 2 * V; ++k) {
        const int c = col<TPR, VEC>(t, 4 * k);
        r.q[k] = make_uint4(0, 0, 0, 0);
        if (c < d) r.q[k] = *reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(base) + off + c);
      }
    }
  } else if (bf16) {
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) {
      const int c = col<TPR, VEC>(t, i);
      u[i] = c < d ? (uint32_t) reinterpret_cast<const unsigned short*>(base)[off + c] : 0u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) {
      const int c = col<TPR, VEC>(t, i);
      u[i] = c < d ? reinterpret_cast<const uint32_t*>(base)[off + c] : 0u;
    }
  }
}

template <int V, bool VEC>
__device__ __forceinline__ void to_floats(const RawRow<V>& r, int bf16, float (&v)[8 * V]) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(r.q);
  if (VEC && bf16) {
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) v[i] = __uint_as_float(bf16 ? u[i] << 16 : u[i]);
  }
}

template <int TPR, int V, bool VEC>
__device__ __forceinline__ void store_row(void* base, int64_t off, int bf16, int t, int d, const float (&v)[8 * V]) {
  if (VEC) {
    if (bf16) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int c = col<TPR, VEC>(t, 8 * k);
        if (c < d) {
          uint4 q;
          __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
          for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[8 * k + 2 * j], v[8 * k + 2 * j + 1]);
          *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(base) + off + c) = q;
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 2 * V; ++k) {
        const int c = col<TPR, VEC>(t, 4 * k);
        if (c < d)
          *reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + off + c) =
              make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) {
      const int c = col<TPR, VEC>(t, i);
      if (c < d) {
        if (bf16) reinterpret_cast<__nv_bfloat16*>(base)[off + c] = __float2bfloat16(v[i]);
        else reinterpret_cast<float*>(base)[off + c] = v[i];
      }
    }
  }
}

// Parameters of the thread's 8 V columns (0 beyond the row, `none` where there is no parameter).
template <int TPR, int V, bool VEC>
__device__ __forceinline__ void load_param(const float* p, int t, int d, float none, float (&v)[8 * V]) {
  if (VEC) {
#pragma unroll
    for (int k = 0; k < 2 * V; ++k) {
      const int c = col<TPR, VEC>(t, 4 * k);
      float4 q = make_float4(none, none, none, none);
      if (p != nullptr) q = c < d ? *reinterpret_cast<const float4*>(p + c) : make_float4(0.f, 0.f, 0.f, 0.f);
      v[4 * k] = q.x; v[4 * k + 1] = q.y; v[4 * k + 2] = q.z; v[4 * k + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) {
      const int c = col<TPR, VEC>(t, i);
      v[i] = p == nullptr ? none : c < d ? p[c] : 0.f;
    }
  }
}

// Rows of at most 512 elements keep the parameters in registers from row to row; wider ones
// read them again from L1, which leaves registers for the row that is on its way.
template <int TPR>
constexpr bool keeps_params() {
  return TPR <= 32;
}
// Whether the next row is loaded while this one is worked on: not where a thread's part of
// a row is so long that it would spill.
template <int TPR, int V>
constexpr bool loads_ahead() {
  return V <= 2 || TPR <= 32;
}
template <int TPR>
constexpr int cta_threads() {
  return TPR < 128 ? 128 : TPR;
}
// CTAs per SM that the registers are cut for: what a launch puts there (ln_ctas) at most. Cut for eight
// where four are launched, rows of 513 to 1024 elements spilled (64 M elements of 1024 fp32: forward 152
// us, cut for four 134; backward 293 and 173).
template <int TPR, int V>
constexpr int ctas_per_sm() {
  return TPR * V <= 256 ? 4 : TPR * V <= 1024 ? 1024 / (TPR * V) : 1;
}

template <int W>
__device__ __forceinline__ float lane_sum(float v) {
#pragma unroll
  for (int m = W / 2; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// Elements of a row of d that warp q of its TPR threads holds.
template <int TPR, int V, bool VEC>
__device__ __forceinline__ int warp_count(int q, int d) {
  int n = 0;
  constexpr int kRun = VEC ? 32 * 8 : 32;  // neighbours per warp and step
  constexpr int kStep = VEC ? TPR * 8 : TPR;
#pragma unroll
  for (int k = 0; k < (VEC ? V : 8 * V); ++k) n += max(0, min(kRun, d - (k * kStep + q * kRun)));
  return n;
}

template <int TPR, int V, bool VEC>
__global__ void __launch_bounds__(cta_threads<TPR>(), ctas_per_sm<TPR, V>()) layer_norm_fwd_kernel(const LnParams p) {
  constexpr int NT = TPR < 128 ? 128 : TPR;
  constexpr int ROWS = NT / TPR;
  constexpr int LW = TPR < 32 ? TPR : 32;  // lanes of a warp that share a row
  constexpr int WPR = TPR / LW;            // warps that share a row
  __shared__ float2 red[2][WPR];
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR, d = p.d;
  float w[8 * V], b[8 * V];
  if (keeps_params<TPR>()) {
    load_param<TPR, V, VEC>(p.w, t, d, 1.f, w);
    load_param<TPR, V, VEC>(p.b, t, d, 0.f, b);
  }
  const float inv_d = 1.f / (float)d;
  // Elements of a row that this warp holds, and those of the warp that this lane joins.
  const int lane = threadIdx.x & 31;
  const float own_inv = WPR == 1 ? inv_d : 1.f / (float)max(1, warp_count<TPR, V, VEC>(t / 32, d));
  const float lane_n = lane < WPR ? (float)warp_count<TPR, V, VEC>(lane, d) : 0.f;
  const float lane_inv = lane_n > 0.f ? 1.f / lane_n : 0.f;
  int par = 0;
  RawRow<V> nx, nr;
  auto fetch = [&](int64_t row) {
    const int dd = row < p.n ? d : 0;  // a slot behind the last row loads and stores nothing
    load_row<TPR, V, VEC>(p.x, row * d, p.x_bf16, t, dd, nx);
    if (p.r != nullptr) load_row<TPR, V, VEC>(p.r, row * d, p.r_bf16, t, dd, nr);
  };
  const int64_t hop = (int64_t)gridDim.x * ROWS;
  fetch((int64_t)blockIdx.x * ROWS + slot);
  for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < p.n; r0 += hop, par ^= 1) {
    const int64_t row = r0 + slot;
    const bool ok = row < p.n;
    const int dd = ok ? d : 0;
    const int64_t off = row * d;
    float v[8 * V], r[8 * V];
    to_floats<V, VEC>(nx, p.x_bf16, v);
    if (p.r != nullptr) to_floats<V, VEC>(nr, p.r_bf16, r);
    if (loads_ahead<TPR, V>() && r0 + hop < p.n) fetch(row + hop);
    if (p.r != nullptr) {
#pragma unroll
      for (int i = 0; i < 8 * V; ++i) {
        v[i] += r[i];
        // The norm is that of the sum as it is stored, which is what the backward reads.
        if (p.s_bf16) v[i] = __bfloat162float(__float2bfloat16(v[i]));
      }
      store_row<TPR, V, VEC>(p.s, off, p.s_bf16, t, dd, v);
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) sum += v[i];
    sum = lane_sum<LW>(sum);
    float mean = sum * own_inv, sq = 0.f;
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) {
      const float e = col<TPR, VEC>(t, i) < d ? v[i] - mean : 0.f;
      sq = fmaf(e, e, sq);
    }
    sq = lane_sum<LW>(sq);
    if (WPR > 1) {
      if ((t & 31) == 0) red[par][t / 32] = make_float2(sum, sq);
      __syncthreads();
      // Lane q joins warp q: the total of the sums, then the squares about the common mean,
      // sum (e - m)^2 = sum (e - m_q)^2 + n_q (m_q - m)^2.
      const float2 e = lane < WPR ? red[par][lane] : make_float2(0.f, 0.f);
      mean = lane_sum<32>(e.x) * inv_d;
      const float dm = lane_n > 0.f ? e.x * lane_inv - mean : 0.f;
      sq = lane_sum<32>(fmaf(lane_n * dm, dm, e.y));
    }
    const float rstd = 1.f / sqrtf(fmaf(sq, inv_d, p.eps));
    if (ok && t == 0 && p.mean != nullptr) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    if (!keeps_params<TPR>()) {
      load_param<TPR, V, VEC>(p.w, t, d, 1.f, w);
      load_param<TPR, V, VEC>(p.b, t, d, 0.f, b);
    }
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) v[i] = fmaf((v[i] - mean) * rstd, w[i], b[i]);
    store_row<TPR, V, VEC>(p.y, off, p.y_bf16, t, dd, v);
    if (!loads_ahead<TPR, V>() && r0 + hop < p.n) fetch(row + hop);
  }
}

template <int TPR, int V, bool VEC>
__global__ void __launch_bounds__(cta_threads<TPR>(), ctas_per_sm<TPR, V>()) layer_norm_bwd_kernel(const LnParams p) {
  constexpr int NT = TPR < 128 ? 128 : TPR;
  constexpr int ROWS = NT / TPR;
  constexpr int LW = TPR < 32 ? TPR : 32;
  constexpr int WPR = TPR / LW;
  __shared__ float2 red[2][WPR];
  __shared__ float join[ROWS > 1 ? NT : 1][ROWS > 1 ? 16 * V + 1 : 1];
  __shared__ float stage[VEC && ROWS == 1 ? NT / 32 : 1][VEC && ROWS == 1 ? 32 * 9 : 1];
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR, d = p.d;
  float w[8 * V], dw[8 * V], db[8 * V];
  if (keeps_params<TPR>()) load_param<TPR, V, VEC>(p.w, t, d, 1.f, w);
#pragma unroll
  for (int i = 0; i < 8 * V; ++i) dw[i] = db[i] = 0.f;
  const float inv_d = 1.f / (float)d;
  int par = 0;
  RawRow<V> nx, ng, ns;
  float nmean = 0.f, nrstd = 0.f;
  auto fetch = [&](int64_t row) {
    const bool in = row < p.n;
    const int dd = in ? d : 0;
    load_row<TPR, V, VEC>(p.x, row * d, p.s_bf16, t, dd, nx);
    load_row<TPR, V, VEC>(p.dy, row * d, p.y_bf16, t, dd, ng);
    nmean = in ? p.mean[row] : 0.f;
    nrstd = in ? p.rstd[row] : 0.f;
  };
  const int64_t hop = (int64_t)gridDim.x * ROWS;
  fetch((int64_t)blockIdx.x * ROWS + slot);
  for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < p.n; r0 += hop, par ^= 1) {
    const int64_t row = r0 + slot;
    const bool ok = row < p.n;
    const int dd = ok ? d : 0;
    const int64_t off = row * d;
    float v[8 * V], g[8 * V];
    to_floats<V, VEC>(nx, p.s_bf16, v);
    to_floats<V, VEC>(ng, p.y_bf16, g);
    const float mean = nmean, rstd = nrstd;
    if (p.ds != nullptr) load_row<TPR, V, VEC>(p.ds, off, p.s_bf16, t, dd, ns);
    if (loads_ahead<TPR, V>() && r0 + hop < p.n) fetch(row + hop);
    if (!keeps_params<TPR>()) load_param<TPR, V, VEC>(p.w, t, d, 1.f, w);
    float a = 0.f, c = 0.f;
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) {
      // g is 0 beyond the row, so what v holds there only reaches sums through g.
      v[i] = (v[i] - mean) * rstd;
      dw[i] = fmaf(g[i], v[i], dw[i]);
      db[i] += g[i];
      g[i] *= w[i];
      a += g[i];
      c = fmaf(g[i], v[i], c);
    }
    a = lane_sum<LW>(a);
    c = lane_sum<LW>(c);
    if (WPR > 1) {
      if ((t & 31) == 0) red[par][t / 32] = make_float2(a, c);
      __syncthreads();
      const int lane = threadIdx.x & 31;
      const float2 e = lane < WPR ? red[par][lane] : make_float2(0.f, 0.f);
      a = lane_sum<32>(e.x);
      c = lane_sum<32>(e.y);
    }
    a *= inv_d;
    c *= inv_d;
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) v[i] = rstd * (g[i] - a - v[i] * c);
    if (p.ds != nullptr) {
      to_floats<V, VEC>(ns, p.s_bf16, g);
#pragma unroll
      for (int i = 0; i < 8 * V; ++i) v[i] += g[i];
    }
    store_row<TPR, V, VEC>(p.dx, off, p.x_bf16, t, dd, v);
    if (p.dr != nullptr) store_row<TPR, V, VEC>(p.dr, off, p.r_bf16, t, dd, v);
    if (!loads_ahead<TPR, V>() && r0 + hop < p.n) fetch(row + hop);
  }
  if (p.part == nullptr) return;
  if (ROWS > 1) {
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) {
      join[threadIdx.x][2 * i] = dw[i];
      join[threadIdx.x][2 * i + 1] = db[i];
    }
    __syncthreads();
    if (slot != 0) return;
#pragma unroll
    for (int i = 0; i < 8 * V; ++i) {
      for (int q = 1; q < ROWS; ++q) {
        dw[i] += join[q * TPR + t][2 * i];
        db[i] += join[q * TPR + t][2 * i + 1];
      }
    }
  }
  float* out = p.part + (int64_t)blockIdx.x * 2 * d;
  if (VEC && ROWS == 1) {
    // A warp's 256 neighbours change places in shared memory, so that its stores are whole lines (as
    // they lie in registers every store took 32 sectors: 512 rows of 2048 15.8 us, this way 6.6).
    const int lane = t & 31, c0 = t / 32 * 256;
    float* mine = stage[t / 32];
#pragma unroll
    for (int k = 0; k < 2 * V; ++k) {
      const float* v = (k < V ? dw : db) + k % V * 8;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) mine[lane * 9 + i] = v[i];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = i * 32 + lane, c = k % V * TPR * 8 + c0 + e;
        if (c < d) out[(k < V ? 0 : d) + c] = mine[e / 8 * 9 + e % 8];
      }
    }
    return;
  }
  store_row<TPR, V, VEC>(out, 0, 0, t, d, dw);
  store_row<TPR, V, VEC>(out, d, 0, t, d, db);
}

// CTAs of a launch: one wave of what an SM holds, so that a CTA sees many rows, always has
// the next one on its way and leaves one row of partial sums for all of them (8192 x 4096:
// backward in two waves 127 us, one 110 us, both before its partial sums left as whole lines, 104 since;
// forward 83 and 73 us).
int rows_per_cta(int64_t d) { return d <= 64 ? 16 : d <= 128 ? 8 : d <= 512 ? 4 : 1; }
int64_t ln_ctas(int64_t n, int64_t d) {
  const int64_t want = semx::cdiv(n, rows_per_cta(d)), most = 148 * (d <= 2048 ? 4 : d <= 4096 ? 2 : 1);
  return want < most ? want : most;
}

template <bool VEC>
int launch_ln(bool bwd, const LnParams& p, cudaStream_t st) {
  const unsigned grid = (unsigned)ln_ctas(p.n, p.d);
  // A row's threads, 8 V elements each.
#define SEMX_LN(DMAX, TPR, V)                                                                             \
  if (p.d <= DMAX) {                                                                                      \
    if (bwd) layer_norm_bwd_kernel<TPR, V, VEC><<<grid, cta_threads<TPR>(), 0, st>>>(p);                  \
    else layer_norm_fwd_kernel<TPR, V, VEC><<<grid, cta_threads<TPR>(), 0, st>>>(p);                      \
    return semx::check_launch(bwd ? "layer_norm_bwd_kernel" : "layer_norm_fwd_kernel");                   \
  }
  SEMX_LN(64, 8, 1)
  SEMX_LN(128, 16, 1)
  SEMX_LN(256, 32, 1)
  SEMX_LN(512, 32, 2)
  SEMX_LN(1024, 128, 1)
  SEMX_LN(2048, 128, 2)
  SEMX_LN(4096, 256, 2)
  SEMX_LN(8192, 512, 2)
  SEMX_LN(16384, 1024, 2)
  SEMX_LN(32768, 1024, 4)
#undef SEMX_LN
  return semx::fail(SEMX_ERR_UNSUPPORTED, "layer_norm: width %d", p.d);
}

int ln_validate(const SemxLayerNormArgs* a, bool bwd) {
  SEMX_REQUIRE(a->n >= 0 && a->d >= 1, SEMX_ERR_SHAPE, "layer_norm: n=%lld, d=%lld", (long long)a->n, (long long)a->d);
  SEMX_REQUIRE(a->d <= kMaxD, SEMX_ERR_UNSUPPORTED, "layer_norm: width %lld > %d", (long long)a->d, kMaxD);
  SEMX_REQUIRE(a->n <= INT64_MAX / kMaxD / 8, SEMX_ERR_SHAPE, "layer_norm: n=%lld", (long long)a->n);
  SEMX_REQUIRE(a->eps >= 0.f, SEMX_ERR_SHAPE, "layer_norm: eps < 0");
  SEMX_REQUIRE(semx::all_aligned({a->x, a->dx}, a->x_bf16 ? 2 : 4) &&
                   semx::all_aligned({a->residual, a->dresidual}, a->r_bf16 ? 2 : 4) &&
                   semx::all_aligned({a->y, a->dy}, a->y_bf16 ? 2 : 4) &&
                   semx::all_aligned({a->sum, a->dsum}, a->s_bf16 ? 2 : 4) &&
                   semx::all_aligned({a->weight, a->bias, a->mean, a->rstd, a->dweight, a->dbias, a->workspace}, 4),
               SEMX_ERR_ALIGN, "layer_norm: a pointer is not on an element");
  if (a->n == 0) return SEMX_OK;
  if (!bwd) {
    SEMX_REQUIRE(a->x && a->y, SEMX_ERR_NULL, "layer_norm: x / y is NULL");
    SEMX_REQUIRE(!a->residual || a->sum, SEMX_ERR_NULL, "layer_norm: a residual needs the sum output");
    SEMX_REQUIRE(!a->mean == !a->rstd, SEMX_ERR_NULL, "layer_norm: one of mean / rstd is NULL");
  } else {
    SEMX_REQUIRE(a->sum && a->mean && a->rstd && a->dy && a->dx, SEMX_ERR_NULL,
                 "layer_norm bwd: sum / mean / rstd / dy / dx is NULL");
  }
  return SEMX_OK;
}

LnParams ln_params(const SemxLayerNormArgs* a) {
  LnParams p = {};
  p.n = a->n; p.d = (int)a->d; p.eps = a->eps;
  p.x_bf16 = a->x_bf16; p.r_bf16 = a->r_bf16; p.y_bf16 = a->y_bf16; p.s_bf16 = a->s_bf16;
  p.x = a->x; p.r = a->residual; p.w = a->weight; p.b = a->bias; p.y = a->y; p.s = a->sum;
  p.mean = a->mean; p.rstd = a->rstd;
  p.dy = a->dy; p.ds = a->dsum; p.dx = a->dx; p.dr = a->dresidual;
  return p;
}

bool vec_ok(int64_t d, std::initializer_list<const void*> ptrs) {
  if (d % 8 != 0) return false;
  for (const void* q : ptrs)
    if (!semx::aligned(q, 16)) return false;  // NULL counts as aligned
  return true;
}

}  // namespace

extern "C" {

size_t semx_layer_norm_args_size(void) { return sizeof(SemxLayerNormArgs); }

size_t semx_layer_norm_workspace_bytes(const SemxLayerNormArgs* a) {
  if (a == nullptr || a->n < 0 || a->d < 1 || a->d > kMaxD) return 0;
  const int64_t rows = ln_ctas(a->n, a->d);
  return (size_t)rows * 2 * a->d * sizeof(float);
}

int semx_layer_norm_fwd(const SemxLayerNormArgs* a, semx_stream_t stream) {
  SEMX_CHECK_ARGS(a, SemxLayerNormArgs);
  int rc = ln_validate(a, false);
  if (rc != SEMX_OK || a->n == 0) return rc;
  semx::DeviceScope scope;
  rc = scope.bind({a->y});
  if (rc != SEMX_OK) return rc;
  const LnParams p = ln_params(a);
  cudaStream_t st = semx::as_stream(stream);
  return vec_ok(a->d, {p.x, p.r, p.y, p.s, p.w, p.b}) ? launch_ln<true>(false, p, st) : launch_ln<false>(false, p, st);
}

int semx_layer_norm_bwd(const SemxLayerNormArgs* a, semx_stream_t stream) {
  SEMX_CHECK_ARGS(a, SemxLayerNormArgs);
  int rc = ln_validate(a, true);
  if (rc != SEMX_OK) return rc;
  const bool params = a->dweight != nullptr || a->dbias != nullptr;
  SEMX_REQUIRE(!params || a->workspace != nullptr, SEMX_ERR_WORKSPACE, "layer_norm bwd: workspace is NULL");
  semx::DeviceScope scope;
  rc = scope.bind({a->dx, a->dweight, a->dbias});
  if (rc != SEMX_OK) return rc;
  cudaStream_t st = semx::as_stream(stream);
  LnParams p = ln_params(a);
  p.x = a->sum;
  float* ws = reinterpret_cast<float*>(a->workspace);
  p.part = params ? ws : nullptr;
  if (a->n > 0) {
    rc = vec_ok(a->d, {p.x, p.dy, p.ds, p.dx, p.dr, p.w, p.part}) ? launch_ln<true>(true, p, st) : launch_ln<false>(true, p, st);
    if (rc != SEMX_OK) return rc;
  }
  if (!params) return SEMX_OK;
  const int64_t rows = ln_ctas(a->n, a->d);
  semx::Segments seg = {};
  seg.n = 2;
  seg.out[0] = a->dweight;
  seg.out[1] = a->dbias;
  seg.len[0] = seg.len[1] = a->d;
  // No rows: the sum over none of them is zero.
  return semx::colsum_once(ws, rows, 2 * a->d, seg, st);
}

}  // extern "C"
