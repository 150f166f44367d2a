// Short causal depthwise convolution with an optional SiLU over sequences that may keep
// their last inputs between calls, forward and backward, for sm_100a.
//
//   pre[t, c] = b[c] + sum_k w[c, k] x[t - (K - 1) + k, c],  y = silu(pre) or pre
//   dpre = dy silu'(pre);  dx[t] = sum_k w[k] dpre[t + K - 1 - k]
//   dw[c, k] = sum_t dpre[t, c] x[t - (K - 1) + k, c];  db[c] = sum_t dpre[t, c]
// Rows in front of a sequence's first row are the K - 1 inputs of its window (entry of the
// state pool), or zeros.
//
// Bound: HBM (2 K + 5 flops per 2 elements moved). A thread owns V neighbouring channels
// and walks over a piece of a sequence with the K inputs of the window
// in registers, so every input is read once but for the K - 1 rows in front of a piece. It
// loads U rows at a time; in the backward U rows are on their way while it uses the U before
// them (in the forward the registers for that cost more threads than it hid: 18 -> 38 us).
// The backward walks the same way: dpre of the K - 1 rows behind the piece is recomputed
// there. dw and db are summed per thread over the piece, written as one row per piece and
// reduced over pieces by the fixed-order column sum.
//
// The window is read and replaced by the thread that runs the sequence's first piece: the
// pool entry is written after that thread has read it, and no other piece looks at it
// (pieces are at least K - 1 rows long).
#include <cuda_bf16.h>

#include "semx_common.cuh"
#include "semx_math.cuh"
#include "semx_reduce.cuh"
#include "semx_seq.cuh"

namespace {

constexpr int kT = 128;
constexpr int kMaxK = 8;
// Channels per thread. More of them, up to 16-byte accesses, leave too few threads to hide the
// latency and need twice the registers (backward 404 x 321 x 256 fp32: four 108 us, two
// 93 us; forward 6151 x 2048 bf16: eight 23 us, two 18 us).
constexpr int kWidth = 2;

struct CvParams {
  semx::SeqMap m;
  int C, ctiles, silu;
  int64_t ldx;
  const void* x;
  const float* w;
  const float* b;
  void* y;
  void* state;
  const void* dy;
  void* dx;
  float* part;  // (pieces, C (K + 1)): dw | db
};

template <bool BF16, int V>
struct Raw {
  typedef uint32_t type;
};
template <>
struct Raw<false, 2> {
  typedef uint2 type;
};

template <bool BF16, int V>
__device__ __forceinline__ typename Raw<BF16, V>::type ld_raw(const void* base, int64_t i) {
  if constexpr (V > 1) {
    return *reinterpret_cast<const typename Raw<BF16, V>::type*>(reinterpret_cast<const char*>(base) + i * (BF16 ? 2 : 4));
  } else if constexpr (BF16) {
    return (uint32_t) reinterpret_cast<const unsigned short*>(base)[i];
  } else {
    return reinterpret_cast<const uint32_t*>(base)[i];
  }
}
template <bool BF16, int V>
__device__ __forceinline__ void st_raw(void* base, int64_t i, const typename Raw<BF16, V>::type& r) {
  if constexpr (V > 1) {
    *reinterpret_cast<typename Raw<BF16, V>::type*>(reinterpret_cast<char*>(base) + i * (BF16 ? 2 : 4)) = r;
  } else if constexpr (BF16) {
    reinterpret_cast<unsigned short*>(base)[i] = (unsigned short)r;
  } else {
    reinterpret_cast<uint32_t*>(base)[i] = r;
  }
}
template <bool BF16, int V>
__device__ __forceinline__ void unpack(const typename Raw<BF16, V>::type& r, float (&v)[V]) {
  if constexpr (V == 2 && BF16) {
    v[0] = __uint_as_float(r << 16); v[1] = __uint_as_float(r & 0xffff0000u);
  } else if constexpr (V == 2) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y);
  } else if constexpr (BF16) {
    v[0] = __uint_as_float(r << 16);
  } else {
    v[0] = __uint_as_float(r);
  }
}
template <bool BF16, int V>
__device__ __forceinline__ void st_vec(void* base, int64_t i, const float (&v)[V]) {
  if constexpr (V == 2 && BF16) {
    *reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<__nv_bfloat16*>(base) + i) = __floats2bfloat162_rn(v[0], v[1]);
  } else if constexpr (V == 2) {
    *reinterpret_cast<float2*>(reinterpret_cast<float*>(base) + i) = make_float2(v[0], v[1]);
  } else if constexpr (BF16) {
    reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16(v[0]);
  } else {
    reinterpret_cast<float*>(base)[i] = v[0];
  }
}

__device__ __forceinline__ float sigmoid(float v) { return semx::rcp_approx(1.f + semx::ex2_approx(-1.44269504f * v)); }

// Input of step t of the piece's sequence (t < 0: the window); `slot` as found.
template <bool BF16, int V, int K>
__device__ __forceinline__ void input(const CvParams& p, const semx::Piece& q, int64_t slot, bool cold, int t, int c,
                                      float (&v)[V]) {
  if (t >= 0) {
    unpack<BF16, V>(ld_raw<BF16, V>(p.x, (q.row0 + t) * p.ldx + c), v);
  } else if (cold) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.f;
  } else {
    unpack<BF16, V>(ld_raw<BF16, V>(p.state, (slot * (K - 1) + (K - 1 + t)) * p.C + c), v);
  }
}

// The CTA's weights (a run of w) go through shared memory, where a thread's V K values are
// one run too: read from global memory they cost as much as 32 rows of x.
template <int V, int K>
struct Weights {
  float v[kT * V * K];
};
template <int V, int K>
__device__ __forceinline__ void stage_weights(Weights<V, K>& s, const float* w, int c0, int C) {
  const int n = min((int)blockDim.x * V, C - c0) * K;
  const float* src = w + (int64_t)c0 * K;
  for (int i = threadIdx.x; i < n; i += blockDim.x) s.v[i] = src[i];
}
template <int V, int K>
__device__ __forceinline__ void own_weights(const Weights<V, K>& s, float (&w)[K][V]) {
  const float* mine = s.v + threadIdx.x * (V * K);
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][i] = mine[i * K + k];
}

template <bool BF16, int V, int K, int U>
__global__ void __launch_bounds__(kT) short_conv_fwd_kernel(const CvParams p) {
  __shared__ Weights<V, K> sw;
  const int64_t j = blockIdx.x / p.ctiles;
  const int c0 = (blockIdx.x % p.ctiles) * blockDim.x * V, c = c0 + threadIdx.x * V;
  stage_weights(sw, p.w, c0, p.C);
  const semx::Piece q = semx::find_piece(p.m, j);
  const int64_t slot = q.live ? semx::find_slot(p.m, q.s) : semx::kNone;
  __syncthreads();
  if (c >= p.C) return;
  float zero[V];
#pragma unroll
  for (int i = 0; i < V; ++i) zero[i] = 0.f;
  semx::for_unused_rows(p.m, j, [&](int64_t r) { st_vec<BF16, V>(p.y, r * p.C + c, zero); });
  if (!q.live) return;
  const bool cold = slot < 0 || (p.m.fresh != nullptr && p.m.fresh[q.s] != 0);
  float w[K][V], b[V];
  own_weights(sw, w);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    b[i] = p.b != nullptr ? p.b[c + i] : 0.f;
    if (slot == semx::kRefused) b[i] = __int_as_float(0x7fffffff);
  }
  float win[K][V];
#pragma unroll
  for (int k = 0; k + 1 < K; ++k) input<BF16, V, K>(p, q, slot, cold, q.t0 - (K - 1) + k, c, win[k]);
  if (K > 1 && q.k == 0 && slot >= 0) {
    // The window left behind: the last K - 1 of (old window, rows).
    float keep[K][V];
#pragma unroll
    for (int k = 0; k + 1 < K; ++k) {
      const int t = q.len - (K - 1) + k;
      if (t < 0) {
        // Entry K - 1 + t of the old window, which win holds (this is the first piece).
#pragma unroll
        for (int i = 0; i < V; ++i) keep[k][i] = 0.f;
#pragma unroll
        for (int o = 0; o + 1 < K; ++o)
          if (o == K - 1 + t) {
#pragma unroll
            for (int i = 0; i < V; ++i) keep[k][i] = win[o][i];
          }
      } else {
        input<BF16, V, K>(p, q, slot, cold, t, c, keep[k]);
      }
    }
#pragma unroll
    for (int k = 0; k + 1 < K; ++k) st_vec<BF16, V>(p.state, (slot * (K - 1) + k) * p.C + c, keep[k]);
  }
  int64_t xo = (q.row0 + q.t0) * p.ldx + c, yo = (q.row0 + q.t0) * p.C + c;
  auto step = [&](const typename Raw<BF16, V>::type& raw) {
    unpack<BF16, V>(raw, win[K - 1]);
    float out[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float a = b[i];
#pragma unroll
      for (int k = 0; k < K; ++k) a = fmaf(w[k][i], win[k][i], a);
      out[i] = p.silu ? a * sigmoid(a) : a;
    }
    st_vec<BF16, V>(p.y, yo, out);
    yo += p.C;
#pragma unroll
    for (int k = 0; k + 1 < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) win[k][i] = win[k + 1][i];
  };
  int t = q.t0;
  for (; t + U <= q.t1; t += U) {
    typename Raw<BF16, V>::type raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = ld_raw<BF16, V>(p.x, xo + u * p.ldx);
    xo += U * p.ldx;
#pragma unroll
    for (int u = 0; u < U; ++u) step(raw[u]);
  }
  for (; t < q.t1; ++t) {
    step(ld_raw<BF16, V>(p.x, xo));
    xo += p.ldx;
  }
}

// Steps t0 .. t1 + K - 2: dpre of each (the ones from t1 on belong to the next piece and
// only feed dx), and dx[t - (K - 1)] once dpre[t] is there.
template <bool BF16, int V, int K, int U>
__global__ void __launch_bounds__(kT) short_conv_bwd_kernel(const CvParams p) {
  __shared__ Weights<V, K> sw;
  const int64_t j = blockIdx.x / p.ctiles;
  const int c0 = (blockIdx.x % p.ctiles) * blockDim.x * V, c = c0 + threadIdx.x * V;
  stage_weights(sw, p.w, c0, p.C);
  const semx::Piece q = semx::find_piece(p.m, j);
  __syncthreads();
  if (c >= p.C) return;
  float zero[V];
#pragma unroll
  for (int i = 0; i < V; ++i) zero[i] = 0.f;
  semx::for_unused_rows(p.m, j, [&](int64_t r) { st_vec<BF16, V>(p.dx, r * p.C + c, zero); });
  float w[K][V], b[V], dw[K][V], db[V];
  own_weights(sw, w);
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int k = 0; k < K; ++k) dw[k][i] = 0.f;
    b[i] = p.b != nullptr ? p.b[c + i] : 0.f;
    db[i] = 0.f;
  }
  float win[K][V], dp[K][V];  // dp[k] = dpre[t - (K - 1) + k]
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) dp[k][i] = 0.f;
    if (k + 1 < K && q.live) input<BF16, V, K>(p, q, semx::kNone, true, q.t0 - (K - 1) + k, c, win[k]);
  }
  const int end = q.t1 > q.t0 ? q.t1 + K - 1 : 0;  // a piece without rows has no steps
  typedef typename Raw<BF16, V>::type R;
  R nx[U], ng[U];  // U rows are always on their way
  auto fetch = [&](int t) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t + u < end) {
        const int tt = min(t + u, q.len - 1);  // rows behind the sequence load its last row and count nothing
        nx[u] = ld_raw<BF16, V>(p.x, (q.row0 + tt) * p.ldx + c);
        ng[u] = ld_raw<BF16, V>(p.dy, (q.row0 + tt) * p.C + c);
      }
    }
  };
  fetch(q.t0);
  for (int t = q.t0; t < end; t += U) {
    R rx[U], rg[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      rx[u] = nx[u];
      rg[u] = ng[u];
    }
    fetch(t + U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t + u < end) {
        float g[V];
        unpack<BF16, V>(rx[u], win[K - 1]);
        unpack<BF16, V>(rg[u], g);
        const bool mine = t + u < q.t1;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float d = g[i];
          if (p.silu) {
            float a = b[i];
#pragma unroll
            for (int k = 0; k < K; ++k) a = fmaf(w[k][i], win[k][i], a);
            const float sg = sigmoid(a);
            d *= sg * fmaf(a, 1.f - sg, 1.f);
          }
          if (t + u >= q.len) d = 0.f;
#pragma unroll
          for (int k = 0; k + 1 < K; ++k) dp[k][i] = dp[k + 1][i];
          dp[K - 1][i] = d;
          if (mine) {
            db[i] += d;
#pragma unroll
            for (int k = 0; k < K; ++k) dw[k][i] = fmaf(d, win[k][i], dw[k][i]);
          }
#pragma unroll
          for (int k = 0; k + 1 < K; ++k) win[k][i] = win[k + 1][i];
        }
        const int to = t + u - (K - 1);
        if (to >= q.t0) {
          float dx[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float a = 0.f;
            // dpre[to + K - 1 - k] = dp[K - 1 - k]
#pragma unroll
            for (int k = 0; k < K; ++k) a = fmaf(w[k][i], dp[K - 1 - k][i], a);
            dx[i] = a;
          }
          st_vec<BF16, V>(p.dx, (q.row0 + to) * p.C + c, dx);
        }
      }
    }
  }
  if (p.part != nullptr && p.m.S > 0) {
    float* row = p.part + j * ((int64_t)p.C * (K + 1));
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int k = 0; k < K; ++k) row[(int64_t)(c + i) * K + k] = dw[k][i];
      row[(int64_t)p.C * K + c + i] = db[i];
    }
  }
}

// One row per sequence. Two channels per thread (one where they do not pair up): with few
// sequences the threads are what hides the latency, and a warp's weights are one run of
// memory. A CTA takes a run of sequences, so that the weights are read once for all of them,
// and loads kAhead rows and windows before it uses them.
constexpr int kAhead = 4;
constexpr int kStepRows = 16;  // sequences per CTA at most

template <bool BF16, int V, int K>
__global__ void __launch_bounds__(kT) short_conv_step_kernel(const CvParams p, int rows) {
  typedef typename Raw<BF16, V>::type R;
  __shared__ int64_t slots[kStepRows];
  const int64_t s0 = (int64_t)(blockIdx.x / p.ctiles) * rows;
  const int n = (int)min((int64_t)rows, p.m.S - s0);
  const int c = ((blockIdx.x % p.ctiles) * kT + threadIdx.x) * V;
  float w[V][K], b[V];
  if (c < p.C) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int k = 0; k < K; ++k) w[i][k] = p.w[(int64_t)(c + i) * K + k];
      b[i] = p.b != nullptr ? p.b[c + i] : 0.f;
    }
  }
  semx::find_slots<kStepRows>(p.m, s0, n, slots);
  if (c >= p.C) return;
  for (int i0 = 0; i0 < n; i0 += kAhead) {
    R rx[kAhead][K];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i0 + u < n) {
        const int64_t s = s0 + i0 + u, slot = slots[i0 + u];
        rx[u][K - 1] = ld_raw<BF16, V>(p.x, s * p.ldx + c);
        const bool cold = slot < 0 || (p.m.fresh != nullptr && p.m.fresh[s] != 0);
#pragma unroll
        for (int k = 0; k + 1 < K; ++k)
          rx[u][k] = cold ? R{} : ld_raw<BF16, V>(p.state, (slot * (K - 1) + k) * p.C + c);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i0 + u < n) {
        const int64_t s = s0 + i0 + u, slot = slots[i0 + u];
        float a[V];
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] = slot == semx::kRefused ? __int_as_float(0x7fffffff) : b[i];
#pragma unroll
        for (int k = 0; k < K; ++k) {
          float x[V];
          unpack<BF16, V>(rx[u][k], x);
#pragma unroll
          for (int i = 0; i < V; ++i) a[i] = fmaf(w[i][k], x[i], a[i]);
        }
        if (p.silu) {
#pragma unroll
          for (int i = 0; i < V; ++i) a[i] *= sigmoid(a[i]);
        }
        st_vec<BF16, V>(p.y, s * p.C + c, a);
        if (slot >= 0) {
#pragma unroll
          for (int k = 0; k + 1 < K; ++k) st_raw<BF16, V>(p.state, (slot * (K - 1) + k) * p.C + c, rx[u][k + 1]);
        }
      }
    }
  }
}

template <bool BF16, int V, int K0>
int launch_step(int K, CvParams& p, cudaStream_t st) {
  if constexpr (K0 <= kMaxK) {
    if (K != K0) return launch_step<BF16, V, K0 + 1>(K, p, st);
    p.ctiles = (int)semx::cdiv(p.C, (int64_t)kT * V);
    // Sequences per CTA: as many as leave four CTAs per SM.
    int rows = kStepRows;
    while (rows > 1 && semx::cdiv(p.m.S, rows) * p.ctiles < 148 * 4) rows /= 2;
    const int64_t grid = semx::cdiv(p.m.S, rows) * p.ctiles;
    if (grid == 0) return SEMX_OK;
    if (grid >= ((int64_t)1 << 31)) return semx::fail(SEMX_ERR_SHAPE, "short_conv: too many sequences");
    short_conv_step_kernel<BF16, V, K0><<<(unsigned)grid, kT, 0, st>>>(p, rows);
    return semx::check_launch("short_conv_step_kernel");
  }
  return semx::fail(SEMX_ERR_UNSUPPORTED, "short_conv: %d taps", K);
}

// Rows of a piece: long pieces re-read few rows (K - 1 in front, and K - 1 behind in the
// backward) and leave few rows of partial sums; short ones fill the GPU. Always long against
// this rule, bf16, 4 taps: 600 x 1024 forward 7.8 and 6.4 us, training pass 26.7 and 17.7;
// 150 x 256 7.8 and 6.1, 26.2 and 15.2; 6151 x 2048 the same.
constexpr int64_t kFill = 148 * 512;  // threads
int64_t piece_rows(int64_t T, int64_t C, bool bwd) {
  int64_t Q = bwd ? 64 : 32;
  while (Q > 8 && semx::cdiv(T, Q) * semx::cdiv(C, (int64_t)kWidth) < kFill) Q /= 2;
  return Q;
}

int cv_validate(const SemxShortConvArgs* a, bool bwd, CvParams* p) {
  SEMX_REQUIRE(a->K >= 1 && a->K <= kMaxK, SEMX_ERR_UNSUPPORTED, "short_conv: %d taps (1..%d)", a->K, kMaxK);
  SEMX_REQUIRE(a->C >= 1 && a->C < (1 << 24), SEMX_ERR_SHAPE, "short_conv: C=%lld", (long long)a->C);
  SEMX_REQUIRE(a->ldx >= a->C && a->ldx < ((int64_t)1 << 31), SEMX_ERR_SHAPE, "short_conv: row stride %lld for %lld channels",
               (long long)a->ldx, (long long)a->C);
  int rc = semx::check_seqs("short_conv", a->S, a->rows, a->L, a->cu_seqlens, a->state, a->slots, a->fresh,
                            a->n_slots, &p->m);
  if (rc != SEMX_OK) return rc;
  // One tap has no window: whatever pool came along is empty.
  if (a->K == 1) p->m.n_slots = 0;
  SEMX_REQUIRE(!bwd || a->state == nullptr, SEMX_ERR_UNSUPPORTED, "short_conv bwd: no state");
  SEMX_REQUIRE(a->w && (a->rows == 0 || a->x), SEMX_ERR_NULL, "short_conv: x / w is NULL");
  if (!bwd) SEMX_REQUIRE(a->rows == 0 || a->y, SEMX_ERR_NULL, "short_conv: y is NULL");
  else SEMX_REQUIRE(a->rows == 0 || (a->dy && a->dx), SEMX_ERR_NULL, "short_conv bwd: dy / dx is NULL");
  SEMX_REQUIRE(semx::all_aligned({a->x, a->y, a->state, a->dy, a->dx}, a->bf16 ? 2 : 4) &&
                   semx::all_aligned({a->w, a->b, a->cu_seqlens, a->slots, a->dw, a->db, a->workspace}, 4),
               SEMX_ERR_ALIGN, "short_conv: a pointer is not on an element");
  p->C = (int)a->C; p->silu = a->silu; p->ldx = a->ldx;
  p->x = a->x; p->w = a->w; p->b = a->b; p->y = a->y; p->state = a->state;
  p->dy = a->dy; p->dx = a->dx;
  return SEMX_OK;
}

// Whether every row allows accesses of V neighbouring channels.
bool cv_allows(const SemxShortConvArgs* a, int64_t V) {
  if (a->C % V != 0 || a->ldx % V != 0) return false;
  for (const void* q : {a->x, (const void*)a->y, (const void*)a->state, a->dy, (const void*)a->dx})
    if (!semx::aligned(q, V * (a->bf16 ? 2 : 4))) return false;
  return true;
}

int64_t cv_pieces(const SemxShortConvArgs* a, semx::SeqMap* m) {
  // The partial rows' number must not depend on alignment: both paths cut alike.
  semx::set_pieces(m, piece_rows(a->rows, a->C, true));
  return m->pieces;
}

template <bool BF16, int V, int K0>
int launch_cv(bool bwd, int K, CvParams& p, cudaStream_t st) {
  // Narrow tensors take narrow CTAs.
  const int nt = (int)semx::cdiv(p.C, (int64_t)V) >= kT ? kT : (int)semx::cdiv(semx::cdiv(p.C, (int64_t)V), 32) * 32;
  p.ctiles = (int)semx::cdiv(p.C, (int64_t)nt * V);
  const int64_t grid = p.m.pieces * p.ctiles;
  if (grid == 0) return SEMX_OK;
  if (grid >= ((int64_t)1 << 31)) return semx::fail(SEMX_ERR_SHAPE, "short_conv: too many pieces");
  if constexpr (K0 <= kMaxK) {
    if (K == K0) {
      if (bwd) short_conv_bwd_kernel<BF16, V, K0, 4><<<(unsigned)grid, nt, 0, st>>>(p);
      else short_conv_fwd_kernel<BF16, V, K0, 4><<<(unsigned)grid, nt, 0, st>>>(p);
      return semx::check_launch(bwd ? "short_conv_bwd_kernel" : "short_conv_fwd_kernel");
    }
    return launch_cv<BF16, V, K0 + 1>(bwd, K, p, st);
  }
  return semx::fail(SEMX_ERR_UNSUPPORTED, "short_conv: %d taps", K);
}

int dispatch_cv(const SemxShortConvArgs* a, bool bwd, CvParams& p, cudaStream_t st) {
  if (!bwd && p.m.cu == nullptr && p.m.L == 1) {
    if (cv_allows(a, 2)) return a->bf16 ? launch_step<true, 2, 1>(a->K, p, st) : launch_step<false, 2, 1>(a->K, p, st);
    return a->bf16 ? launch_step<true, 1, 1>(a->K, p, st) : launch_step<false, 1, 1>(a->K, p, st);
  }
  if (!cv_allows(a, kWidth))
    return a->bf16 ? launch_cv<true, 1, 1>(bwd, a->K, p, st) : launch_cv<false, 1, 1>(bwd, a->K, p, st);
  return a->bf16 ? launch_cv<true, kWidth, 1>(bwd, a->K, p, st) : launch_cv<false, kWidth, 1>(bwd, a->K, p, st);
}

}  // namespace

extern "C" {

size_t semx_short_conv_args_size(void) { return sizeof(SemxShortConvArgs); }

size_t semx_short_conv_workspace_bytes(const SemxShortConvArgs* a) {
  if (a == nullptr) return 0;
  CvParams p = {};
  SemxShortConvArgs b = *a;
  b.w = reinterpret_cast<const float*>(256);
  b.x = b.dy = reinterpret_cast<const float*>(256);
  b.dx = reinterpret_cast<void*>(256);
  if (cv_validate(&b, true, &p) != SEMX_OK) return 0;
  const int64_t rows = cv_pieces(a, &p.m), cols = a->C * (a->K + 1);
  return (size_t)rows * cols * sizeof(float);
}

int semx_short_conv_fwd(const SemxShortConvArgs* a, semx_stream_t stream) {
  SEMX_CHECK_ARGS(a, SemxShortConvArgs);
  CvParams p = {};
  int rc = cv_validate(a, false, &p);
  if (rc != SEMX_OK || semx::nothing_to_do(p.m)) return rc;
  semx::DeviceScope scope;
  rc = scope.bind({a->y, a->state});
  if (rc != SEMX_OK) return rc;
  semx::set_pieces(&p.m, piece_rows(a->rows, a->C, false));
  // Without a sequence every row is a row behind the last one.
  if (p.m.S == 0 && p.m.T > 0) p.m.pieces = p.m.T;
  return dispatch_cv(a, false, p, semx::as_stream(stream));
}

int semx_short_conv_bwd(const SemxShortConvArgs* a, semx_stream_t stream) {
  SEMX_CHECK_ARGS(a, SemxShortConvArgs);
  CvParams p = {};
  int rc = cv_validate(a, true, &p);
  if (rc != SEMX_OK) return rc;
  const bool params = a->dw != nullptr || a->db != nullptr;
  SEMX_REQUIRE(!params || a->workspace != nullptr, SEMX_ERR_WORKSPACE, "short_conv bwd: workspace is NULL");
  semx::DeviceScope scope;
  rc = scope.bind({a->dx, a->dw, a->db});
  if (rc != SEMX_OK) return rc;
  cudaStream_t st = semx::as_stream(stream);
  const int64_t rows = cv_pieces(a, &p.m), cols = a->C * (a->K + 1);
  if (p.m.S == 0 && p.m.T > 0) p.m.pieces = p.m.T;
  float* ws = reinterpret_cast<float*>(a->workspace);
  p.part = params ? ws : nullptr;
  if (a->rows > 0) {
    rc = dispatch_cv(a, true, p, st);
    if (rc != SEMX_OK) return rc;
  }
  if (!params) return SEMX_OK;
  semx::Segments seg = {};
  seg.n = 2;
  seg.out[0] = a->dw;
  seg.out[1] = a->db;
  seg.len[0] = a->C * a->K;
  seg.len[1] = a->C;
  return semx::colsum_once(ws, a->rows > 0 && a->S > 0 ? rows : 0, cols, seg, st);
}

}  // extern "C"
