// Gated linear recurrence (one real mode per channel, decay and input gated per token), forward,
// backward and single tokens, for sm_100a.
//
//   rho = sigmoid(r + r_bias), iota = sigmoid(i + i_bias), la = -rate_scale softplus(rate) rho
//   a = exp(la), left = 1 - a^2, gain = sqrt(max(left, 1e-6))
//   h_t = a_t h_{t-1} + gain_t iota_t x_t;   y = h silu(z)  (h without z)
// Backward, with g_t = dy_t silu(z_t) + a_{t+1} g_{t+1}:
//   dz = dy h silu'(z), dx = g gain iota, di = g gain x iota (1 - iota)
//   dla = g a h_{t-1} - (left > 1e-6) g iota x a^2 / gain, dr = -speed dla rho (1 - rho)
// with speed = rate_scale softplus(rate).
//
// Bound: HBM (5 values per element forward, 9 backward); what each element needs of the
// special-function unit (7 to 14 operations) comes next.
//
// Split: a tile is 64 steps of one sequence by 64 channels; a CTA reads it once. A thread has
// kSeg neighbouring steps of four neighbouring channels (whole sectors of a row per warp), so the
// recurrence inside a tile is 16 segments: each thread folds its steps into one map
// h -> A h + B, 64 threads (one per channel) fold the segments and find the tile's entry state,
// and each thread runs its steps again from its segment's entry state, on registers.
// Tiles of a sequence are linked inside the one launch: each leaves its map (A, B), and takes the
// maps of the tiles in front of it in its group of 16 and the state that the last tile of the group
// before left. Which maps are folded in which order depends on the numbers alone, so results do
// not change from run to run. Tickets number the tiles in the order in which CTAs start, so a tile
// only waits for tiles that run already. The backward runs the same from the last tile on.
#include "semx_reduce.cuh"
#include "state_scan.cuh"

namespace {

using namespace semx_scan;

constexpr int kT = 256;
constexpr int kSegs = 16, kSeg = 4, kRows = kSegs * kSeg;  // segments, steps of each, steps of a tile
constexpr int kCh = 64;                                    // channels of a tile
constexpr int kGroup = 16;                                 // tiles between two states handed on
constexpr unsigned kPolls = 1u << 22;
constexpr float kLeast = 1e-6f;  // of 1 - a^2, as the gamma gain of the selective-LRU scans has it

__device__ unsigned int g_link_timeouts;

struct GlParams {
  semx::SeqMap m;
  int C, ctiles, bf16, access;
  float scale;
  int64_t ldx, ldr, ldi, ldz;
  const void* x;
  const void* r;
  const void* i;
  const void* z;
  const float* rate;
  const float* r_bias;
  const float* i_bias;
  void* y;
  float* state;
  float* ckpt;  // (tiles, C) state in front of each tile
  const void* dy;
  void* dx;
  void* dr;
  void* di;
  void* dz;
  float* part;   // (tiles, 3, C) partial drate | dr_bias | di_bias
  int* ticket;   // NULL: no sequence has more than one tile
  int* flags;    // (tiles, ctiles, 2): 1 the tile's map is there, 2 the state behind it too
  float2* maps;  // (tiles, C)
  float* left;   // (tiles, C) state behind the last tile of each group
};

// exp(la) - 1 for -0.35 <= la <= 0: Taylor's series up to la^7 (the rest is 1.6e-8 of it).
__device__ __forceinline__ float expm1_near(float la) {
  float q = fmaf(la, 1.f / 5040.f, 1.f / 720.f);
  q = fmaf(q, la, 1.f / 120.f);
  q = fmaf(q, la, 1.f / 24.f);
  q = fmaf(q, la, 1.f / 6.f);
  q = fmaf(q, la, 0.5f);
  return fmaf(la * la, q, la);
}

// Decay a and 1 - a^2. The series near 0 keeps the decay exact to its rounding (a state
// multiplies hundreds of them) and 1 - a^2 = -e (2 + e) free of cancellation; the special-function
// exponential is 2 steps off, which a decay below 0.7 forgets at once.
__device__ __forceinline__ void decay(float la, bool slow, float* a, float* left) {
  float e = expm1_near(la);
  *a = 1.f + e;
  *left = -e * (2.f + e);
  if (!slow) {
    const float f = semx::ex2_approx(la * kLog2e);
    const bool far = la < -0.35f;
    if (far) {
      *a = f;
      *left = fmaf(-f, f, 1.f);
    }
  }
}

// sigmoid(v) and 1 - sigmoid(v), the latter free of cancellation.
__device__ __forceinline__ void sigmoids(float v, float* s, float* rest) {
  const float e = semx::ex2_approx(-kLog2e * v);
  *s = semx::rcp_approx(1.f + e);
  *rest = v < -80.f ? 1.f : e * *s;
}

struct Quad {
  float v[4];
};
__device__ __forceinline__ Quad quad(float4 f) { return Quad{{f.x, f.y, f.z, f.w}}; }

__device__ __forceinline__ int load_flag(const int* f) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(f) : "memory");
  return v;
}
__device__ __forceinline__ void store_flag(int* f, int v) {
  asm volatile("st.release.gpu.global.s32 [%0], %1;" ::"l"(f), "r"(v) : "memory");
}

// Where tile number `at` in the order of the recurrence is among the pieces: j0 + dir at.
struct Chain {
  int64_t j0;
  int dir, at;
  bool next;  // a tile follows
};

// One warp, a lane per channel (c, or none: ok false). (A, B): the tile's map; the first tile of a
// sequence has its entry state in it (A = 0). Returns the state in front of the tile.
__device__ float link_in(const GlParams& p, const Chain& q, int ct, int half, int c, bool ok, float A, float B) {
  const int lane = threadIdx.x & 31;
  const int64_t me = q.j0 + (int64_t)q.dir * q.at;
  int* flag = p.flags + (me * p.ctiles + ct) * 2 + half;
  if (q.next) {
    if (ok) __stcg(&p.maps[me * p.C + c], make_float2(A, B));
    __threadfence();
    __syncwarp();
    if (lane == 0) store_flag(flag, 1);
  }
  if (q.at == 0) return 0.f;
  const int g0 = q.at / kGroup * kGroup, n = q.at - g0;
  // Lanes below n wait for the maps of the tiles in front in the group, lane kGroup for the state
  // that the group before left.
  const bool waits = lane < n || (lane == kGroup && g0 > 0);
  const int64_t of = q.j0 + (int64_t)q.dir * (lane < n ? g0 + lane : g0 - 1);
  // Offsets that decrease can name a piece that is none.
  const bool there = waits && of >= 0 && of < p.m.pieces;
  const int* theirs = p.flags + (of * p.ctiles + ct) * 2 + half;
  const int want = lane < n ? 1 : 2;
  bool done = false;
  for (unsigned tries = 0; tries < kPolls && !done; ++tries)
    done = __all_sync(0xffffffffu, !there || load_flag(theirs) >= want);
  if (!done && lane == 0) atomicAdd(&g_link_timeouts, 1u);
  __syncwarp();
  float a = 1.f, b = 0.f;
#pragma unroll 1
  for (int e = 0; e < n; e += 5) {  // 15 maps at most, 5 on their way at a time
    float2 m[5];
#pragma unroll
    for (int u = 0; u < 5; ++u) {
      const int64_t j = q.j0 + (int64_t)q.dir * (g0 + e + u);
      m[u] = e + u < n && ok && j >= 0 && j < p.m.pieces ? __ldcg(&p.maps[j * p.C + c]) : make_float2(1.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < 5; ++u) {
      b = fmaf(m[u].x, b, m[u].y);
      a *= m[u].x;
    }
  }
  float h = 0.f;
  if (g0 > 0) {
    const int64_t j = q.j0 + (int64_t)q.dir * (g0 - 1);
    if (ok && j >= 0 && j < p.m.pieces) h = __ldcg(&p.left[j * p.C + c]);
  }
  if (!done) return __int_as_float(0x7fffffff);
  // A sequence's first tile (A = 0) leaves no way for what stands in front of it.
  return g0 > 0 ? fmaf(a, h, b) : b;
}

// Hands on the state behind the tile: the last tile of a group writes it. Every tile raises its
// flag, so that nothing waits for long whatever the offsets are.
__device__ __forceinline__ void link_out(const GlParams& p, const Chain& q, int ct, int half, int c, bool ok, float h) {
  const int64_t me = q.j0 + (int64_t)q.dir * q.at;
  if (q.next && q.at % kGroup == kGroup - 1) {
    if (ok) __stcg(&p.left[me * p.C + c], h);
    __threadfence();
  }
  __syncwarp();
  if ((threadIdx.x & 31) == 0) store_flag(p.flags + (me * p.ctiles + ct) * 2 + half, 2);
}

// Number of the tile that this CTA takes.
__device__ __forceinline__ int64_t take_tile(const GlParams& p, int* slot) {
  if (p.ticket == nullptr) return blockIdx.x;
  if (threadIdx.x == 0) *slot = atomicAdd(p.ticket, 1);
  __syncthreads();
  return *slot;
}

// Per channel of the tile: speed = rate_scale softplus(rate), both biases, and with SLOPE the
// derivative of speed.
template <bool SLOPE>
__device__ __forceinline__ void tile_params(const GlParams& p, int c0, float (*par)[kCh]) {
  if (threadIdx.x < kCh) {
    const int c = min(c0 + (int)threadIdx.x, p.C - 1);
    const float rate = p.rate[c], s = p.scale * semx::softplus(rate);
    par[0][threadIdx.x] = s > 3.4e38f ? 3.4e38f : s;  // an infinite one times a closed gate is no number
    par[1][threadIdx.x] = p.r_bias != nullptr ? p.r_bias[c] : 0.f;
    par[2][threadIdx.x] = p.i_bias != nullptr ? p.i_bias[c] : 0.f;
    if (SLOPE) par[3][threadIdx.x] = p.scale * semx::softplus_grad(rate);
  }
}
__device__ __forceinline__ Quad shared_quad(const float* row, int c) {
  return quad(*reinterpret_cast<const float4*>(row + c));
}

// LINK: sequences of several tiles.
template <int ACC, bool LINK>
__global__ void __launch_bounds__(kT, 3) gated_lru_fwd_kernel(const GlParams p) {
  typedef typename RawQuad<ACC>::type Raw;
  __shared__ __align__(16) float par[3][kCh];
  __shared__ __align__(16) float mA[kSegs][kCh], mB[kSegs][kCh];
  __shared__ int ticket;
  const int tid = threadIdx.x;
  const int64_t tile = LINK ? take_tile(p, &ticket) : (int64_t)blockIdx.x;
  const int64_t j = tile / p.ctiles;
  const int ct = (int)(tile % p.ctiles), c0 = ct * kCh;
  const int seg = tid / 16, lc = tid % 16 * 4, nn = min(4, p.C - c0 - lc);
  const int64_t ch = nn > 0 ? c0 + lc : 0;
  const Piece q = find_piece(p.m, j);
  const bool gated = p.z != nullptr;
  if (seg == 0 && nn > 0)
    for_unused_rows(p.m, j, [&](int64_t row) {
      store_quad<ACC>(p.y, row * p.C + ch, p.bf16, nn, make_float4(0.f, 0.f, 0.f, 0.f));
    });
  if (!q.live) {
    if (LINK && tid < 2) store_flag(p.flags + (j * p.ctiles + ct) * 2 + tid, 2);
    return;
  }
  const int t0 = q.t0 + seg * kSeg;
  Raw rx[kSeg], rr[kSeg], ri[kSeg], rz[kSeg];
#pragma unroll
  for (int u = 0; u < kSeg; ++u) {
    rx[u] = rr[u] = ri[u] = rz[u] = Raw{};
    if (t0 + u < q.t1 && nn > 0) {
      const int64_t row = q.row0 + t0 + u;
      rr[u] = load_quad<ACC>(p.r, row * p.ldr + ch, p.bf16, nn);
      ri[u] = load_quad<ACC>(p.i, row * p.ldi + ch, p.bf16, nn);
      rx[u] = load_quad<ACC>(p.x, row * p.ldx + ch, p.bf16, nn);
      if (gated) rz[u] = load_quad<ACC>(p.z, row * p.ldz + ch, p.bf16, nn);
    }
  }
  tile_params<false>(p, c0, par);
  const bool first = q.k == 0, last = q.t1 == q.len;
  int64_t slot = semx::kNone;
  if (p.m.n_slots > 0 && (first || last)) slot = find_slot(p.m, q.s);
  __syncthreads();
  const Quad speed = shared_quad(par[0], lc), rb = shared_quad(par[1], lc), ib = shared_quad(par[2], lc);
  const bool slow = fmaxf(fmaxf(speed.v[0], speed.v[1]), fmaxf(speed.v[2], speed.v[3])) <= 0.35f;
  float a[kSeg][4], b[kSeg][4];
  float A[4] = {1.f, 1.f, 1.f, 1.f}, B[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < kSeg; ++u) {
    const Quad x = quad(quad_floats<ACC>(rx[u], p.bf16)), r = quad(quad_floats<ACC>(rr[u], p.bf16)),
               i = quad(quad_floats<ACC>(ri[u], p.bf16));
    const bool in = t0 + u < q.t1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float left;
      decay(-speed.v[k] * sigmoid(r.v[k] + rb.v[k]), slow, &a[u][k], &left);
      left = left < kLeast ? kLeast : left;
      b[u][k] = left * semx::rsqrt_approx(left) * sigmoid(i.v[k] + ib.v[k]) * x.v[k];
      if (!in) a[u][k] = 1.f, b[u][k] = 0.f;  // rows behind the last one keep the state
      A[k] *= a[u][k];
      B[k] = fmaf(a[u][k], B[k], b[u][k]);
    }
  }
  *reinterpret_cast<float4*>(&mA[seg][lc]) = make_float4(A[0], A[1], A[2], A[3]);
  *reinterpret_cast<float4*>(&mB[seg][lc]) = make_float4(B[0], B[1], B[2], B[3]);
  __syncthreads();
  if (tid < kCh) {
    const int c = c0 + tid;
    const bool ok = c < p.C;
    float h = 0.f;
    if (first && ok && slot != semx::kNone) {
      const bool fresh = p.m.fresh != nullptr && p.m.fresh[q.s] != 0;
      h = slot == semx::kRefused ? __int_as_float(0x7fffffff) : fresh ? 0.f : p.state[slot * p.C + c];
    }
    Chain link = {j - q.k, 1, q.k, !last};
    if (LINK && q.len > p.m.Q) {
      float fA = 1.f, fB = h;
#pragma unroll
      for (int s = 0; s < kSegs; ++s) {
        fA *= mA[s][tid];
        fB = fmaf(mA[s][tid], fB, mB[s][tid]);
      }
      const float in = link_in(p, link, ct, tid / 32, c, ok, first ? 0.f : fA, fB);
      if (!first) h = in;
    }
    if (p.ckpt != nullptr && ok) p.ckpt[j * p.C + c] = h;
#pragma unroll
    for (int s = 0; s < kSegs; ++s) {
      const float next = fmaf(mA[s][tid], h, mB[s][tid]);
      mB[s][tid] = h;  // from here on the segment's entry state
      h = next;
    }
    if (LINK) link_out(p, link, ct, tid / 32, c, ok, h);
    if (last && ok && slot >= 0) p.state[slot * p.C + c] = h;
  }
  __syncthreads();
  Quad h = shared_quad(mB[seg], lc);
#pragma unroll
  for (int u = 0; u < kSeg; ++u) {
    Quad y;
    const Quad z = quad(quad_floats<ACC>(rz[u], p.bf16));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      h.v[k] = fmaf(a[u][k], h.v[k], b[u][k]);
      y.v[k] = gated ? h.v[k] * (z.v[k] * sigmoid(z.v[k])) : h.v[k];
    }
    if (t0 + u < q.t1 && nn > 0)
      store_quad<ACC>(p.y, (q.row0 + t0 + u) * p.C + ch, p.bf16, nn, make_float4(y.v[0], y.v[1], y.v[2], y.v[3]));
  }
}

template <int ACC, bool LINK>
__global__ void __launch_bounds__(kT, 2) gated_lru_bwd_kernel(const GlParams p) {
  typedef typename RawQuad<ACC>::type Raw;
  __shared__ __align__(16) float par[4][kCh];
  __shared__ __align__(16) float mA[kSegs][kCh], mB[kSegs][kCh], mG[kSegs][kCh];
  __shared__ int ticket;
  const int tid = threadIdx.x;
  const int64_t total = p.m.pieces * p.ctiles;
  const int64_t tile = LINK ? total - 1 - take_tile(p, &ticket) : (int64_t)blockIdx.x;
  const int64_t j = tile / p.ctiles;
  const int ct = (int)(tile % p.ctiles), c0 = ct * kCh;
  const int seg = tid / 16, lc = tid % 16 * 4, nn = min(4, p.C - c0 - lc);
  const int64_t ch = nn > 0 ? c0 + lc : 0;
  const Piece q = find_piece(p.m, j);
  const bool gated = p.z != nullptr;
  if (seg == 0 && nn > 0)
    for_unused_rows(p.m, j, [&](int64_t row) {
      const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
      store_quad<ACC>(p.dx, row * p.C + ch, p.bf16, nn, zero);
      store_quad<ACC>(p.dr, row * p.C + ch, p.bf16, nn, zero);
      store_quad<ACC>(p.di, row * p.C + ch, p.bf16, nn, zero);
      if (gated) store_quad<ACC>(p.dz, row * p.C + ch, p.bf16, nn, zero);
    });
  if (!q.live || q.len == 0) {
    if (LINK && tid < 2) store_flag(p.flags + (j * p.ctiles + ct) * 2 + tid, 2);
    if (p.part != nullptr && tid < kCh && c0 + tid < p.C)
      for (int n = 0; n < 3; ++n) p.part[(j * 3 + n) * p.C + c0 + tid] = 0.f;
    return;
  }
  const int t0 = q.t0 + seg * kSeg;
  Raw rx[kSeg], rr[kSeg], ri[kSeg], rz[kSeg], rg[kSeg];
#pragma unroll
  for (int u = 0; u < kSeg; ++u) {
    rx[u] = rr[u] = ri[u] = rz[u] = rg[u] = Raw{};
    if (t0 + u < q.t1 && nn > 0) {
      const int64_t row = q.row0 + t0 + u;
      rr[u] = load_quad<ACC>(p.r, row * p.ldr + ch, p.bf16, nn);
      ri[u] = load_quad<ACC>(p.i, row * p.ldi + ch, p.bf16, nn);
      rx[u] = load_quad<ACC>(p.x, row * p.ldx + ch, p.bf16, nn);
      if (gated) rz[u] = load_quad<ACC>(p.z, row * p.ldz + ch, p.bf16, nn);
      rg[u] = load_quad<ACC>(p.dy, row * p.C + ch, p.bf16, nn);
    }
  }
  tile_params<true>(p, c0, par);
  __syncthreads();
  const Quad speed = shared_quad(par[0], lc), rb = shared_quad(par[1], lc), ib = shared_quad(par[2], lc);
  const bool slow = fmaxf(fmaxf(speed.v[0], speed.v[1]), fmaxf(speed.v[2], speed.v[3])) <= 0.35f;
  float a[kSeg][4], b[kSeg][4], d[kSeg][4];  // b: gain iota x; d: the gradient that reaches h from y
  float A[4] = {1.f, 1.f, 1.f, 1.f}, B[4] = {0.f, 0.f, 0.f, 0.f}, G[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < kSeg; ++u) {
    const Quad x = quad(quad_floats<ACC>(rx[u], p.bf16)), r = quad(quad_floats<ACC>(rr[u], p.bf16)),
               i = quad(quad_floats<ACC>(ri[u], p.bf16)), z = quad(quad_floats<ACC>(rz[u], p.bf16)),
               dy = quad(quad_floats<ACC>(rg[u], p.bf16));
    const bool in = t0 + u < q.t1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float left;
      decay(-speed.v[k] * sigmoid(r.v[k] + rb.v[k]), slow, &a[u][k], &left);
      left = left < kLeast ? kLeast : left;
      b[u][k] = left * semx::rsqrt_approx(left) * sigmoid(i.v[k] + ib.v[k]) * x.v[k];
      d[u][k] = gated ? dy.v[k] * (z.v[k] * sigmoid(z.v[k])) : dy.v[k];
      if (!in) a[u][k] = 1.f, b[u][k] = 0.f;
      A[k] *= a[u][k];
      B[k] = fmaf(a[u][k], B[k], b[u][k]);
    }
  }
  // What reaches the step in front of the segment: a_t (d_t + what reaches step t from behind).
#pragma unroll
  for (int u = kSeg - 1; u >= 0; --u)
#pragma unroll
    for (int k = 0; k < 4; ++k) G[k] = a[u][k] * (d[u][k] + G[k]);
  *reinterpret_cast<float4*>(&mA[seg][lc]) = make_float4(A[0], A[1], A[2], A[3]);
  *reinterpret_cast<float4*>(&mB[seg][lc]) = make_float4(B[0], B[1], B[2], B[3]);
  *reinterpret_cast<float4*>(&mG[seg][lc]) = make_float4(G[0], G[1], G[2], G[3]);
  __syncthreads();
  if (tid < kCh) {
    const int c = c0 + tid;
    const bool ok = c < p.C;
    float h = ok ? p.ckpt[j * p.C + c] : 0.f, g = 0.f;
    if (LINK) {
      const int tiles = (int)((q.len + p.m.Q - 1) / p.m.Q);
      const Chain link = {j - q.k + tiles - 1, -1, tiles - 1 - q.k, q.k > 0};
      float fA = 1.f, fG = 0.f;
#pragma unroll
      for (int s = kSegs - 1; s >= 0; --s) {
        fA *= mA[s][tid];
        fG = fmaf(mA[s][tid], fG, mG[s][tid]);
      }
      if (tiles > 1) g = link_in(p, link, ct, tid / 32, c, ok, link.at == 0 ? 0.f : fA, fG);
      link_out(p, link, ct, tid / 32, c, ok, fmaf(fA, g, fG));
    }
#pragma unroll
    for (int s = 0; s < kSegs; ++s) {
      const float next = fmaf(mA[s][tid], h, mB[s][tid]);
      mB[s][tid] = h;
      h = next;
    }
#pragma unroll
    for (int s = kSegs - 1; s >= 0; --s) {
      const float next = fmaf(mA[s][tid], g, mG[s][tid]);
      mG[s][tid] = g;  // from here on what reaches the segment's last step from behind
      g = next;
    }
  }
  __syncthreads();
  {
    Quad h = shared_quad(mB[seg], lc);
#pragma unroll
    for (int u = 0; u < kSeg; ++u)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float next = fmaf(a[u][k], h.v[k], b[u][k]);
        b[u][k] = h.v[k];  // from here on h_{t-1}
        h.v[k] = next;
      }
  }
  Quad g = shared_quad(mG[seg], lc);
  float sum[3][4] = {};
#pragma unroll
  for (int u = kSeg - 1; u >= 0; --u) {
    const Quad x = quad(quad_floats<ACC>(rx[u], p.bf16)), r = quad(quad_floats<ACC>(rr[u], p.bf16)),
               i = quad(quad_floats<ACC>(ri[u], p.bf16)), z = quad(quad_floats<ACC>(rz[u], p.bf16)),
               dy = quad(quad_floats<ACC>(rg[u], p.bf16));
    const bool in = t0 + u < q.t1;
    Quad dx, dr, di, dz;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float gt = d[u][k] + g.v[k];
      float rho, shut_r, iota, shut_i;
      sigmoids(r.v[k] + rb.v[k], &rho, &shut_r);
      sigmoids(i.v[k] + ib.v[k], &iota, &shut_i);
      float at, left;
      decay(-speed.v[k] * rho, slow, &at, &left);
      const bool open = left > kLeast;
      left = left < kLeast ? kLeast : left;
      const float inv = semx::rsqrt_approx(left), gain = left * inv;
      const float ah = at * b[u][k];
      if (gated) {
        float s, rest;
        sigmoids(z.v[k], &s, &rest);
        const float h = fmaf(gain * iota, x.v[k], ah);
        dz.v[k] = dy.v[k] * h * (s * fmaf(z.v[k], rest, 1.f));
      }
      const float gi = gt * iota;
      dx.v[k] = gi * gain;
      di.v[k] = dx.v[k] * x.v[k] * shut_i;
      const float dla = gt * ah - (open ? gi * x.v[k] * (at * at) * inv : 0.f);
      dr.v[k] = -speed.v[k] * dla * rho * shut_r;
      g.v[k] = in ? at * gt : g.v[k];
      if (in) {
        sum[0][k] = fmaf(rho, dla, sum[0][k]);
        sum[1][k] += dr.v[k];
        sum[2][k] += di.v[k];
      }
    }
    if (in && nn > 0) {
      const int64_t o = (q.row0 + t0 + u) * p.C + ch;
      store_quad<ACC>(p.dx, o, p.bf16, nn, make_float4(dx.v[0], dx.v[1], dx.v[2], dx.v[3]));
      store_quad<ACC>(p.dr, o, p.bf16, nn, make_float4(dr.v[0], dr.v[1], dr.v[2], dr.v[3]));
      store_quad<ACC>(p.di, o, p.bf16, nn, make_float4(di.v[0], di.v[1], di.v[2], di.v[3]));
      if (gated) store_quad<ACC>(p.dz, o, p.bf16, nn, make_float4(dz.v[0], dz.v[1], dz.v[2], dz.v[3]));
    }
  }
  if (p.part == nullptr) return;
  __syncthreads();
  *reinterpret_cast<float4*>(&mA[seg][lc]) = make_float4(sum[0][0], sum[0][1], sum[0][2], sum[0][3]);
  *reinterpret_cast<float4*>(&mB[seg][lc]) = make_float4(sum[1][0], sum[1][1], sum[1][2], sum[1][3]);
  *reinterpret_cast<float4*>(&mG[seg][lc]) = make_float4(sum[2][0], sum[2][1], sum[2][2], sum[2][3]);
  __syncthreads();
  if (tid < 3 * kCh) {
    const int n = tid / kCh, k = tid % kCh;
    float(*m)[kCh] = n == 0 ? mA : n == 1 ? mB : mG;
    float acc = 0.f;
#pragma unroll
    for (int s = 0; s < kSegs; ++s) acc += m[s][k];
    if (c0 + k < p.C) p.part[(j * 3 + n) * p.C + c0 + k] = n == 0 ? -par[3][k] * acc : acc;
  }
}

// One token per sequence: a thread has four channels of one, a CTA a run of sequences (their slots
// are looked up together, the parameters read once).
constexpr int kStepT = 128, kStepRows = 8;
template <int ACC>
__global__ void __launch_bounds__(kStepT) gated_lru_step_kernel(const GlParams p, int rows) {
  typedef typename RawQuad<ACC>::type Raw;
  constexpr int F = fp32_beside(ACC);
  __shared__ int64_t slots[kStepRows];
  const int64_t s0 = (int64_t)(blockIdx.x / p.ctiles) * rows;
  const int n = (int)min((int64_t)rows, p.m.S - s0);
  const int64_t c = ((int64_t)(blockIdx.x % p.ctiles) * kStepT + threadIdx.x) * 4;
  const int nn = (int)min((int64_t)4, p.C - c);
  float speed[4] = {}, rb[4] = {}, ib[4] = {};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < nn) {
      const float s = p.scale * semx::softplus(p.rate[c + k]);
      speed[k] = s > 3.4e38f ? 3.4e38f : s;
      if (p.r_bias != nullptr) rb[k] = p.r_bias[c + k];
      if (p.i_bias != nullptr) ib[k] = p.i_bias[c + k];
    }
  semx::find_slots<kStepRows>(p.m, s0, n, slots);
  if (nn <= 0) return;
  constexpr int kAhead = 2;
  for (int n0 = 0; n0 < n; n0 += kAhead) {
    Raw rx[kAhead], rr[kAhead], ri[kAhead], rz[kAhead];
    float4 old[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (n0 + u < n) {
        const int64_t s = s0 + n0 + u, slot = slots[n0 + u];
        rx[u] = load_quad<ACC>(p.x, s * p.ldx + c, p.bf16, nn);
        rr[u] = load_quad<ACC>(p.r, s * p.ldr + c, p.bf16, nn);
        ri[u] = load_quad<ACC>(p.i, s * p.ldi + c, p.bf16, nn);
        if (p.z != nullptr) rz[u] = load_quad<ACC>(p.z, s * p.ldz + c, p.bf16, nn);
        old[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (slot >= 0) old[u] = quad_floats<F>(load_quad<F>(p.state, slot * p.C + c, 0, nn), 0);
      }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (n0 + u < n) {
        const int64_t s = s0 + n0 + u, slot = slots[n0 + u];
        const Quad x = quad(quad_floats<ACC>(rx[u], p.bf16)), r = quad(quad_floats<ACC>(rr[u], p.bf16)),
                   i = quad(quad_floats<ACC>(ri[u], p.bf16));
        Quad h = quad(old[u]), y;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float a, left;
          decay(-speed[k] * sigmoid(r.v[k] + rb[k]), false, &a, &left);
          left = left < kLeast ? kLeast : left;
          h.v[k] = fmaf(a, h.v[k], left * semx::rsqrt_approx(left) * sigmoid(i.v[k] + ib[k]) * x.v[k]);
          if (slot == semx::kRefused) h.v[k] = __int_as_float(0x7fffffff);
          y.v[k] = h.v[k];
        }
        if (p.z != nullptr) {
          const Quad z = quad(quad_floats<ACC>(rz[u], p.bf16));
#pragma unroll
          for (int k = 0; k < 4; ++k) y.v[k] *= z.v[k] * sigmoid(z.v[k]);
        }
        if (slot >= 0)
          store_quad<F>(p.state, slot * p.C + c, 0, nn, make_float4(h.v[0], h.v[1], h.v[2], h.v[3]));
        store_quad<ACC>(p.y, s * p.C + c, p.bf16, nn, make_float4(y.v[0], y.v[1], y.v[2], y.v[3]));
      }
  }
}

int gl_validate(const SemxGatedLruArgs* a, bool bwd, GlParams* p) {
  SEMX_REQUIRE(a->C >= 1 && a->C < (1 << 24), SEMX_ERR_SHAPE, "gated_lru: C=%lld", (long long)a->C);
  const int64_t top = (int64_t)1 << 31;
  SEMX_REQUIRE(a->ldx >= a->C && a->ldr >= a->C && a->ldi >= a->C && (a->z == nullptr || a->ldz >= a->C) &&
                   a->ldx < top && a->ldr < top && a->ldi < top && a->ldz < top,
               SEMX_ERR_SHAPE, "gated_lru: row strides %lld %lld %lld %lld", (long long)a->ldx, (long long)a->ldr,
               (long long)a->ldi, (long long)a->ldz);
  SEMX_REQUIRE(a->rate_scale > 0.f && a->rate_scale < 3.4e38f, SEMX_ERR_SHAPE, "gated_lru: rate_scale=%g",
               (double)a->rate_scale);
  int rc = semx::check_seqs("gated_lru", a->S, a->rows, a->L, a->cu_seqlens, a->state, a->slots, a->fresh, a->n_slots,
                            &p->m);
  if (rc != SEMX_OK) return rc;
  SEMX_REQUIRE(!bwd || a->state == nullptr, SEMX_ERR_UNSUPPORTED, "gated_lru bwd: no state");
  const bool none = a->rows == 0;
  SEMX_REQUIRE(a->rate && (none || (a->x && a->r && a->i)), SEMX_ERR_NULL, "gated_lru: x / r / i / rate is NULL");
  if (!bwd) {
    SEMX_REQUIRE(none || a->y, SEMX_ERR_NULL, "gated_lru: y is NULL");
  } else {
    SEMX_REQUIRE(none || (a->dy && a->dx && a->d_r && a->d_i && a->ckpt && (a->z == nullptr || a->dz)), SEMX_ERR_NULL,
                 "gated_lru bwd: dy / dx / d_r / d_i / dz / ckpt is NULL");
  }
  SEMX_REQUIRE(semx::all_aligned({a->x, a->r, a->i, a->z, a->y, a->dy, a->dx, a->d_r, a->d_i, a->dz}, a->bf16 ? 2 : 4) &&
                   semx::all_aligned({a->rate, a->r_bias, a->i_bias, a->cu_seqlens, a->state, a->slots, a->ckpt,
                                      a->drate, a->dr_bias, a->di_bias}, 4) &&
                   semx::aligned(a->workspace, 8),
               SEMX_ERR_ALIGN, "gated_lru: a pointer is not on an element");
  p->C = (int)a->C; p->bf16 = a->bf16; p->scale = a->rate_scale;
  p->ctiles = (int)semx::cdiv(a->C, (int64_t)kCh);
  p->ldx = a->ldx; p->ldr = a->ldr; p->ldi = a->ldi; p->ldz = a->ldz;
  p->x = a->x; p->r = a->r; p->i = a->i; p->z = a->z;
  p->rate = a->rate; p->r_bias = a->r_bias; p->i_bias = a->i_bias;
  p->y = a->y; p->state = a->state; p->ckpt = a->ckpt;
  p->dy = a->dy; p->dx = a->dx; p->dr = a->d_r; p->di = a->d_i; p->dz = a->dz;
  // Four neighbours per access where every row and base is on four elements.
  p->access = kAny;
  if (a->C % 4 == 0 && a->ldx % 4 == 0 && a->ldr % 4 == 0 && a->ldi % 4 == 0 && (a->z == nullptr || a->ldz % 4 == 0) &&
      semx::all_aligned({a->x, a->r, a->i, a->z, a->y, a->dy, a->dx, a->d_r, a->d_i, a->dz}, a->bf16 ? 8 : 16) &&
      semx::aligned(a->state, 16))
    p->access = a->bf16 ? kBf16 : kFp32;
  semx::set_pieces(&p->m, kRows);
  return SEMX_OK;
}

// Whether a sequence can have more than one tile.
bool gl_linked(const GlParams& p) { return p.m.cu != nullptr ? p.m.T > kRows : p.m.L > kRows; }

size_t round8(size_t n) { return (n + 7) / 8 * 8; }
size_t link_ints(const GlParams& p) { return round8(1 + (size_t)p.m.pieces * p.ctiles * 2); }
size_t link_bytes(const GlParams& p) {
  return gl_linked(p) ? link_ints(p) * sizeof(int) + (size_t)p.m.pieces * p.C * (sizeof(float2) + sizeof(float)) : 0;
}

// Lays the links into the workspace and clears ticket and flags.
int set_links(GlParams* p, void* workspace, cudaStream_t st) {
  if (!gl_linked(*p)) return SEMX_OK;
  SEMX_REQUIRE(workspace != nullptr, SEMX_ERR_WORKSPACE, "gated_lru: workspace is NULL");
  const size_t ints = link_ints(*p);
  p->ticket = reinterpret_cast<int*>(workspace);
  p->flags = p->ticket + 1;
  p->maps = reinterpret_cast<float2*>(p->ticket + ints);
  p->left = reinterpret_cast<float*>(p->maps + (size_t)p->m.pieces * p->C);
  const cudaError_t e = cudaMemsetAsync(workspace, 0, ints * sizeof(int), st);
  SEMX_REQUIRE(e == cudaSuccess, SEMX_ERR_LAUNCH, "gated_lru: cudaMemsetAsync: %s", cudaGetErrorString(e));
  return SEMX_OK;
}

template <int ACC>
int launch_gl(bool bwd, const GlParams& p, cudaStream_t st) {
  const int64_t grid = p.m.pieces * p.ctiles;
  if (grid == 0) return SEMX_OK;
  if (grid >= ((int64_t)1 << 30)) return semx::fail(SEMX_ERR_SHAPE, "gated_lru: too many tiles");
  const unsigned n = (unsigned)grid;
  const bool linked = p.ticket != nullptr;
  if (!bwd) {
    if (linked) gated_lru_fwd_kernel<ACC, true><<<n, kT, 0, st>>>(p);
    else gated_lru_fwd_kernel<ACC, false><<<n, kT, 0, st>>>(p);
    return semx::check_launch("gated_lru_fwd_kernel");
  }
  if (linked) gated_lru_bwd_kernel<ACC, true><<<n, kT, 0, st>>>(p);
  else gated_lru_bwd_kernel<ACC, false><<<n, kT, 0, st>>>(p);
  return semx::check_launch("gated_lru_bwd_kernel");
}

int dispatch_gl(bool bwd, const GlParams& p, cudaStream_t st) {
  if (p.access == kBf16) return launch_gl<kBf16>(bwd, p, st);
  if (p.access == kFp32) return launch_gl<kFp32>(bwd, p, st);
  return launch_gl<kAny>(bwd, p, st);
}

GlParams gl_sizes(const SemxGatedLruArgs* a, bool bwd, int* rc) {
  SemxGatedLruArgs b = *a;
  float* any = reinterpret_cast<float*>(256);
  b.x = b.r = b.i = any;
  b.rate = any;
  b.y = any;
  b.dy = any;
  b.dx = b.d_r = b.d_i = b.dz = any;
  b.ckpt = any;
  GlParams p = {};
  *rc = gl_validate(&b, bwd, &p);
  return p;
}

}  // namespace

namespace semx {
int link_timeouts(uint32_t* count) {
  unsigned v = 0;
  const cudaError_t e = cudaMemcpyFromSymbol(&v, g_link_timeouts, sizeof(v));
  if (e != cudaSuccess) return fail(SEMX_ERR_LAUNCH, "link_timeouts: %s", cudaGetErrorString(e));
  *count = v;
  return SEMX_OK;
}
}  // namespace semx

extern "C" {

size_t semx_gated_lru_args_size(void) { return sizeof(SemxGatedLruArgs); }

size_t semx_gated_lru_ckpt_bytes(const SemxGatedLruArgs* a) {
  if (a == nullptr) return 0;
  int rc;
  const GlParams p = gl_sizes(a, false, &rc);
  return rc == SEMX_OK ? (size_t)p.m.pieces * p.C * sizeof(float) : 0;
}

size_t semx_gated_lru_workspace_bytes(const SemxGatedLruArgs* a, int32_t backward) {
  if (a == nullptr) return 0;
  int rc;
  const GlParams p = gl_sizes(a, backward != 0, &rc);
  if (rc != SEMX_OK) return 0;
  return link_bytes(p) + (backward != 0 ? (size_t)p.m.pieces * 3 * p.C * sizeof(float) : 0);
}

int semx_gated_lru_fwd(const SemxGatedLruArgs* a, semx_stream_t stream) {
  SEMX_CHECK_ARGS(a, SemxGatedLruArgs);
  GlParams p = {};
  int rc = gl_validate(a, false, &p);
  if (rc != SEMX_OK || semx::nothing_to_do(p.m)) return rc;
  semx::DeviceScope scope;
  rc = scope.bind({a->y, a->state});
  if (rc != SEMX_OK) return rc;
  cudaStream_t st = semx::as_stream(stream);
  rc = set_links(&p, a->workspace, st);
  if (rc != SEMX_OK) return rc;
  // Without a sequence every row is a row behind the last one.
  if (p.m.S == 0 && p.m.T > 0 && p.m.pieces == 0) p.m.pieces = 1;
  return dispatch_gl(false, p, st);
}

int semx_gated_lru_bwd(const SemxGatedLruArgs* a, semx_stream_t stream) {
  SEMX_CHECK_ARGS(a, SemxGatedLruArgs);
  GlParams p = {};
  int rc = gl_validate(a, true, &p);
  if (rc != SEMX_OK) return rc;
  const bool params = a->drate != nullptr || a->dr_bias != nullptr || a->di_bias != nullptr;
  semx::DeviceScope scope;
  rc = scope.bind({a->dx, a->drate, a->dr_bias, a->di_bias});
  if (rc != SEMX_OK) return rc;
  cudaStream_t st = semx::as_stream(stream);
  if (p.m.T > 0) {
    rc = set_links(&p, a->workspace, st);
    if (rc != SEMX_OK) return rc;
    if (params) {
      SEMX_REQUIRE(a->workspace != nullptr, SEMX_ERR_WORKSPACE, "gated_lru bwd: workspace is NULL");
      p.part = reinterpret_cast<float*>(reinterpret_cast<char*>(a->workspace) + link_bytes(p));
    }
    const int64_t pieces = p.m.pieces;
    if (p.m.S == 0 && pieces == 0) p.m.pieces = 1, p.part = nullptr;
    rc = dispatch_gl(true, p, st);
    p.m.pieces = pieces;
    if (rc != SEMX_OK) return rc;
  }
  if (!params) return SEMX_OK;
  semx::Segments seg = {};
  seg.n = 3;
  seg.out[0] = a->drate;
  seg.out[1] = a->dr_bias;
  seg.out[2] = a->di_bias;
  seg.len[0] = seg.len[1] = seg.len[2] = a->C;
  return semx::colsum_once(p.part, p.m.T > 0 ? p.m.pieces : 0, 3 * a->C, seg, st);
}

int semx_gated_lru_step(const SemxGatedLruArgs* a, semx_stream_t stream) {
  SEMX_CHECK_ARGS(a, SemxGatedLruArgs);
  GlParams p = {};
  int rc = gl_validate(a, false, &p);
  if (rc != SEMX_OK) return rc;
  SEMX_REQUIRE(a->cu_seqlens == nullptr && (a->L == 1 || a->S == 0), SEMX_ERR_SHAPE, "gated_lru_step: one row per sequence");
  SEMX_REQUIRE(a->state != nullptr, SEMX_ERR_NULL, "gated_lru_step: state is NULL");
  SEMX_REQUIRE(a->fresh == nullptr, SEMX_ERR_UNSUPPORTED, "gated_lru_step: no fresh flags");
  if (p.m.S == 0) return SEMX_OK;
  semx::DeviceScope scope;
  rc = scope.bind({a->y});
  if (rc != SEMX_OK) return rc;
  cudaStream_t st = semx::as_stream(stream);
  p.ctiles = (int)semx::cdiv(a->C, (int64_t)kStepT * 4);
  int rows = kStepRows;
  while (rows > 1 && semx::cdiv(p.m.S, rows) * p.ctiles < 148 * 4) rows /= 2;
  const int64_t grid = semx::cdiv(p.m.S, rows) * p.ctiles;
  if (grid >= ((int64_t)1 << 31)) return semx::fail(SEMX_ERR_SHAPE, "gated_lru_step: too many sequences");
  const unsigned n = (unsigned)grid;
  if (p.access == kBf16) gated_lru_step_kernel<kBf16><<<n, kStepT, 0, st>>>(p, rows);
  else if (p.access == kFp32) gated_lru_step_kernel<kFp32><<<n, kStepT, 0, st>>>(p, rows);
  else gated_lru_step_kernel<kAny><<<n, kStepT, 0, st>>>(p, rows);
  return semx::check_launch("gated_lru_step_kernel");
}

}  // extern "C"
