// Backward of the selective state scan, for sm_100a.
//
// With dv = dy silu(z) (dy without z), from the last step of a sequence to its first:
//   g = C dv + carry;  carry = exp(d A) g  (the gradient of the state in front of the step)
//   u = carry h_prev;  gB = sum_n g B;  uA = sum_n u A
//   dB += g d x, dC += dv h (summed over the channels of the group), dA += u d,
//   dx = d gB + D dv, dd = uA + x gB, ddt = dd softplus'(dt + bias), dz = dy v silu'(z),
//   dD += dv x, ddt_bias += ddt
//
// Bound: instruction issue, then the special-function unit. The forward left the state in
// front of every kBlock steps, so a block's states and poles are rebuilt from it in
// registers and the adjoint runs back through them: every exponential is evaluated once
// (one that kept fewer states would evaluate them twice).
//
// Split: a thread owns kCPT channels and 4 modes of them, GM neighbouring lanes the modes
// of a channel. Sums over modes (gB, uA) are exchanged between those lanes, sums over
// channels (dB, dC) between the other lanes of the warp, each by halving: a lane hands over
// half of its values and adds the other half, so that k values over as many lanes cost
// k - 1 exchanges. Two channels per thread halve the values that have to be exchanged.
// The four warps' sums are joined in shared memory, the channel tiles' by a second kernel
// in tile order; the parameters' gradients are one row per piece, reduced by the
// fixed-order column sum. Nothing depends on the order in which CTAs run.
// As in the forward, few long sequences are cut into pieces: a first pass (LOCAL) runs the
// carry of each piece from zero, the pieces are joined from the last one, and each piece
// then starts from its true carry.
#include "state_scan.cuh"
#include "semx_reduce.cuh"

namespace {

using namespace semx_scan;

constexpr int kWarps = kThreads / 32;
constexpr float kLn2 = 0.6931471805599453f;

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

template <int GM>
constexpr int channels_per_thread() {
  return GM == 1 ? 1 : 2;
}
template <int GM>
constexpr int channels_per_cta() {
  return kWarps * (32 / GM) * channels_per_thread<GM>();
}

// Sums v over LANES lanes that are STRIDE apart, by halving; afterwards v[0 .. NV / LANES)
// (at least one) of a lane are the totals of values [idx, idx + NV / LANES), idx the top
// bits of its number among the lanes. More lanes than values: the rest hold the same totals.
template <int NV, int LANES, int STRIDE>
__device__ __forceinline__ void halve_sum(float (&v)[NV], int lane) {
  if constexpr (LANES > 1 && NV > 1) {
    constexpr int M = LANES / 2 * STRIDE, H = NV / 2;
    const bool hi = lane & M;
    float w[H];
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const float keep = hi ? v[H + i] : v[i], send = hi ? v[i] : v[H + i];
      w[i] = keep + __shfl_xor_sync(0xffffffffu, send, M);
    }
    halve_sum<H, LANES / 2, STRIDE>(w, lane);
#pragma unroll
    for (int i = 0; i < H; ++i) v[i] = w[i];
  } else if constexpr (LANES > 1) {
#pragma unroll
    for (int m = LANES / 2; m >= 1; m /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], m * STRIDE);
  }
}

template <int GM, bool LOCAL>
__global__ void __launch_bounds__(kThreads) state_scan_bwd_kernel(const ScanParams p) {
  constexpr int CPT = channels_per_thread<GM>(), CL = 32 / GM, CH = channels_per_cta<GM>(), NP = 4 * GM;
  constexpr int TS = kThreads / CH;  // steps between a thread's (step, channel) pairs
  constexpr int E = kBlock / TS > 0 ? kBlock / TS : 1;
  constexpr int EB = (kBlock * NP + kThreads - 1) / kThreads;
  constexpr int NV1 = 2 * CPT, NO1 = NV1 / GM > 0 ? NV1 / GM : 1;
  constexpr int NO2 = 8 / CL > 0 ? 8 / CL : 1;
  __shared__ __align__(16) float4 sp[kBlock][CH];  // (d, d x, dv, -)
  __shared__ __align__(16) float sB[kBlock][NP];
  __shared__ __align__(16) float sC[kBlock][NP];
  __shared__ float2 so[LOCAL ? 1 : kBlock][LOCAL ? 1 : CH];                      // (gB, uA)
  __shared__ float sw[LOCAL ? 1 : kWarps][LOCAL ? 1 : kBlock][LOCAL ? 1 : 2 * NP];  // dB | dC of a warp

  const int64_t j = blockIdx.x / p.ctiles;
  const int ct = blockIdx.x % p.ctiles;
  const int grp = ct / p.tpg, cg0 = (ct % p.tpg) * CH, c_base = grp * p.cpg;
  const Piece q = find_piece(p.m, j);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;

  const int ec = tid % CH, et = tid / CH;
  const bool eok = cg0 + ec < p.cpg;
  const int ech = c_base + min(cg0 + ec, p.cpg - 1);
  if (!LOCAL && eok && et == 0)
    for (int64_t r = rows_end(p.m) + j; r < p.m.T; r += p.m.pieces) {
      store(p.dx, r * p.C + ech, p.bf16, 0.f);
      store(p.ddt, r * p.C + ech, p.dt_bf16, 0.f);
      if (p.z != nullptr) store(p.dz, r * p.C + ech, p.bf16, 0.f);
    }

  const int lm = lane % GM, cl = lane / GM;
  const int sc = (warp * CL + cl) * CPT;  // first of the thread's channels in the tile
  const int n0 = lm * 4;
  bool cok[CPT];
  int ch[CPT];
  float A2[CPT][4], dA[CPT][4], carry[CPT][4];
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    cok[i] = cg0 + sc + i < p.cpg;
    ch[i] = c_base + min(cg0 + sc + i, p.cpg - 1);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const bool ok = n0 + n < p.N;
      A2[i][n] = ok ? p.A[(int64_t)ch[i] * p.N + n0 + n] * kLog2e : 0.f;
      dA[i][n] = 0.f;
      carry[i][n] = !LOCAL && ok && q.live && p.entry != nullptr ? p.entry[(j * p.C + ch[i]) * p.N + n0 + n] : 0.f;
    }
  }
  const float bias = p.dt_bias != nullptr ? p.dt_bias[ech] : 0.f;
  const float Dc = p.D != nullptr ? p.D[ech] : 0.f;
  float accD = 0.f, accb = 0.f, dsum = 0.f;

  uint32_t rx[E], rd[E], rg[E], rz[E], rv[E], rB[EB], rC[EB];
  float hn[CPT][4];
  const int64_t blk0 = q.live ? piece_base(p.m, q.s, kBlock) : 0;
  auto fetch = [&](int t0) {
    const int64_t row = q.row0 + t0 + et;
    const bool ok = eok && et < kBlock;
    fetch_pairs<E, TS>(rd, p.dt, p.dt_bf16, row * p.lddt + ech, TS * p.lddt, t0 + et, q.t1, ok);
    fetch_pairs<E, TS>(rg, p.dy, p.bf16, row * p.C + ech, (int64_t)TS * p.C, t0 + et, q.t1, ok);
    if (p.z != nullptr) fetch_pairs<E, TS>(rz, p.z, p.bf16, row * p.ldz + ech, TS * p.ldz, t0 + et, q.t1, ok);
    if (!LOCAL) {
      fetch_pairs<E, TS>(rx, p.x, p.bf16, row * p.ldx + ech, TS * p.ldx, t0 + et, q.t1, ok);
      if (p.z != nullptr) fetch_pairs<E, TS>(rv, p.v, p.bf16, row * p.C + ech, (int64_t)TS * p.C, t0 + et, q.t1, ok);
    }
#pragma unroll
    for (int i = 0; i < EB; ++i) {
      const int e = tid + i * kThreads, t = e / NP, n = e % NP;
      const bool in = t < kBlock && n < p.N && t0 + t < q.t1;
      const int64_t r = q.row0 + t0 + t;
      if (!LOCAL) rB[i] = in ? load_raw(p.B, r * p.ldb + (int64_t)grp * p.N + n, p.bf16) : 0u;
      rC[i] = in ? load_raw(p.Cm, r * p.ldc + (int64_t)grp * p.N + n, p.bf16) : 0u;
    }
    if (!LOCAL) {
#pragma unroll
      for (int i = 0; i < CPT; ++i)
#pragma unroll
        for (int n = 0; n < 4; ++n)
          hn[i][n] = n0 + n < p.N ? p.ckpt[((blk0 + t0 / kBlock) * p.C + ch[i]) * p.N + n0 + n] : 0.f;
    }
  };

  const int tl = q.t1 > q.t0 ? q.t0 + (q.t1 - 1 - q.t0) / kBlock * kBlock : q.t0 - kBlock;
  if (tl >= q.t0) fetch(tl);
  for (int t0 = tl; t0 >= q.t0; t0 -= kBlock) {
    float xv[E], dv[E], gv[E], sg[E];  // x, d, dv, softplus'
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int t = et + i * TS;
      if (t < kBlock) {
        const bool in = t0 + t < q.t1 && eok;
        const float raw = as_float(rd[i], p.dt_bf16) + bias;
        float d = p.softplus ? softplus2(raw, raw).x : raw;
        if (!in) d = 0.f;
        float g = as_float(rg[i], p.bf16);
        if (p.z != nullptr) {
          const float z = as_float(rz[i], p.bf16), s = sigmoid(z);
          if (!LOCAL && in)
            store(p.dz, (q.row0 + t0 + t) * p.C + ech, p.bf16,
                  g * as_float(rv[i], p.bf16) * (s * fmaf(z, 1.f - s, 1.f)));
          g *= z * s;
        }
        if (!in) g = 0.f;
        const float x = LOCAL ? 0.f : as_float(rx[i], p.bf16);
        sp[t][ec] = make_float4(d, d * x, g, 0.f);
        xv[i] = x;
        dv[i] = d;
        gv[i] = g;
        sg[i] = !LOCAL && p.softplus ? semx::softplus_grad(raw) : 1.f;
        if (LOCAL) dsum += d;
      }
    }
#pragma unroll
    for (int i = 0; i < EB; ++i) {
      const int e = tid + i * kThreads;
      if (e < kBlock * NP) {
        if (!LOCAL) (&sB[0][0])[e] = as_float(rB[i], p.bf16);
        (&sC[0][0])[e] = as_float(rC[i], p.bf16);
      }
    }
    float a[kBlock][CPT][4], h[kBlock + 1][CPT][4];
    if (!LOCAL) {
#pragma unroll
      for (int i = 0; i < CPT; ++i)
#pragma unroll
        for (int n = 0; n < 4; ++n) h[0][i][n] = hn[i][n];
    }
    __syncthreads();
    if (t0 - kBlock >= q.t0) fetch(t0 - kBlock);
#pragma unroll
    for (int t = 0; t < kBlock; ++t) {
      float4 B4 = make_float4(0.f, 0.f, 0.f, 0.f);
      if (!LOCAL) B4 = *reinterpret_cast<const float4*>(&sB[t][n0]);
      const float Bn[4] = {B4.x, B4.y, B4.z, B4.w};
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        const float4 s = sp[t][sc + i];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          a[t][i][n] = pole(s.x, A2[i][n]);
          if (!LOCAL) h[t + 1][i][n] = fmaf(a[t][i][n], h[t][i][n], s.y * Bn[n]);
        }
      }
    }
#pragma unroll
    for (int t = kBlock - 1; t >= 0; --t) {
      const float4 C4 = *reinterpret_cast<const float4*>(&sC[t][n0]);
      const float Cn[4] = {C4.x, C4.y, C4.z, C4.w};
      if (LOCAL) {
#pragma unroll
        for (int i = 0; i < CPT; ++i) {
          const float4 s = sp[t][sc + i];
#pragma unroll
          for (int n = 0; n < 4; ++n) carry[i][n] = a[t][i][n] * fmaf(Cn[n], s.z, carry[i][n]);
        }
      } else {
        const float4 B4 = *reinterpret_cast<const float4*>(&sB[t][n0]);
        const float Bn[4] = {B4.x, B4.y, B4.z, B4.w};
        float v1[NV1], v2[8];
#pragma unroll
        for (int i = 0; i < CPT; ++i) {
          const float4 s = sp[t][sc + i];
          float gB = 0.f, uA = 0.f;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float g = fmaf(Cn[n], s.z, carry[i][n]);
            carry[i][n] = a[t][i][n] * g;
            const float u = carry[i][n] * h[t][i][n];
            gB = fmaf(g, Bn[n], gB);
            uA = fmaf(u, A2[i][n], uA);
            dA[i][n] = fmaf(u, s.x, dA[i][n]);
            v2[n] = i == 0 ? g * s.y : fmaf(g, s.y, v2[n]);
            v2[4 + n] = i == 0 ? h[t + 1][i][n] * s.z : fmaf(h[t + 1][i][n], s.z, v2[4 + n]);
          }
          v1[2 * i] = gB;
          v1[2 * i + 1] = uA;
        }
        halve_sum<NV1, GM, 1>(v1, lane);
        halve_sum<8, CL, GM>(v2, lane);
        // Value k of (channel, {gB, uA}) is float sc * 2 + k of the step's row.
        constexpr int SPARE1 = GM > NV1 ? GM / NV1 : 1;
        if (lm % SPARE1 == 0) {
#pragma unroll
          for (int k = 0; k < NO1; ++k) reinterpret_cast<float*>(&so[t][sc])[lm / SPARE1 * NO1 + k] = v1[k];
        }
        constexpr int SPARE2 = CL > 8 ? CL / 8 : 1;
        if (cl % SPARE2 == 0) {
#pragma unroll
          for (int k = 0; k < NO2; ++k) {
            const int id = cl / SPARE2 * NO2 + k;  // (dB, dC) x 4 modes
            sw[warp][t][(id / 4) * NP + n0 + id % 4] = v2[k];
          }
        }
      }
    }
    __syncthreads();
    if (!LOCAL) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int t = et + i * TS;
        if (t < kBlock && t0 + t < q.t1 && eok) {
          const int64_t o = (q.row0 + t0 + t) * p.C + ech;
          const float2 s = so[t][ec];
          store(p.dx, o, p.bf16, fmaf(dv[i], s.x, Dc * gv[i]));
          const float ddt = fmaf(s.y, kLn2, xv[i] * s.x) * sg[i];
          store(p.ddt, o, p.dt_bf16, ddt);
          accb += ddt;
          accD = fmaf(gv[i], xv[i], accD);
        }
      }
      for (int e = tid; e < kBlock * 2 * NP; e += kThreads) {
        const int t = e / (2 * NP), v = e % (2 * NP), n = v % NP;
        if (n < p.N && t0 + t < q.t1) {
          float s = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) s += sw[w][t][v];
          p.pBC[((int64_t)ct * p.m.T + q.row0 + t0 + t) * 2 * p.N + (v / NP) * p.N + n] = s;
        }
      }
    }
  }
  float* red = reinterpret_cast<float*>(&sp[0][0]);
  if (LOCAL) {
    if (!q.live) return;
#pragma unroll
    for (int i = 0; i < CPT; ++i)
      if (cok[i])
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (n0 + n < p.N) p.entry[(j * p.C + ch[i]) * p.N + n0 + n] = carry[i][n];
    red[tid] = dsum;
    __syncthreads();
    if (tid < CH && eok) {
      float s = 0.f;
      for (int i = 0; i < TS; ++i) s += red[i * CH + tid];
      p.dsum[j * p.C + ech] = s;
    }
  } else if (p.part != nullptr) {
    // Every piece index writes its row, zeros where there is no such piece.
    float* row = p.part + j * ((int64_t)p.C * (p.N + 2));
#pragma unroll
    for (int i = 0; i < CPT; ++i)
      if (cok[i])
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (n0 + n < p.N) row[(int64_t)ch[i] * p.N + n0 + n] = dA[i][n];
    __syncthreads();
    red[tid] = accD;
    red[kThreads + tid] = accb;
    __syncthreads();
    if (tid < CH && eok) {
      float s = 0.f, b = 0.f;
      for (int i = 0; i < TS; ++i) {
        s += red[i * CH + tid];
        b += red[kThreads + i * CH + tid];
      }
      row[(int64_t)p.C * p.N + ech] = s;
      row[(int64_t)p.C * (p.N + 1) + ech] = b;
    }
  }
}

// Joins the pieces' carries from the last piece of a sequence: entry[j] becomes the gradient
// of the state behind piece j. One thread per (sequence, channel, mode).
__global__ void __launch_bounds__(kThreads) state_scan_join_back_kernel(const ScanParams p) {
  const int64_t per = (int64_t)p.C * p.N;
  const int64_t tiles = (per + kThreads - 1) / kThreads;
  const int64_t s = blockIdx.x / tiles;
  const int64_t i = (blockIdx.x % tiles) * kThreads + threadIdx.x;
  if (i >= per) return;
  const int64_t c = i / p.N;
  const float A2 = p.A[i] * kLog2e;
  const int64_t row0 = seq_start(p.m, s);
  const int64_t len = p.m.cu == nullptr ? p.m.L : max(seq_start(p.m, s + 1), row0) - row0;
  const int64_t base = piece_base(p.m, s, p.m.Q), n = (len + p.m.Q - 1) / p.m.Q;
  float carry = 0.f;
  for (int64_t k = n - 1; k >= 0; --k) {
    const int64_t j = base + k;
    const float local = p.entry[j * per + i];
    p.entry[j * per + i] = carry;
    carry = fmaf(semx::ex2_approx(p.dsum[j * p.C + c] * A2), carry, local);
  }
}

// dB and dC: the channel tiles' sums in tile order.
__global__ void __launch_bounds__(256) state_scan_bc_kernel(const ScanParams p, void* dB, void* dC) {
  const int64_t per = (int64_t)p.G * p.N;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= 2 * per * p.m.T) return;
  const int64_t kind = e / (per * p.m.T), r = e % (per * p.m.T) / per, gn = e % per;
  const int64_t g = gn / p.N, n = gn % p.N;
  float s = 0.f;
  if (r < rows_end(p.m))
    for (int i = 0; i < p.tpg; ++i) s += p.pBC[((g * p.tpg + i) * p.m.T + r) * 2 * p.N + kind * p.N + n];
  store(kind == 0 ? dB : dC, r * per + gn, p.bf16, s);
}

int tile_channels(int N) {
  const int gm = lanes_for(N, 4);
  return kWarps * (32 / gm) * (gm == 1 ? 1 : 2);
}

void set_tiles(ScanParams& p) {
  p.tpg = (int)semx::cdiv(p.cpg, (int64_t)tile_channels(p.N));
  p.ctiles = p.G * p.tpg;
}

int64_t bwd_rows_per_piece(const ScanParams& p) {
  const int64_t ctas = (int64_t)p.m.S * p.ctiles;
  const int64_t rows = p.m.S > 0 ? p.m.T / p.m.S : 0;
  if (ctas >= 148 * 2 || rows <= 64) return 0;
  const int64_t cut = semx::cdiv((int64_t)148 * 4, ctas > 0 ? ctas : 1);
  const int64_t Q = semx::cdiv(semx::cdiv(p.m.T, p.m.S * cut), kBlock) * kBlock;
  return Q < 32 ? 32 : Q;
}

struct Layout {
  size_t entry, dsum, pbc, part, groups, total;
};
Layout layout(const ScanParams& p, int64_t Q) {
  Layout l = {};
  const size_t pieces = (size_t)p.m.pieces;
  size_t at = 0;
  l.entry = at;
  at += Q > 0 ? pieces * p.C * p.N : 0;
  l.dsum = at;
  at += Q > 0 ? pieces * p.C : 0;
  l.pbc = at;
  at += (size_t)p.ctiles * p.m.T * 2 * p.N;
  l.part = at;
  at += pieces * p.C * (p.N + 2);
  l.groups = at;
  at += semx::colsum_group_floats(p.m.pieces, (int64_t)p.C * (p.N + 2));
  l.total = at;
  return l;
}

template <bool LOCAL>
int launch_bwd(const ScanParams& p, cudaStream_t st) {
  const int gm = lanes_for(p.N, 4);
  const int64_t grid = p.m.pieces * p.ctiles;
  if (grid == 0) return SEMX_OK;
  if (grid >= ((int64_t)1 << 31)) return semx::fail(SEMX_ERR_SHAPE, "state_scan bwd: too many pieces");
  switch (gm) {
#define SEMX_GM(V)                                                                       \
  case V:                                                                                \
    state_scan_bwd_kernel<V, LOCAL><<<(unsigned)grid, kThreads, 0, st>>>(p);             \
    return semx::check_launch("state_scan_bwd_kernel");
    SEMX_GM(1)
    SEMX_GM(2)
    SEMX_GM(4)
    SEMX_GM(8)
    SEMX_GM(16)
    SEMX_GM(32)
#undef SEMX_GM
  }
  return semx::fail(SEMX_ERR_UNSUPPORTED, "state_scan bwd: %d modes", p.N);
}

}  // namespace

namespace semx_scan {

size_t scan_bwd_workspace(ScanParams& p) {
  set_tiles(p);
  const int64_t Q = bwd_rows_per_piece(p);
  semx::set_pieces(&p.m, Q);
  if (p.m.S == 0 && p.m.T > 0) p.m.pieces = 1;
  return layout(p, Q).total * sizeof(float);
}

}  // namespace semx_scan

extern "C" {

int semx_state_scan_bwd(const SemxStateScanArgs* a, semx_stream_t stream) {
  SEMX_CHECK_ARGS(a, SemxStateScanArgs);
  ScanParams p = {};
  int rc = scan_validate(a, true, &p);
  if (rc != SEMX_OK) return rc;
  SEMX_REQUIRE(a->workspace != nullptr, SEMX_ERR_WORKSPACE, "state_scan bwd: workspace is NULL");
  semx::DeviceScope scope;
  rc = scope.bind({a->dx, a->dA, a->dD, a->ddt_bias});
  if (rc != SEMX_OK) return rc;
  cudaStream_t st = semx::as_stream(stream);
  set_tiles(p);
  const int64_t Q = bwd_rows_per_piece(p);
  semx::set_pieces(&p.m, Q);
  if (p.m.S == 0 && p.m.T > 0) p.m.pieces = 1;
  const Layout l = layout(p, Q);
  float* ws = reinterpret_cast<float*>(a->workspace);
  p.pBC = ws + l.pbc;
  const bool params = a->dA != nullptr || a->dD != nullptr || a->ddt_bias != nullptr;
  p.part = params ? ws + l.part : nullptr;
  if (p.m.T > 0) {
    if (Q > 0 && p.m.S > 0) {
      p.entry = ws + l.entry;
      p.dsum = ws + l.dsum;
      rc = launch_bwd<true>(p, st);
      if (rc != SEMX_OK) return rc;
      const int64_t grid = p.m.S * semx::cdiv((int64_t)p.C * p.N, kThreads);
      if (grid >= ((int64_t)1 << 31)) return semx::fail(SEMX_ERR_SHAPE, "state_scan bwd: too many sequences");
      state_scan_join_back_kernel<<<(unsigned)grid, kThreads, 0, st>>>(p);
      rc = semx::check_launch("state_scan_join_back_kernel");
      if (rc != SEMX_OK) return rc;
    }
    rc = launch_bwd<false>(p, st);
    if (rc != SEMX_OK) return rc;
    const int64_t grid = semx::cdiv(2 * (int64_t)p.G * p.N * p.m.T, 256);
    if (grid >= ((int64_t)1 << 31)) return semx::fail(SEMX_ERR_SHAPE, "state_scan bwd: too many rows");
    state_scan_bc_kernel<<<(unsigned)grid, 256, 0, st>>>(p, a->dB, a->dC);
    rc = semx::check_launch("state_scan_bc_kernel");
    if (rc != SEMX_OK) return rc;
  }
  if (!params) return SEMX_OK;
  semx::Segments seg = {};
  seg.n = 3;
  seg.out[0] = a->dA;
  seg.out[1] = a->dD;
  seg.out[2] = a->ddt_bias;
  seg.len[0] = a->C * a->N;
  seg.len[1] = seg.len[2] = a->C;
  return semx::colsum(ws + l.part, p.m.T > 0 ? p.m.pieces : 0, a->C * (a->N + 2), ws + l.groups, seg, st);
}

}  // extern "C"
