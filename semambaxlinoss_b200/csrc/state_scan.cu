// Selective state scan over whole sequences, forward, for sm_100a.
//
//   d = softplus(dt + dt_bias);  h[n] = exp(d A[n]) h[n] + d x B[n]
//   v = sum_n C[n] h[n] + D x;   y = v silu(z)
//
// Bound: the special-function unit. A step of a channel takes N exponentials (16 lanes per
// clock per SM) and 4 N multiply-adds, against 8 to 16 bytes moved. So every exponential is
// evaluated once where the batch fills the GPU, and everything else is kept off the units
// that evaluate them: A is scaled by log2(e) once, d and d x are evaluated once per (step,
// channel) and shared through shared memory.
//
// Split: a thread owns one channel and 4 modes of it (two pairs, each in one register pair
// for the two-wide multiply-adds), GL neighbouring lanes a channel; a CTA of 128 threads
// owns 128 / GL channels of one piece of a sequence and walks over it in tiles of steps. The tile's operands are loaded into registers while the tile before is
// computed, converted and put into shared memory; the sums over modes go back through
// shared memory, so that the step, the D skip, the gate and the stores run two channels per
// thread with neighbouring channels in neighbouring threads.
//
// Long sequences that leave the GPU idle are cut into pieces. A first pass (LOCAL) runs each
// piece from zero and keeps its last state and the sum of its steps d; since all of a
// piece's poles multiply to exp(A sum d), joining the pieces costs one multiply-add per
// piece and mode; then every piece is run from its true entry state. That evaluates the
// exponentials twice.
#include <cuda_bf16.h>

#include "state_scan.cuh"

namespace {

using namespace semx_scan;

// Steps per tile: at most 1024 (step, channel) pairs and 2048 (step, mode) pairs.
template <int GL>
constexpr int tile_steps() {
  return GL <= 4 ? 8 * GL : GL == 8 ? 32 : 16;
}

template <int GL, bool LOCAL>
__global__ void __launch_bounds__(kThreads, GL >= 4 ? 4 : 2) state_scan_fwd_kernel(const ScanParams p) {
  constexpr int NP = 4 * GL, CH = kThreads / GL, TT = tile_steps<GL>();
  constexpr int TS = kThreads / (CH / 2);                  // rows that the CTA loads at a time
  constexpr int E = (TT + TS - 1) / TS;                    // (step, channel pair)s of a thread
  constexpr int EB = (TT * NP + kThreads - 1) / kThreads;  // (step, mode)s of a thread
  constexpr int RS = GL < 4 ? GL : 4;                      // steps whose sums are exchanged together
  constexpr int YS = CH + 8;                               // row of sys: the RS rows fall into other banks
  __shared__ __align__(16) float4 sdt[TT][CH];             // (d, d, d x, d x)
  __shared__ __align__(16) float sys[LOCAL ? 1 : TT][LOCAL ? 2 : YS];
  __shared__ __align__(16) float sB[TT][NP];
  __shared__ __align__(16) float sC[LOCAL ? 1 : TT][LOCAL ? 1 : NP];

  const int64_t j = blockIdx.x / p.ctiles;
  const int ct = blockIdx.x % p.ctiles;
  const int grp = ct / p.tpg;         // group of channels that share B and C
  const int cg0 = (ct % p.tpg) * CH;  // first channel of the tile in the group
  const int c_base = grp * p.cpg;
  const Piece q = find_piece(p.m, j);
  const int64_t slot = LOCAL || !q.live ? semx::kNone : find_slot(p.m, q.s);
  const int tid = threadIdx.x;

  // The channel pair of this thread in loads and stores; its steps are et, et + TS, ...
  const int ec = tid % (CH / 2) * 2, et = tid / (CH / 2);
  const bool eok = cg0 + ec < p.cpg, two = cg0 + ec + 1 < p.cpg;
  const bool vec = p.vec2 != 0;
  const int ech = c_base + min(cg0 + ec, p.cpg - 1), ech1 = two ? ech + 1 : ech;
  if (!LOCAL && eok && et == 0)
    for (int64_t r = rows_end(p.m) + j; r < p.m.T; r += p.m.pieces) {
      store_pair(p.y, r * p.C + ech, p.bf16, vec, two, 0.f, 0.f);
      if (p.v != nullptr) store_pair(p.v, r * p.C + ech, p.bf16, vec, two, 0.f, 0.f);
    }
  if (!q.live) return;

  // The channel and modes of this thread in the scan.
  const int lm = tid % GL, sc = tid / GL;
  const bool cok = cg0 + sc < p.cpg;
  const int ch = c_base + min(cg0 + sc, p.cpg - 1);
  const int n0 = lm * 4;
  const bool cold = slot < 0 || (p.m.fresh != nullptr && p.m.fresh[q.s] != 0);
  f2 A2[2], h[2];
  {
    float a[4], s[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const bool ok = n0 + n < p.N;
      a[n] = ok ? p.A[(int64_t)ch * p.N + n0 + n] * kLog2e : 0.f;
      s[n] = 0.f;
      if (!LOCAL && ok) {
        if (p.entry != nullptr) s[n] = p.entry[(j * p.C + ch) * p.N + n0 + n];
        else if (!cold) s[n] = p.state[(slot * p.C + ch) * p.N + n0 + n];
      }
    }
    A2[0] = pack2(a[0], a[1]); A2[1] = pack2(a[2], a[3]);
    h[0] = pack2(s[0], s[1]); h[1] = pack2(s[2], s[3]);
  }
  const f2 pole_bias = pack2(kPoleBias, kPoleBias);
  const float bias0 = p.dt_bias != nullptr ? p.dt_bias[ech] : 0.f, bias1 = p.dt_bias != nullptr ? p.dt_bias[ech1] : 0.f;
  float D0 = 0.f, D1 = 0.f;
  if (!LOCAL) {
    if (p.D != nullptr) { D0 = p.D[ech]; D1 = p.D[ech1]; }
    if (slot == semx::kRefused) D0 = D1 = __int_as_float(0x7fffffff);
  }
  float dsum0 = 0.f, dsum1 = 0.f;
  // States that a training forward keeps: of step 0 of the piece on, every kBlock steps.
  float* ck = nullptr;
  if (!LOCAL && p.ckpt != nullptr && cok)
    ck = p.ckpt + ((piece_base(p.m, q.s, kBlock) + q.t0 / kBlock) * p.C + ch) * p.N + n0;
  const int64_t ck_step = (int64_t)p.C * p.N;
  const bool ck_vec = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.ckpt) & 15) == 0;

  uint2 rx[E], rd[E], rz[E];
  uint32_t rB[EB], rC[EB];
  auto fetch = [&](int t0) {
    const int64_t row = q.row0 + t0 + et;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const bool ok = eok && et + i * TS < TT && t0 + et + i * TS < q.t1;
      const int64_t r = row + i * TS;
      rx[i] = rd[i] = rz[i] = make_uint2(0u, 0u);
      if (ok) {
        rx[i] = load_pair(p.x, r * p.ldx + ech, p.bf16, vec, two);
        rd[i] = load_pair(p.dt, r * p.lddt + ech, p.dt_bf16, vec, two);
        if (!LOCAL && p.z != nullptr) rz[i] = load_pair(p.z, r * p.ldz + ech, p.bf16, vec, two);
      }
    }
#pragma unroll
    for (int i = 0; i < EB; ++i) {
      const int e = tid + i * kThreads, t = e / NP, n = e % NP;
      const bool ok = t < TT && n < p.N && t0 + t < q.t1;
      const int64_t r = q.row0 + t0 + t;
      rB[i] = ok ? load_raw(p.B, r * p.ldb + (int64_t)grp * p.N + n, p.bf16) : 0u;
      if (!LOCAL) rC[i] = ok ? load_raw(p.Cm, r * p.ldc + (int64_t)grp * p.N + n, p.bf16) : 0u;
    }
  };
  if (q.t0 < q.t1) fetch(q.t0);
  for (int t0 = q.t0; t0 < q.t1; t0 += TT) {
    float2 xv[E], zv[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int t = et + i * TS;
      if (t < TT) {
        const float2 x = pair_floats(rx[i], p.bf16);
        float2 d = pair_floats(rd[i], p.dt_bf16);
        d.x += bias0;
        d.y += bias1;
        if (p.softplus) {
          d.x = softplus(d.x);
          d.y = softplus(d.y);
        }
        if (t0 + t >= q.t1) d.x = d.y = 0.f;  // a row behind the piece: pole 1, no drive
        sdt[t][ec] = make_float4(d.x, d.x, d.x * x.x, d.x * x.x);
        sdt[t][ec + 1] = make_float4(d.y, d.y, d.y * x.y, d.y * x.y);
        xv[i] = x;
        if (!LOCAL && p.z != nullptr) zv[i] = pair_floats(rz[i], p.bf16);
        if (LOCAL) {
          dsum0 += d.x;
          dsum1 += d.y;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < EB; ++i) {
      const int e = tid + i * kThreads;
      if (e < TT * NP) {
        (&sB[0][0])[e] = as_float(rB[i], p.bf16);
        if (!LOCAL) (&sC[0][0])[e] = as_float(rC[i], p.bf16);
      }
    }
    __syncthreads();
    if (t0 + TT < q.t1) fetch(t0 + TT);

    const int nt = min(TT, q.t1 - t0);
#pragma unroll 1
    for (int tb = 0; tb < nt; tb += 4) {
      if (!LOCAL && ck != nullptr && (tb & (kBlock - 1)) == 0) {
        const float2 a = unpack2(h[0]), b = unpack2(h[1]);
        if (ck_vec) {
          if (n0 < p.N) *reinterpret_cast<float4*>(ck) = make_float4(a.x, a.y, b.x, b.y);
        } else {
          if (n0 < p.N) ck[0] = a.x;
          if (n0 + 1 < p.N) ck[1] = a.y;
          if (n0 + 2 < p.N) ck[2] = b.x;
          if (n0 + 3 < p.N) ck[3] = b.y;
        }
        ck += ck_step;
      }
      float acc[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int t = tb + u;
        const ulonglong2 d = *reinterpret_cast<const ulonglong2*>(&sdt[t][sc]);
        const ulonglong2 Bn = *reinterpret_cast<const ulonglong2*>(&sB[t][n0]);
        h[0] = fma2(poles2(d.x, A2[0], pole_bias), h[0], mul2(d.y, Bn.x));
        h[1] = fma2(poles2(d.x, A2[1], pole_bias), h[1], mul2(d.y, Bn.y));
        if (!LOCAL) {
          const ulonglong2 Cn = *reinterpret_cast<const ulonglong2*>(&sC[t][n0]);
          const float2 v = unpack2(fma2(h[1], Cn.y, mul2(h[0], Cn.x)));
          acc[u] = v.x + v.y;
        }
      }
      if (!LOCAL) {
        // Lane m (mod RS) of a channel's lanes ends with the sums of steps m, m + RS, ...
#pragma unroll
        for (int u = 0; u < 4; u += RS) {
          float part[RS];
#pragma unroll
          for (int k = 0; k < RS; ++k) part[k] = acc[u + k];
          const float s = lanes_scatter_sum<GL, RS>(part, lm);
          if (lm < RS) sys[tb + u + lm][sc] = s;
        }
      }
    }
    __syncthreads();
    if (!LOCAL) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int t = et + i * TS;
        if (t < TT && t0 + t < q.t1 && eok) {
          const int64_t o = (q.row0 + t0 + t) * p.C + ech;
          const float2 s = *reinterpret_cast<const float2*>(&sys[t][ec]);
          float v0 = fmaf(D0, xv[i].x, s.x), v1 = fmaf(D1, xv[i].y, s.y);
          if (p.v != nullptr) store_pair(p.v, o, p.bf16, vec, two, v0, v1);
          if (p.z != nullptr) {
            v0 *= zv[i].x * sigmoid(zv[i].x);
            v1 *= zv[i].y * sigmoid(zv[i].y);
          }
          store_pair(p.y, o, p.bf16, vec, two, v0, v1);
        }
      }
    }
  }
  const float2 ha = unpack2(h[0]), hb = unpack2(h[1]);
  const float last[4] = {ha.x, ha.y, hb.x, hb.y};
  if (LOCAL) {
    if (cok)
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (n0 + n < p.N) p.entry[(j * p.C + ch) * p.N + n0 + n] = last[n];
    // Sum of the steps: the threads of a channel in order.
    float* red = reinterpret_cast<float*>(&sdt[0][0]);
    __syncthreads();
    red[et * CH + ec] = dsum0;
    red[et * CH + ec + 1] = dsum1;
    __syncthreads();
    if (tid < CH && cg0 + tid < p.cpg) {
      float s = 0.f;
      for (int i = 0; i < TS; ++i) s += red[i * CH + tid];
      p.dsum[j * p.C + c_base + cg0 + tid] = s;
    }
  } else if (p.entry == nullptr && slot >= 0 && cok) {
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (n0 + n < p.N) p.state[(slot * p.C + ch) * p.N + n0 + n] = last[n];
  }
}

// Joins the pieces of a sequence: entry[j] becomes the state in front of piece j, the last
// state goes to the pool. One thread per (sequence, channel, mode).
__global__ void __launch_bounds__(kThreads) state_scan_join_kernel(const ScanParams p) {
  const int64_t per = (int64_t)p.C * p.N;
  const int64_t tiles = (per + kThreads - 1) / kThreads;
  const int64_t s = blockIdx.x / tiles;
  const int64_t i = (blockIdx.x % tiles) * kThreads + threadIdx.x;
  const int64_t slot = find_slot(p.m, s);
  if (i >= per) return;
  const int64_t c = i / p.N;
  const float A2 = p.A[i] * kLog2e;
  const int64_t row0 = seq_start(p.m, s);
  const int64_t len = p.m.cu == nullptr ? p.m.L : max(seq_start(p.m, s + 1), row0) - row0;
  const int64_t base = piece_base(p.m, s, p.m.Q), n = (len + p.m.Q - 1) / p.m.Q;
  const bool cold = slot < 0 || (p.m.fresh != nullptr && p.m.fresh[s] != 0);
  float h = cold ? 0.f : p.state[slot * per + i];
  for (int64_t k = 0; k < n; ++k) {
    const int64_t j = base + k;
    const float local = p.entry[j * per + i];
    p.entry[j * per + i] = h;
    h = fmaf(semx::ex2_approx(p.dsum[j * p.C + c] * A2), h, local);
  }
  if (slot >= 0) p.state[slot * per + i] = h;
}

template <bool LOCAL>
int launch_fwd(ScanParams& p, cudaStream_t st) {
  const int gl = lanes_for(p.N, 4);
  p.tpg = (int)semx::cdiv(p.cpg, (int64_t)(kThreads / gl));
  p.ctiles = p.G * p.tpg;
  const int64_t grid = p.m.pieces * p.ctiles;
  if (grid == 0) return SEMX_OK;
  if (grid >= ((int64_t)1 << 31)) return semx::fail(SEMX_ERR_SHAPE, "state_scan: too many pieces");
  switch (gl) {
#define SEMX_GL(GV)                                                                     \
  case GV:                                                                              \
    state_scan_fwd_kernel<GV, LOCAL><<<(unsigned)grid, kThreads, 0, st>>>(p);           \
    return semx::check_launch("state_scan_fwd_kernel");
    SEMX_GL(1)
    SEMX_GL(2)
    SEMX_GL(4)
    SEMX_GL(8)
    SEMX_GL(16)
    SEMX_GL(32)
#undef SEMX_GL
  }
  return semx::fail(SEMX_ERR_UNSUPPORTED, "state_scan: %d modes", p.N);
}

}  // namespace

namespace semx_scan {

int scan_validate(const SemxStateScanArgs* a, bool bwd, ScanParams* p) {
  SEMX_REQUIRE(a->N >= 1 && a->N <= kMaxN, SEMX_ERR_UNSUPPORTED, "state_scan: N=%lld (1..%d)", (long long)a->N, kMaxN);
  SEMX_REQUIRE(a->C >= 1 && a->C < (1 << 24), SEMX_ERR_SHAPE, "state_scan: C=%lld", (long long)a->C);
  SEMX_REQUIRE(a->G >= 1 && a->C % a->G == 0, SEMX_ERR_SHAPE, "state_scan: %lld channels in %lld groups",
               (long long)a->C, (long long)a->G);
  const int64_t top = (int64_t)1 << 31;
  SEMX_REQUIRE(a->ldx >= a->C && a->lddt >= a->C && (a->z == nullptr || a->ldz >= a->C) && a->ldb >= a->G * a->N &&
                   a->ldc >= a->G * a->N && a->ldx < top && a->lddt < top && a->ldz < top && a->ldb < top && a->ldc < top,
               SEMX_ERR_SHAPE, "state_scan: row strides %lld %lld %lld %lld %lld", (long long)a->ldx,
               (long long)a->lddt, (long long)a->ldz, (long long)a->ldb, (long long)a->ldc);
  int rc = semx::check_seqs("state_scan", a->S, a->rows, a->L, a->cu_seqlens, a->state, a->slots, a->fresh,
                            a->n_slots, &p->m);
  if (rc != SEMX_OK) return rc;
  SEMX_REQUIRE(!bwd || a->state == nullptr, SEMX_ERR_UNSUPPORTED, "state_scan bwd: no state");
  const bool none = a->rows == 0;
  SEMX_REQUIRE(a->A && (none || (a->x && a->dt && a->B && a->Cm)), SEMX_ERR_NULL, "state_scan: x / dt / A / B / C is NULL");
  if (!bwd) {
    SEMX_REQUIRE(none || a->y, SEMX_ERR_NULL, "state_scan: y is NULL");
  } else {
    SEMX_REQUIRE(none || (a->dy && a->dx && a->ddt && a->dB && a->dC && a->ckpt), SEMX_ERR_NULL,
                 "state_scan bwd: dy / dx / ddt / dB / dC / ckpt is NULL");
    SEMX_REQUIRE(none || a->z == nullptr || (a->dz && a->v), SEMX_ERR_NULL, "state_scan bwd: dz / v is NULL");
  }
  p->C = (int)a->C; p->N = (int)a->N; p->G = (int)a->G; p->cpg = (int)(a->C / a->G);
  p->bf16 = a->bf16; p->dt_bf16 = a->dt_bf16; p->softplus = a->softplus;
  p->ldx = a->ldx; p->lddt = a->lddt; p->ldz = a->ldz; p->ldb = a->ldb; p->ldc = a->ldc;
  p->x = a->x; p->dt = a->dt; p->A = a->A; p->B = a->B; p->Cm = a->Cm; p->D = a->D; p->z = a->z;
  p->dt_bias = a->dt_bias; p->y = a->y; p->state = a->state; p->v = a->v; p->ckpt = a->ckpt;
  p->dy = a->dy; p->dx = a->dx; p->ddt = a->ddt; p->dz = a->dz;
  const uintptr_t align = a->bf16 ? 4 : 8;
  p->vec2 = p->cpg % 2 == 0 && a->ldx % 2 == 0 && a->lddt % 2 == 0 && (a->z == nullptr || a->ldz % 2 == 0) &&
            semx::aligned(a->dt, a->dt_bf16 ? 4 : 8) && semx::aligned(a->ddt, a->dt_bf16 ? 4 : 8);
  for (const void* t : {a->x, a->z, (const void*)a->y, (const void*)a->v, a->dy, (const void*)a->dx, (const void*)a->dz})
    if (!semx::aligned(t, align)) p->vec2 = 0;
  return SEMX_OK;
}

}  // namespace semx_scan

namespace {

// Rows per piece of a forward (0: whole sequences).
int64_t fwd_rows_per_piece(const ScanParams& p) {
  const int64_t warps = (int64_t)p.m.S * p.C * lanes_for(p.N, 4) / 32;
  const int64_t rows = p.m.S > 0 ? p.m.T / p.m.S : 0;
  if (warps >= 148 * 8 || rows <= 64) return 0;
  const int64_t cut = semx::cdiv((int64_t)148 * 16, warps > 0 ? warps : 1);
  const int64_t Q = semx::cdiv(semx::cdiv(p.m.T, p.m.S * cut), 32) * 32;
  return Q < 32 ? 32 : Q;
}

size_t split_floats(const ScanParams& p) { return (size_t)p.m.pieces * p.C * (p.N + 1); }

}  // namespace

extern "C" {

size_t semx_state_scan_args_size(void) { return sizeof(SemxStateScanArgs); }

size_t semx_state_scan_ckpt_bytes(const SemxStateScanArgs* a) {
  if (a == nullptr || a->S < 0 || a->rows < 0 || a->C < 1 || a->N < 1) return 0;
  const int64_t blocks = a->cu_seqlens == nullptr ? a->S * semx::cdiv(a->L, kBlock) : a->rows / kBlock + a->S;
  return (size_t)blocks * a->C * a->N * sizeof(float);
}

int semx_state_scan_fwd(const SemxStateScanArgs* a, semx_stream_t stream) {
  SEMX_CHECK_ARGS(a, SemxStateScanArgs);
  ScanParams p = {};
  int rc = scan_validate(a, false, &p);
  if (rc != SEMX_OK) return rc;
  semx::DeviceScope scope;
  rc = scope.bind({a->y, a->state});
  if (rc != SEMX_OK) return rc;
  cudaStream_t st = semx::as_stream(stream);
  const int64_t Q = fwd_rows_per_piece(p);
  semx::set_pieces(&p.m, Q);
  if (p.m.S == 0 && p.m.T > 0) p.m.pieces = 1;  // nothing but rows behind the last sequence
  if (Q > 0 && p.m.S > 0) {
    SEMX_REQUIRE(a->workspace != nullptr, SEMX_ERR_WORKSPACE, "state_scan: workspace is NULL");
    p.entry = reinterpret_cast<float*>(a->workspace);
    p.dsum = p.entry + (size_t)p.m.pieces * p.C * p.N;
    rc = launch_fwd<true>(p, st);
    if (rc != SEMX_OK) return rc;
    const int64_t grid = p.m.S * semx::cdiv((int64_t)p.C * p.N, kThreads);
    if (grid >= ((int64_t)1 << 31)) return semx::fail(SEMX_ERR_SHAPE, "state_scan: too many sequences");
    state_scan_join_kernel<<<(unsigned)grid, kThreads, 0, st>>>(p);
    rc = semx::check_launch("state_scan_join_kernel");
    if (rc != SEMX_OK) return rc;
  }
  return launch_fwd<false>(p, st);
}

size_t semx_state_scan_workspace_bytes(const SemxStateScanArgs* a, int32_t backward) {
  if (a == nullptr) return 0;
  SemxStateScanArgs b = *a;
  float* any = reinterpret_cast<float*>(256);
  b.x = b.dt = b.B = b.Cm = any;
  b.A = any;
  b.y = any;
  b.dy = any;
  b.dx = b.ddt = b.dz = b.dB = b.dC = b.v = any;
  b.ckpt = any;
  ScanParams p = {};
  if (scan_validate(&b, backward != 0, &p) != SEMX_OK) return 0;
  if (backward != 0) return scan_bwd_workspace(p);
  const int64_t Q = fwd_rows_per_piece(p);
  semx::set_pieces(&p.m, Q);
  return Q > 0 ? split_floats(p) * sizeof(float) : 0;
}

}  // extern "C"
