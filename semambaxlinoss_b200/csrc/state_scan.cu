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
// Split: a thread owns one channel and MPT modes of it, GL neighbouring lanes a channel; a
// CTA of 128 threads owns 128 / GL channels of one piece of a sequence and walks over it in
// tiles of kTT steps. The tile's operands are loaded into registers while the tile before is
// computed, converted and put into shared memory; the sums over modes go back through
// shared memory, so that the D skip, the gate and the stores run one (step, channel) per
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

constexpr int kTT = 16;  // steps per tile

template <int MPT, int GL, bool LOCAL>
__global__ void __launch_bounds__(kThreads) state_scan_fwd_kernel(const ScanParams p) {
  constexpr int NP = MPT * GL, CH = kThreads / GL, TT = kTT;
  constexpr int E = TT * CH / kThreads > 0 ? TT * CH / kThreads : 1;  // (step, channel) pairs per thread
  constexpr int EB = (TT * NP + kThreads - 1) / kThreads;             // (step, mode) pairs per thread
  constexpr int RS = GL < 4 ? GL : 4;  // lanes whose sums are exchanged step by step
  __shared__ float2 sdt[TT][CH];       // (d, d x)
  __shared__ float sys[LOCAL ? 1 : TT][LOCAL ? 1 : CH];
  __shared__ __align__(16) float sB[TT][NP];
  __shared__ __align__(16) float sC[LOCAL ? 1 : TT][LOCAL ? 1 : NP];

  const int64_t j = blockIdx.x / p.ctiles;
  const int ct = blockIdx.x % p.ctiles;
  const int grp = ct / p.tpg;                     // group of channels that share B and C
  const int cg0 = (ct % p.tpg) * CH;              // first channel of the tile in the group
  const int c_base = grp * p.cpg;
  const Piece q = find_piece(p.m, j);
  const int64_t slot = LOCAL || !q.live ? semx::kNone : find_slot(p.m, q.s);
  const int tid = threadIdx.x;

  // The pair of this thread in loads and stores: steps tid / CH + i kThreads / CH of channel ec.
  const int ec = tid % CH, et = tid / CH;
  const bool eok = cg0 + ec < p.cpg;
  const int ech = c_base + min(cg0 + ec, p.cpg - 1);
  if (!LOCAL && eok && et == 0)
    for (int64_t r = rows_end(p.m) + j; r < p.m.T; r += p.m.pieces) {
      store(p.y, r * p.C + ech, p.bf16, 0.f);
      if (p.v != nullptr) store(p.v, r * p.C + ech, p.bf16, 0.f);
    }
  if (!q.live) return;

  // The channel and modes of this thread in the scan.
  const int lane_m = tid % GL, sc = tid / GL;
  const bool cok = cg0 + sc < p.cpg;
  const int ch = c_base + min(cg0 + sc, p.cpg - 1);
  const int n0 = lane_m * MPT;
  float A2[MPT], h[MPT];
  const bool cold = slot < 0 || (p.m.fresh != nullptr && p.m.fresh[q.s] != 0);
#pragma unroll
  for (int n = 0; n < MPT; ++n) {
    const bool ok = n0 + n < p.N;
    A2[n] = ok ? p.A[(int64_t)ch * p.N + n0 + n] * kLog2e : 0.f;
    h[n] = 0.f;
    if (!LOCAL && ok) {
      if (p.entry != nullptr) h[n] = p.entry[(j * p.C + ch) * p.N + n0 + n];
      else if (!cold) h[n] = p.state[(slot * p.C + ch) * p.N + n0 + n];
    }
  }
  const float bias = p.dt_bias != nullptr ? p.dt_bias[ech] : 0.f;
  const float Dc = LOCAL ? 0.f : (slot == semx::kRefused ? __int_as_float(0x7fffffff) : (p.D != nullptr ? p.D[ech] : 0.f));
  float dsum = 0.f;

  uint32_t rx[E], rd[E], rz[E], rB[EB], rC[EB];
  auto fetch = [&](int t0) {
    const int64_t row = q.row0 + t0 + et;
    fetch_pairs<E, kThreads / CH>(rx, p.x, p.bf16, row * p.ldx + ech, (kThreads / CH) * p.ldx, t0 + et, q.t1, eok && et < TT);
    fetch_pairs<E, kThreads / CH>(rd, p.dt, p.dt_bf16, row * p.lddt + ech, (kThreads / CH) * p.lddt, t0 + et, q.t1, eok && et < TT);
    if (!LOCAL && p.z != nullptr)
      fetch_pairs<E, kThreads / CH>(rz, p.z, p.bf16, row * p.ldz + ech, (kThreads / CH) * p.ldz, t0 + et, q.t1, eok && et < TT);
#pragma unroll
    for (int i = 0; i < EB; ++i) {
      const int e = tid + i * kThreads, t = e / NP, n = e % NP;
      const bool ok = t < TT && n < p.N && t0 + t < q.t1;
      const int64_t r = q.row0 + t0 + t;
      rB[i] = ok ? load_raw(p.B, r * p.ldb + (int64_t)grp * p.N + n, p.bf16) : 0u;
      if (!LOCAL) rC[i] = ok ? load_raw(p.Cm, r * p.ldc + (int64_t)grp * p.N + n, p.bf16) : 0u;
    }
  };
  fetch(q.t0);
  for (int t0 = q.t0; t0 < q.t1; t0 += TT) {
    float xv[E], zv[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int t = et + i * (kThreads / CH);
      if (t < TT) {
        const float x = as_float(rx[i], p.bf16);
        float d = as_float(rd[i], p.dt_bf16) + bias;
        if (p.softplus) d = softplus(d);
        if (!(t0 + t < q.t1 && eok)) d = 0.f;  // a row behind the piece: pole 1, no drive
        sdt[t][ec] = make_float2(d, d * x);
        xv[i] = x;
        zv[i] = !LOCAL && p.z != nullptr ? as_float(rz[i], p.bf16) : 0.f;
        if (LOCAL) dsum += d;
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

#pragma unroll
    for (int tb = 0; tb < TT; tb += RS) {
      float acc[RS];
#pragma unroll
      for (int u = 0; u < RS; ++u) {
        const int t = tb + u;
        if (!LOCAL && p.ckpt != nullptr && t % kBlock == 0 && t0 + t < q.t1 && cok) {
          float* o = p.ckpt + ((piece_base(p.m, q.s, kBlock) + (t0 + t) / kBlock) * p.C + ch) * p.N + n0;
#pragma unroll
          for (int n = 0; n < MPT; ++n)
            if (n0 + n < p.N) o[n] = h[n];
        }
        const float2 d = sdt[t][sc];
        acc[u] = 0.f;
#pragma unroll
        for (int n = 0; n < MPT; ++n) {
          const float a = semx::ex2_approx(d.x * A2[n]);
          h[n] = fmaf(a, h[n], d.y * sB[t][n0 + n]);
          if (!LOCAL) acc[u] = fmaf(h[n], sC[t][n0 + n], acc[u]);
        }
      }
      if (!LOCAL) {
        // Lane m (mod RS) of a channel's lanes ends with the sum of step tb + m.
        const float s = lanes_scatter_sum<GL>(acc, lane_m);
        if (lane_m < RS) sys[tb + lane_m][sc] = s;
      }
    }
    __syncthreads();
    if (!LOCAL) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int t = et + i * (kThreads / CH);
        if (t < TT && t0 + t < q.t1 && eok) {
          const int64_t o = (q.row0 + t0 + t) * p.C + ech;
          float v = fmaf(Dc, xv[i], sys[t][ec]);
          if (p.v != nullptr) store(p.v, o, p.bf16, v);
          if (p.z != nullptr) v *= zv[i] * sigmoid(zv[i]);
          store(p.y, o, p.bf16, v);
        }
      }
    }
  }
  if (LOCAL) {
    if (cok)
#pragma unroll
      for (int n = 0; n < MPT; ++n)
        if (n0 + n < p.N) p.entry[(j * p.C + ch) * p.N + n0 + n] = h[n];
    // Sum of the steps: the threads of a channel in order.
    float* red = reinterpret_cast<float*>(&sdt[0][0]);
    red[tid] = dsum;
    __syncthreads();
    if (tid < CH && eok) {
      float s = 0.f;
      for (int i = 0; i < kThreads / CH; ++i) s += red[i * CH + tid];
      p.dsum[j * p.C + ech] = s;
    }
  } else if (p.entry == nullptr && slot >= 0 && cok) {
#pragma unroll
    for (int n = 0; n < MPT; ++n)
      if (n0 + n < p.N) p.state[(slot * p.C + ch) * p.N + n0 + n] = h[n];
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
int launch_fwd(ScanParams& p, int mpt, cudaStream_t st) {
  const int gl = lanes_for(p.N, mpt);
  const int64_t ch = kThreads / gl;
  p.tpg = (int)semx::cdiv(p.cpg, ch);
  p.ctiles = p.G * p.tpg;
  const int64_t grid = p.m.pieces * p.ctiles;
  if (grid == 0) return SEMX_OK;
  if (grid >= ((int64_t)1 << 31)) return semx::fail(SEMX_ERR_SHAPE, "state_scan: too many pieces");
#define SEMX_GL(M, GV)                                                                            \
  if (mpt == M && gl == GV) {                                                                     \
    state_scan_fwd_kernel<M, GV, LOCAL><<<(unsigned)grid, kThreads, 0, st>>>(p);                  \
    return semx::check_launch("state_scan_fwd_kernel");                                           \
  }
  SEMX_GL(16, 1)
  SEMX_GL(4, 1)
  SEMX_GL(4, 2)
  SEMX_GL(4, 4)
  SEMX_GL(4, 8)
  SEMX_GL(4, 16)
  SEMX_GL(4, 32)
#undef SEMX_GL
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
  return SEMX_OK;
}

}  // namespace semx_scan

namespace {

// How a forward is run: modes per thread, and rows per piece (0: whole sequences).
struct Plan {
  int mpt;
  int64_t Q;
};
Plan fwd_plan(const ScanParams& p) {
  const int64_t work = (int64_t)p.m.S * p.C;
  Plan plan = {4, 0};
  if (p.N <= 16 && p.N > 4 && work >= 148 * 256) plan.mpt = 16;
  const int64_t warps = work * lanes_for(p.N, plan.mpt) / 32;
  const int64_t rows = p.m.S > 0 ? p.m.T / p.m.S : 0;
  if (warps < 148 * 8 && rows > 64) {
    const int64_t cut = semx::cdiv((int64_t)148 * 16, warps > 0 ? warps : 1);
    int64_t Q = semx::cdiv(semx::cdiv(p.m.T, p.m.S * cut), 16) * 16;
    plan.Q = Q < 32 ? 32 : Q;
  }
  return plan;
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
  const Plan plan = fwd_plan(p);
  semx::set_pieces(&p.m, plan.Q);
  if (p.m.S == 0 && p.m.T > 0) p.m.pieces = 1;  // nothing but rows behind the last sequence
  if (plan.Q > 0 && p.m.S > 0) {
    SEMX_REQUIRE(a->workspace != nullptr, SEMX_ERR_WORKSPACE, "state_scan: workspace is NULL");
    p.entry = reinterpret_cast<float*>(a->workspace);
    p.dsum = p.entry + (size_t)p.m.pieces * p.C * p.N;
    rc = launch_fwd<true>(p, plan.mpt, st);
    if (rc != SEMX_OK) return rc;
    const int64_t grid = p.m.S * semx::cdiv((int64_t)p.C * p.N, kThreads);
    if (grid >= ((int64_t)1 << 31)) return semx::fail(SEMX_ERR_SHAPE, "state_scan: too many sequences");
    state_scan_join_kernel<<<(unsigned)grid, kThreads, 0, st>>>(p);
    rc = semx::check_launch("state_scan_join_kernel");
    if (rc != SEMX_OK) return rc;
  }
  return launch_fwd<false>(p, plan.mpt, st);
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
  const Plan plan = fwd_plan(p);
  semx::set_pieces(&p.m, plan.Q);
  return plan.Q > 0 ? split_floats(p) * sizeof(float) : 0;
}

}  // extern "C"
