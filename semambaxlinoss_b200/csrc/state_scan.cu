// Selective state scan over whole sequences, forward, for sm_100a.
//
//   d = softplus(dt + dt_bias);  h[n] = exp(d A[n]) h[n] + d x B[n]
//   v = sum_n C[n] h[n] + D x;   y = v silu(z)
//
// Bound: the special-function unit. A step of a channel takes N exponentials (16 lanes per
// clock per SM) and 4 N multiply-adds, against 8 to 16 bytes moved. So every exponential is
// evaluated once where the batch fills the GPU, and everything else is kept off the units
// that evaluate them: A is scaled by log2(e) once, d and d x are evaluated once per (step,
// channel) and shared through shared memory. Measured: 404 x 321 x 256 fp32 training forward
// 232 us (exponentials alone 114, its bytes 142); in 4 x 2047 x 2048 bf16 the unit is busy 58 %
// of the main pass and 77 % of the first one (profiles/selective_state_scan.md).
//
// Split: a thread owns two channels and 4 modes of each (two pairs, each in one register pair
// for the two-wide multiply-adds), GL neighbouring lanes a channel; a CTA of 128 threads
// owns 256 / GL channels of one piece of a sequence and walks over it in tiles of steps. The
// tile's operands are loaded while the tile before is computed, converted and put into shared
// memory; the sums over modes go back through shared memory, so that the step, the D skip,
// the gate and the stores run four neighbouring channels per thread.
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

// Channels per thread: the values of B and C that a thread reads from shared memory serve
// both of them (with one channel per thread shared memory was the bound, at 3 to 4 cycles a
// load: 153 us where two take less for a prompt of 8191 x 2048).
constexpr int kCPT = 2;

template <int GL>
constexpr int channels_per_cta() {
  return kThreads / GL * kCPT;
}
template <int GL>
constexpr int tile_steps() {
  return GL >= 4 ? 16 : 8;
}

// Rows that are read four elements at a time go straight into shared memory, every thread's
// into slots of its own, where x and z stay until the tile's results need them again (404 x
// 321 x 256 fp32: through registers 243 us, this way 232; with the registers cut for five CTAs
// per SM instead of four 250). The first pass needs them once and is faster without (4 x 2047
// x 2048 bf16: 89 us and 91).
template <int GL, bool LOCAL, int ACC>
__host__ __device__ constexpr bool stages() {
  return !LOCAL && ACC != kAny && GL >= 4;
}

template <int GL, bool LOCAL, int ACC>
__global__ void __launch_bounds__(kThreads, GL >= 4 ? 4 : 2) state_scan_fwd_kernel(const ScanParams p) {
  constexpr int CH = channels_per_cta<GL>(), TT = tile_steps<GL>();
  constexpr int TS = kThreads / (CH / 4);                  // rows that the CTA loads at a time
  constexpr int E = (TT + TS - 1) / TS;                    // (step, four channels) of a thread
  constexpr int ML = kThreads / GL;                        // rows of B and C loaded at a time
  constexpr int EB = (TT + ML - 1) / ML;                   // (step, four modes) of a thread
  constexpr int RS = GL < 4 ? GL : 4;                      // steps whose sums are exchanged together
  constexpr int YS = CH + 8;                               // row of sys: RS rows fall into other banks
  typedef typename RawQuad<ACC>::type Quad;
  __shared__ __align__(16) float4 sdt[TT][CH / 2];         // (d, d', d x, d' x') of two channels
  __shared__ __align__(16) float sys[LOCAL ? 1 : TT][LOCAL ? 4 : YS];
  __shared__ __align__(16) float4 sB[TT][GL];
  __shared__ __align__(16) float4 sC[LOCAL ? 1 : TT][LOCAL ? 1 : GL];
  constexpr bool STAGE = stages<GL, LOCAL, ACC>();
  __shared__ __align__(16) Quad rows[STAGE ? 2 : 1][STAGE ? 3 : 1][STAGE ? E : 1][STAGE ? kThreads : 1];  // x, dt, z

  const int64_t j = blockIdx.x / p.ctiles;
  const int ct = blockIdx.x % p.ctiles;
  const int grp = ct / p.tpg;         // group of channels that share B and C
  const int cg0 = (ct % p.tpg) * CH;  // first channel of the tile in the group
  const int c_base = grp * p.cpg;
  const Piece q = find_piece(p.m, j);
  const int64_t slot = LOCAL || !q.live ? semx::kNone : find_slot(p.m, q.s);
  const int tid = threadIdx.x;

  // The four channels of this thread in loads and stores (en of them exist); its steps are
  // et, et + TS, ...
  const int ec = tid % (CH / 4) * 4, et = tid / (CH / 4);
  const int en = min(4, p.cpg - cg0 - ec);
  const int64_t ech = c_base + (en > 0 ? cg0 + ec : 0);
  const bool has_z = !LOCAL && p.z != nullptr;
  if (!LOCAL && en > 0 && et == 0)
    for_unused_rows(p.m, j, [&](int64_t r) {
      store_quad<ACC>(p.y, r * p.C + ech, p.bf16, en, make_float4(0.f, 0.f, 0.f, 0.f));
      if (p.v != nullptr) store_quad<fp32_beside(ACC)>(p.v, r * p.C + ech, 0, en, make_float4(0.f, 0.f, 0.f, 0.f));
    });
  // A sequence of one piece needs neither a first pass nor joining: its piece starts from the
  // pool's entry and leaves its state there.
  const bool split = p.entry != nullptr && q.len > p.m.Q;
  if (!q.live || (LOCAL && !split)) return;

  // The channels and modes of this thread in the scan.
  const int lm = tid % GL, cp = tid / GL, sc = cp * kCPT;
  const int n0 = lm * 4;
  const bool cold = slot < 0 || (p.m.fresh != nullptr && p.m.fresh[q.s] != 0);
  int nn[kCPT];  // modes of the channel that this thread holds
  const int64_t at0 = (int64_t)(c_base + cg0 + sc) * p.N + n0;  // (channel, first mode) of an array (C, N)
  float A2[kCPT][4];
  f2 h[kCPT][2];
#pragma unroll
  for (int i = 0; i < kCPT; ++i) {
    nn[i] = cg0 + sc + i < p.cpg ? min(4, p.N - n0) : 0;
    const float4 a = load_params(p.A, at0 + i * p.N, nn[i]);
    A2[i][0] = log2_rate(a.x); A2[i][1] = log2_rate(a.y); A2[i][2] = log2_rate(a.z); A2[i][3] = log2_rate(a.w);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!LOCAL) {
      if (split) s = load_params(p.entry, j * p.C * p.N + at0 + i * p.N, nn[i]);
      else if (!cold) s = load_params(p.state, slot * p.C * p.N + at0 + i * p.N, nn[i]);
    }
    h[i][0] = pack2(s.x, s.y);
    h[i][1] = pack2(s.z, s.w);
  }
  const float4 bias = load_params(p.dt_bias, ech, en);
  float4 D = LOCAL ? make_float4(0.f, 0.f, 0.f, 0.f) : load_params(p.D, ech, en);
  if (slot == semx::kRefused) D.x = D.y = D.z = D.w = __int_as_float(0x7fffffff);
  float4 dsum = make_float4(0.f, 0.f, 0.f, 0.f);
  // States that a training forward keeps: of step 0 of the piece on, every kBlock steps.
  float* ck = nullptr;
  const int64_t ck_step = (int64_t)p.C * p.N;
  if (!LOCAL && p.ckpt != nullptr) ck = p.ckpt + (piece_base(p.m, q.s, kBlock) + q.t0 / kBlock) * ck_step;
  const bool mode_quads = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.ckpt) & 15) == 0;

  Quad rx[E], rd[E], rz[E], rB[EB], rC[EB];
  // Element offsets of the thread's first row; they move on by a tile at a time.
  int64_t ox = (q.row0 + q.t0 + et) * p.ldx + ech, od = (q.row0 + q.t0 + et) * p.lddt + ech;
  int64_t oz = (q.row0 + q.t0 + et) * p.ldz + ech, oy = (q.row0 + q.t0 + et) * p.C + ech;
  const int tb0 = tid / GL;  // its (step, four modes): steps tb0, tb0 + ML, ...
  int64_t oB = (q.row0 + q.t0 + tb0) * p.ldb + (int64_t)grp * p.N + n0;
  int64_t oC = (q.row0 + q.t0 + tb0) * p.ldc + (int64_t)grp * p.N + n0;
  const int bn = min(4, p.N - n0);
  int par = 0;  // STAGE: which of the two buffers the next fetch fills
  auto fetch = [&](int left) {  // rows of the piece from this tile on
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if constexpr (STAGE) {
        const bool in = en > 0 && et + i * TS < min(TT, left);
        copy_quad<ACC>(&rows[par][0][i][tid], p.x, ox + i * TS * p.ldx, in);
        copy_quad<ACC>(&rows[par][1][i][tid], p.dt, od + i * TS * p.lddt, in);
        if (has_z) copy_quad<ACC>(&rows[par][2][i][tid], p.z, oz + i * TS * p.ldz, in);
        continue;
      }
      rx[i] = rd[i] = rz[i] = Quad{};
      if (en > 0 && et + i * TS < min(TT, left)) {
        rx[i] = load_quad<ACC>(p.x, ox + i * TS * p.ldx, p.bf16, en);
        rd[i] = load_quad<ACC>(p.dt, od + i * TS * p.lddt, p.dt_bf16, en);
        if (has_z) rz[i] = load_quad<ACC>(p.z, oz + i * TS * p.ldz, p.bf16, en);
      }
    }
    par ^= 1;
    ox += TT * p.ldx;
    od += TT * p.lddt;
    oz += TT * p.ldz;
#pragma unroll
    for (int i = 0; i < EB; ++i) {
      rB[i] = rC[i] = Quad{};
      if (bn > 0 && tb0 + i * ML < min(TT, left)) {
        rB[i] = load_quad<ACC>(p.B, oB + i * ML * p.ldb, p.bf16, bn);
        if (!LOCAL) rC[i] = load_quad<ACC>(p.Cm, oC + i * ML * p.ldc, p.bf16, bn);
      }
    }
    oB += TT * p.ldb;
    oC += TT * p.ldc;
  };
  if (q.t0 < q.t1) fetch(q.t1 - q.t0);
  for (int t0 = q.t0; t0 < q.t1; t0 += TT) {
    const int left = q.t1 - t0, nt = min(TT, left);
    float4 xv[E], zv[E];
    const int now = STAGE ? par ^ 1 : 0;  // the buffer of this tile
    if constexpr (STAGE) copies_done();
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int t = et + i * TS;
      if (t < TT) {
        if constexpr (STAGE) {
          rx[i] = rows[now][0][i][tid];
          rd[i] = rows[now][1][i][tid];
        }
        const float4 x = quad_floats<ACC>(rx[i], p.bf16);
        float4 d = quad_floats<ACC>(rd[i], p.dt_bf16);
        d.x += bias.x; d.y += bias.y; d.z += bias.z; d.w += bias.w;
        if (p.softplus) d = softplus4(d);
        if (t >= nt) d = make_float4(0.f, 0.f, 0.f, 0.f);  // a row behind the piece: pole 1, no drive
        sdt[t][ec / 2] = make_float4(d.x, d.y, d.x * x.x, d.y * x.y);
        sdt[t][ec / 2 + 1] = make_float4(d.z, d.w, d.z * x.z, d.w * x.w);
        if constexpr (!STAGE) {
          xv[i] = x;
          if (has_z) zv[i] = quad_floats<ACC>(rz[i], p.bf16);
        }
        if (LOCAL) {
          dsum.x += d.x; dsum.y += d.y; dsum.z += d.z; dsum.w += d.w;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < EB; ++i) {
      if (tb0 + i * ML < TT) {
        sB[tb0 + i * ML][lm] = quad_floats<ACC>(rB[i], p.bf16);
        if (!LOCAL) sC[tb0 + i * ML][lm] = quad_floats<ACC>(rC[i], p.bf16);
      }
    }
    __syncthreads();
    if (left > TT) fetch(left - TT);

#pragma unroll 1
    for (int tb = 0; tb < nt; tb += 4) {
      if (!LOCAL && ck != nullptr && (tb & (kBlock - 1)) == 0) {
#pragma unroll
        for (int i = 0; i < kCPT; ++i) {
          const float2 a = unpack2(h[i][0]), b = unpack2(h[i][1]);
          if (mode_quads) {
            if (nn[i] > 0) *reinterpret_cast<float4*>(ck + at0 + i * p.N) = make_float4(a.x, a.y, b.x, b.y);
          } else {
            store_quad<kAny>(ck, at0 + i * p.N, 0, nn[i], make_float4(a.x, a.y, b.x, b.y));
          }
        }
        ck += ck_step;
      }
      float acc[kCPT][4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int t = tb + u;
        const float4 d = sdt[t][cp];
        const float4 Bn = sB[t][lm];
        ulonglong2 Cn;
        if (!LOCAL) Cn = *reinterpret_cast<const ulonglong2*>(&sC[t][lm]);
#pragma unroll
        for (int i = 0; i < kCPT; ++i) {
          const float dd = i == 0 ? d.x : d.y, dx = i == 0 ? d.z : d.w;
          h[i][0] = fma2(pack2(pole(dd, A2[i][0]), pole(dd, A2[i][1])), h[i][0], pack2(dx * Bn.x, dx * Bn.y));
          h[i][1] = fma2(pack2(pole(dd, A2[i][2]), pole(dd, A2[i][3])), h[i][1], pack2(dx * Bn.z, dx * Bn.w));
          if (!LOCAL) {
            const float2 v = unpack2(fma2(h[i][1], Cn.y, mul2(h[i][0], Cn.x)));
            acc[i][u] = v.x + v.y;
          }
        }
      }
      if (!LOCAL) {
        // Lane m (mod RS) of a channel's lanes ends with the sums of steps m, m + RS, ...
#pragma unroll
        for (int u = 0; u < 4; u += RS) {
          float s[kCPT];
#pragma unroll
          for (int i = 0; i < kCPT; ++i) {
            float part[RS];
#pragma unroll
            for (int k = 0; k < RS; ++k) part[k] = acc[i][u + k];
            s[i] = lanes_scatter_sum<GL, RS>(part, lm);
          }
          if (lm < RS) *reinterpret_cast<float2*>(&sys[tb + u + lm][sc]) = make_float2(s[0], s[1]);
        }
      }
    }
    __syncthreads();
    if (!LOCAL) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int t = et + i * TS;
        if (t < nt && en > 0) {
          const int64_t o = oy + i * TS * (int64_t)p.C;
          const float4 s = *reinterpret_cast<const float4*>(&sys[t][ec]);
          if constexpr (STAGE) {
            xv[i] = quad_floats<ACC>(rows[now][0][i][tid], p.bf16);
            if (has_z) zv[i] = quad_floats<ACC>(rows[now][2][i][tid], p.bf16);
          }
          float4 v = make_float4(fmaf(D.x, xv[i].x, s.x), fmaf(D.y, xv[i].y, s.y), fmaf(D.z, xv[i].z, s.z),
                                 fmaf(D.w, xv[i].w, s.w));
          if (p.v != nullptr) store_quad<fp32_beside(ACC)>(p.v, o, 0, en, v);
          if (has_z) v = gate4(v, zv[i]);
          store_quad<ACC>(p.y, o, p.bf16, en, v);
        }
      }
      oy += TT * (int64_t)p.C;
    }
  }
  float* out = LOCAL ? p.entry + j * p.C * p.N : !split && slot >= 0 ? p.state + slot * p.C * p.N : nullptr;
  if (out != nullptr) {
#pragma unroll
    for (int i = 0; i < kCPT; ++i) {
      const float2 a = unpack2(h[i][0]), b = unpack2(h[i][1]);
      store_quad<kAny>(out, at0 + i * p.N, 0, nn[i], make_float4(a.x, a.y, b.x, b.y));
    }
  }
  if (LOCAL) {
    // Sum of the steps: the threads of a channel in order.
    __syncthreads();
    if (et < TT) sdt[0][et * (CH / 4) + ec / 4] = dsum;  // at most TT CH / 4 entries
    __syncthreads();
    if (et == 0 && en > 0) {
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int i = 0; i < (TS < TT ? TS : TT); ++i) {
        const float4 d = sdt[0][i * (CH / 4) + ec / 4];
        s.x += d.x; s.y += d.y; s.z += d.z; s.w += d.w;
      }
      store_quad<kAny>(p.dsum, j * p.C + ech, 0, en, s);
    }
  }
}

// Joins the pieces of the sequences that have more than one: entry[j] becomes the state in
// front of piece j, the last state goes to the pool. A thread owns a (channel, mode); a CTA
// walks over every gridDim.y-th sequence.
__global__ void __launch_bounds__(kThreads) state_scan_join_kernel(const ScanParams p) {
  const int64_t per = (int64_t)p.C * p.N;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (!any_split(p.m)) return;
  const int64_t c = min(i, per - 1) / p.N;
  const float A2 = log2_rate(p.A[min(i, per - 1)]);
  for (int64_t s = blockIdx.y; s < p.m.S; s += gridDim.y) {
    const int64_t row0 = seq_start(p.m, s);
    const int64_t len = p.m.cu == nullptr ? p.m.L : max(seq_start(p.m, s + 1), row0) - row0;
    if (len <= p.m.Q) continue;
    const int64_t slot = find_slot(p.m, s);
    if (i >= per) continue;
    const int64_t base = piece_base(p.m, s, p.m.Q), n = (len + p.m.Q - 1) / p.m.Q;
    const bool cold = slot < 0 || (p.m.fresh != nullptr && p.m.fresh[s] != 0);
    float h = cold ? 0.f : p.state[slot * per + i];
    // Batches of loads ahead of the chain: entry is written where it was read.
    constexpr int U = 8;
    for (int64_t k = 0; k < n; k += U) {
      float local[U], decay[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t j = base + k + u;
        local[u] = k + u < n ? p.entry[j * per + i] : 0.f;
        decay[u] = k + u < n ? p.dsum[j * p.C + c] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (k + u < n) {
          p.entry[(base + k + u) * per + i] = h;
          h = fmaf(semx::ex2_approx(decay[u] * A2), h, local[u]);
        }
      }
    }
    if (slot >= 0) p.state[slot * per + i] = h;
  }
}

template <bool LOCAL>
int launch_fwd(ScanParams& p, cudaStream_t st) {
  const int gl = lanes_for(p.N, 4);
  p.tpg = (int)semx::cdiv(p.cpg, (int64_t)(kThreads / gl * kCPT));
  p.ctiles = p.G * p.tpg;
  const int64_t grid = p.m.pieces * p.ctiles;
  if (grid == 0) return SEMX_OK;
  if (grid >= ((int64_t)1 << 31)) return semx::fail(SEMX_ERR_SHAPE, "state_scan: too many pieces");
  switch (gl) {
#define SEMX_GL(GV)                                                                                              \
  case GV:                                                                                                       \
    if (p.access == kBf16) state_scan_fwd_kernel<GV, LOCAL, kBf16><<<(unsigned)grid, kThreads, 0, st>>>(p);      \
    else if (p.access == kFp32) state_scan_fwd_kernel<GV, LOCAL, kFp32><<<(unsigned)grid, kThreads, 0, st>>>(p); \
    else state_scan_fwd_kernel<GV, LOCAL, kAny><<<(unsigned)grid, kThreads, 0, st>>>(p);                         \
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
  SEMX_REQUIRE(semx::all_aligned({a->x, a->B, a->Cm, a->z, a->y, a->dy, a->dx, a->dz, a->dB, a->dC}, a->bf16 ? 2 : 4) &&
                   semx::all_aligned({a->dt, a->ddt}, a->dt_bf16 ? 2 : 4) &&
                   semx::all_aligned({a->A, a->D, a->dt_bias, a->cu_seqlens, a->state, a->slots, a->v, a->ckpt, a->dA, a->dD,
                                      a->ddt_bias, a->workspace}, 4),
               SEMX_ERR_ALIGN, "state_scan: a pointer is not on an element");
  p->C = (int)a->C; p->N = (int)a->N; p->G = (int)a->G; p->cpg = (int)(a->C / a->G);
  p->bf16 = a->bf16; p->dt_bf16 = a->dt_bf16; p->softplus = a->softplus;
  p->ldx = a->ldx; p->lddt = a->lddt; p->ldz = a->ldz; p->ldb = a->ldb; p->ldc = a->ldc;
  p->x = a->x; p->dt = a->dt; p->A = a->A; p->B = a->B; p->Cm = a->Cm; p->D = a->D; p->z = a->z;
  p->dt_bias = a->dt_bias; p->y = a->y; p->state = a->state; p->v = a->v; p->ckpt = a->ckpt;
  p->dy = a->dy; p->dx = a->dx; p->ddt = a->ddt; p->dz = a->dz;
  // Four neighbours per access: one type, and every row, group and base on four elements.
  p->access = kAny;
  if ((a->bf16 != 0) == (a->dt_bf16 != 0) && p->cpg % 4 == 0 && p->N % 4 == 0 && a->ldx % 4 == 0 && a->lddt % 4 == 0 &&
      (a->z == nullptr || a->ldz % 4 == 0) && a->ldb % 4 == 0 && a->ldc % 4 == 0) {
    bool ok = semx::aligned(a->v, 16);
    for (const void* t : {a->x, a->dt, a->B, a->Cm, a->z, (const void*)a->y, a->dy, (const void*)a->dx,
                          (const void*)a->ddt, (const void*)a->dz})
      ok = ok && semx::aligned(t, a->bf16 ? 8 : 16);
    if (ok) p->access = a->bf16 ? kBf16 : kFp32;
  }
  return SEMX_OK;
}

}  // namespace semx_scan

namespace {

// Rows per piece of a forward (0: whole sequences). Pieces cost the exponentials twice, so
// only batches that leave half of the GPU idle are cut (4 x 2047 x 2048: whole 275 us, in
// pieces 216 us), into two waves of the four CTAs that an SM holds: the second evens out
// what the first leaves uneven (one wave 235 us, three 212 us, but of shorter pieces). Three
// launches against one pay from about 100 rows on (one sequence of 256 channels: 100 rows
// 15.9 us whole and 15.7 in pieces, 256 rows 34.8 and 15.9), and pieces of 32 rows still do
// (512 rows: pieces of at least 64 rows 22.0 us, 32 rows 16.6). Batches that fill the GPU are
// cut at outlier_rows() if their lengths are not known to be equal. A packed batch that leaves half of
// the GPU idle and has at most 96 rows a sequence on average runs whole, however long one of them is
// (256 channels, 63 sequences of 4 rows and one of 4000: 437 us; that one alone, in pieces, 37).
constexpr int64_t kResident = 148 * 4;
int64_t fwd_rows_per_piece(const ScanParams& p) {
  const int64_t ch = kThreads / lanes_for(p.N, 4) * kCPT;
  const int64_t ctas = p.m.S * p.G * semx::cdiv(p.cpg, ch);
  const int64_t rows = p.m.S > 0 ? semx::cdiv(p.m.T, p.m.S) : 0;
  if (2 * ctas > kResident) return p.m.cu != nullptr && p.m.S > 1 ? outlier_rows(rows) : 0;
  if (rows <= 96) return 0;
  const int64_t Q = semx::cdiv(semx::cdiv(rows, 2 * kResident / ctas), 16) * 16;
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
  if (rc != SEMX_OK || semx::nothing_to_do(p.m)) return rc;
  semx::DeviceScope scope;
  rc = scope.bind({a->y, a->state});
  if (rc != SEMX_OK) return rc;
  cudaStream_t st = semx::as_stream(stream);
  const int64_t Q = fwd_rows_per_piece(p);
  semx::set_pieces(&p.m, Q);
  if (p.m.S == 0 && p.m.T > 0) p.m.pieces = 1;  // nothing but unused rows
  if (Q > 0 && p.m.S > 0) {
    SEMX_REQUIRE(a->workspace != nullptr, SEMX_ERR_WORKSPACE, "state_scan: workspace is NULL");
    p.entry = reinterpret_cast<float*>(a->workspace);
    p.dsum = p.entry + (size_t)p.m.pieces * p.C * p.N;
    rc = launch_fwd<true>(p, st);
    if (rc != SEMX_OK) return rc;
    state_scan_join_kernel<<<join_grid(p), kThreads, 0, st>>>(p);
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
  b.dx = b.ddt = b.dz = b.dB = b.dC = any;
  b.v = b.ckpt = any;
  ScanParams p = {};
  if (scan_validate(&b, backward != 0, &p) != SEMX_OK) return 0;
  if (backward != 0) return scan_bwd_workspace(p);
  const int64_t Q = fwd_rows_per_piece(p);
  semx::set_pieces(&p.m, Q);
  return Q > 0 ? split_floats(p) * sizeof(float) : 0;
}

}  // extern "C"
