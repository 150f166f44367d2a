// Backward of the selective state scan, for sm_100a.
//
// With dv = dy silu(z) (dy without z), from the last step of a sequence to its first:
//   g = C dv + carry;  carry = exp(d A) g  (the gradient of the state in front of the step)
//   u = carry h_prev;  gB = sum_n g B;  uA = sum_n u A
//   dB += g d x, dC += dv h (summed over the channels of the group), dA += u d,
//   dx = d gB + D dv, dd = uA + x gB, ddt = dd softplus'(dt + bias), dz = dy v silu'(z),
//   dD += dv x, ddt_bias += ddt
//
// Bound: instructions (24 per (step, channel, mode) of a warp, a quarter of them the exchanges
// between lanes) and shared memory's path to the registers, at 59 % and 61 % of their rates in
// 4 x 2047 x 2048 bf16 (312 us of 425 with its first pass and the join; profiles/selective_state_scan.md).
// The forward left the state in front of every kBlock steps; a block's states and poles are
// rebuilt from it in registers, half a block at a time, and the adjoint runs back through
// them: one and a half exponentials per (step, channel, mode).
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
constexpr int kCPT = 2;  // channels per thread
constexpr float kLn2 = 0.6931471805599453f;

template <int GM>
constexpr int channels_per_cta() {
  return kThreads / GM * kCPT;
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

// fp32 rows fetch x, v, z and the block's entry states for the next tile straight into shared
// memory, every thread into slots of its own: in registers they leave room for two CTAs per SM
// only (404 x 321 x 256 fp32: in registers 704 us, three CTAs that spill 752, this way 614).
// bf16 rows take half of the registers (4 x 2047 x 2048: in registers 307 us, this way 312, both
// before v was fp32).
template <int GM, bool LOCAL, int ACC>
__host__ __device__ constexpr bool stages() {
  return !LOCAL && ACC == kFp32 && GM >= 4;
}

template <int GM, bool LOCAL, int ACC>
struct BwdShared {
  static constexpr bool STAGE = stages<GM, LOCAL, ACC>();
  static constexpr int CH = channels_per_cta<GM>(), R = LOCAL ? 1 : kBlock;
  static constexpr int TS = kThreads / (CH / 4), E = (kBlock + TS - 1) / TS;
  float4 sd[kBlock][CH / 2];  // (d, d', d x, d' x') of two channels
  float2 sv[kBlock][CH / 2];  // (dv, dv')
  float4 sC[kBlock][GM];
  float4 sB[R][LOCAL ? 1 : GM];
  float so[R][LOCAL ? 4 : 2 * CH];                       // (gB, uA) per channel
  float4 sw[LOCAL ? 1 : kWarps][R][LOCAL ? 1 : 2 * GM];  // dB | dC of a warp
  float4 spar[2][CH / 4];             // dt_bias and D of the CTA's channels
  // Values that a thread leaves for itself: its sums for dD and ddt_bias, softplus' of its
  // rows, its states in front of the block.
  float4 sums[2][kThreads];
  float4 sg[LOCAL ? 1 : E][LOCAL ? 1 : kThreads];
  float4 sh[STAGE ? 2 : 1][LOCAL ? 1 : kCPT][LOCAL ? 1 : kThreads];
  uint4 rows[STAGE ? 2 : 1][STAGE ? 3 : 1][STAGE ? kThreads : 1];  // x, v, z of this tile and the next
};

// CTAs per SM that the registers are cut for (4 x 2047 x 2048 bf16: two 358 us, three 305).
template <int GM, bool LOCAL, int ACC>
__host__ __device__ constexpr int bwd_ctas() {
  return LOCAL ? 4 : ACC != kAny && GM >= 4 ? 3 : 2;
}

template <int GM, bool LOCAL, int ACC>
__global__ void __launch_bounds__(kThreads, (bwd_ctas<GM, LOCAL, ACC>())) state_scan_bwd_kernel(const ScanParams p) {
  constexpr int CL = 32 / GM, CH = channels_per_cta<GM>(), NP = 4 * GM;
  constexpr int TS = kThreads / (CH / 4);       // rows that the CTA loads at a time
  constexpr int E = (kBlock + TS - 1) / TS;     // (step, four channels) of a thread
  constexpr int ML = kThreads / GM;             // rows of B and C loaded at a time
  constexpr int EB = (kBlock + ML - 1) / ML;    // (step, four modes) of a thread
  constexpr int NV1 = 2 * kCPT, NO1 = NV1 / GM > 0 ? NV1 / GM : 1;
  constexpr int NO2 = 8 / CL > 0 ? 8 / CL : 1;
  constexpr int HALF = kBlock / 2;
  typedef typename RawQuad<ACC>::type Quad;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  typedef BwdShared<GM, LOCAL, ACC> Shared;
  constexpr bool STAGE = Shared::STAGE;
  static_assert(!STAGE || E == 1, "one row of a tile per thread");
  Shared& sm = *reinterpret_cast<Shared*>(raw_smem);
  auto& sd = sm.sd;
  auto& sv = sm.sv;
  auto& sC = sm.sC;
  auto& sB = sm.sB;
  auto& so = sm.so;
  auto& sw = sm.sw;
  auto& spar = sm.spar;
  auto& sums = sm.sums;
  auto& sg = sm.sg;
  auto& sh = sm.sh;

  const int64_t j = blockIdx.x / p.ctiles;
  const int ct = blockIdx.x % p.ctiles;
  const int grp = ct / p.tpg, cg0 = (ct % p.tpg) * CH, c_base = grp * p.cpg;
  const Piece q = find_piece(p.m, j);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
  // A sequence of one piece needs neither a first pass nor joining.
  const bool split = p.entry != nullptr && q.live && q.len > p.m.Q;
  if (LOCAL && !split) return;

  // The four channels of this thread in loads and stores (en of them exist).
  const int eq = tid % (CH / 4), ec = eq * 4, et = tid / (CH / 4);
  const int en = min(4, p.cpg - cg0 - ec);
  const int64_t ech = c_base + (en > 0 ? cg0 + ec : 0);
  const bool has_z = p.z != nullptr;
  const float4 zero4 = make_float4(0.f, 0.f, 0.f, 0.f);
  if (!LOCAL && en > 0 && et == 0)
    for_unused_rows(p.m, j, [&](int64_t r) {
      store_quad<ACC>(p.dx, r * p.C + ech, p.bf16, en, zero4);
      store_quad<ACC>(p.ddt, r * p.C + ech, p.dt_bf16, en, zero4);
      if (has_z) store_quad<ACC>(p.dz, r * p.C + ech, p.bf16, en, zero4);
    });

  // The channels and modes of this thread in the scan.
  const int lm = lane % GM, cl = lane / GM, n0 = lm * 4;
  const int cp = warp * CL + cl, sc = cp * kCPT;
  int nn[kCPT];  // modes of the channel that this thread holds
  const int64_t at0 = (int64_t)(c_base + cg0 + sc) * p.N + n0;  // (channel, first mode) of an array (C, N)
  f2 A2[kCPT][2], dA[kCPT][2], carry[kCPT][2];
#pragma unroll
  for (int i = 0; i < kCPT; ++i) {
    nn[i] = cg0 + sc + i < p.cpg ? min(4, p.N - n0) : 0;
    const float4 a = load_params(p.A, at0 + i * p.N, nn[i]);
    A2[i][0] = pack2(log2_rate(a.x), log2_rate(a.y));
    A2[i][1] = pack2(log2_rate(a.z), log2_rate(a.w));
    float4 s = zero4;
    if (!LOCAL && split) s = load_params(p.entry, j * p.C * p.N + at0 + i * p.N, nn[i]);
    carry[i][0] = pack2(s.x, s.y);
    carry[i][1] = pack2(s.z, s.w);
    dA[i][0] = dA[i][1] = 0ull;
  }
  if (et == 0) {
    spar[0][eq] = load_params(p.dt_bias, ech, en);
    spar[1][eq] = load_params(p.D, ech, en);
  }
  sums[0][tid] = sums[1][tid] = zero4;  // LOCAL: the second is the sum of the steps
  __syncthreads();
  const bool mode_quads = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.ckpt) & 15) == 0;
  const bool bc_quads = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.pBC) & 15) == 0;
  auto poles = [&](float d, f2 A) {
    const float2 a = unpack2(A);
    return pack2(pole(d, a.x), pole(d, a.y));
  };
  auto drive = [&](float dx, f2 B) {
    const float2 b = unpack2(B);
    return pack2(dx * b.x, dx * b.y);
  };

  const int tl = q.t1 > q.t0 ? q.t0 + (q.t1 - 1 - q.t0) / kBlock * kBlock : q.t0 - kBlock;
  const int tb0 = tid / GM, bl = tid % GM, bn = min(4, p.N - bl * 4);
  const float* ck = LOCAL || !q.live ? nullptr : p.ckpt + (piece_base(p.m, q.s, kBlock) + tl / kBlock) * p.C * p.N + at0;
  Quad rx[E], rd[E], rg[E], rz[E], rB[EB], rC[EB];
  uint4 rv[E];  // fp32 whatever the rows' type
  float4 hn[kCPT];
  int par = 0;  // STAGE: which of the two buffers the next fetch fills
  auto fetch = [&](int t0, int rows) {  // rows of the tile that exist
    if constexpr (STAGE) {
      const bool in = en > 0 && et < rows;
      const int64_t r = q.row0 + t0 + et;
      copy_quad<kFp32>(&sm.rows[par][0][tid], p.x, r * p.ldx + ech, in);
      if (has_z) {
        copy_quad<kFp32>(&sm.rows[par][1][tid], p.v, r * p.C + ech, in);
        copy_quad<kFp32>(&sm.rows[par][2][tid], p.z, r * p.ldz + ech, in);
      }
#pragma unroll
      for (int i = 0; i < kCPT; ++i)
        copy_quad<kFp32>(reinterpret_cast<uint4*>(&sh[par][i][tid]), nn[i] > 0 ? ck : p.ckpt, i * p.N, nn[i] > 0);
      par ^= 1;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      rx[i] = rd[i] = rg[i] = rz[i] = Quad{};
      rv[i] = uint4{};
      if (en > 0 && et + i * TS < rows) {
        const int64_t r = q.row0 + t0 + et + i * TS;
        rd[i] = load_quad<ACC>(p.dt, r * p.lddt + ech, p.dt_bf16, en);
        rg[i] = load_quad<ACC>(p.dy, r * p.C + ech, p.bf16, en);
        if (has_z && !STAGE) rz[i] = load_quad<ACC>(p.z, r * p.ldz + ech, p.bf16, en);
        if (!LOCAL && !STAGE) {
          rx[i] = load_quad<ACC>(p.x, r * p.ldx + ech, p.bf16, en);
          if (has_z) rv[i] = load_quad<fp32_beside(ACC)>(p.v, r * p.C + ech, 0, en);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < EB; ++i) {
      rB[i] = rC[i] = Quad{};
      if (bn > 0 && tb0 + i * ML < rows) {
        const int64_t r = q.row0 + t0 + tb0 + i * ML, b = (int64_t)grp * p.N + bl * 4;
        if (!LOCAL) rB[i] = load_quad<ACC>(p.B, r * p.ldb + b, p.bf16, bn);
        rC[i] = load_quad<ACC>(p.Cm, r * p.ldc + b, p.bf16, bn);
      }
    }
    if (!LOCAL && !STAGE) {
#pragma unroll
      for (int i = 0; i < kCPT; ++i) {
        hn[i] = zero4;
        if (mode_quads) {
          if (nn[i] > 0) hn[i] = *reinterpret_cast<const float4*>(ck + i * p.N);
        } else {
          hn[i] = load_params(ck, i * p.N, nn[i]);
        }
      }
    }
    if (!LOCAL) ck -= (int64_t)p.C * p.N;
  };

  if (tl >= q.t0) fetch(tl, min(kBlock, q.t1 - tl));
#pragma unroll 1
  for (int t0 = tl; t0 >= q.t0; t0 -= kBlock) {
    const int nt = min(kBlock, q.t1 - t0);
    Quad kx[E];  // x
    const int now = STAGE ? par ^ 1 : 0;  // the buffer of this tile
    if constexpr (STAGE) copies_done();
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int t = et + i * TS;
      if (t < kBlock) {
        const bool in = t < nt && en > 0;
        const float4 bias = spar[0][eq];
        float4 d = quad_floats<ACC>(rd[i], p.dt_bf16), g = quad_floats<ACC>(rg[i], p.bf16);
        d.x += bias.x; d.y += bias.y; d.z += bias.z; d.w += bias.w;
        float4 slope = make_float4(1.f, 1.f, 1.f, 1.f);
        if (p.softplus) {
          float4 e;
          const float4 raw = d;
          d = make_float4(softplus(raw.x, &e.x), softplus(raw.y, &e.y), softplus(raw.z, &e.z), softplus(raw.w, &e.w));
          if (!LOCAL)
            slope = make_float4(softplus_slope(raw.x, e.x), softplus_slope(raw.y, e.y), softplus_slope(raw.z, e.z),
                                softplus_slope(raw.w, e.w));
        }
        if (has_z) {
          float4 z;
          if constexpr (STAGE) z = quad_floats<kFp32>(sm.rows[now][2][tid], 0);
          else z = quad_floats<ACC>(rz[i], p.bf16);
          const float4 s = make_float4(sigmoid(z.x), sigmoid(z.y), sigmoid(z.z), sigmoid(z.w));
          if (!LOCAL && in) {
            float4 v;
            if constexpr (STAGE) v = quad_floats<kFp32>(sm.rows[now][1][tid], 0);
            else v = quad_floats<fp32_beside(ACC)>(rv[i], 0);
            store_quad<ACC>(p.dz, (q.row0 + t0 + t) * p.C + ech, p.bf16, en,
                            make_float4(g.x * v.x * (s.x * fmaf(z.x, 1.f - s.x, 1.f)),
                                        g.y * v.y * (s.y * fmaf(z.y, 1.f - s.y, 1.f)),
                                        g.z * v.z * (s.z * fmaf(z.z, 1.f - s.z, 1.f)),
                                        g.w * v.w * (s.w * fmaf(z.w, 1.f - s.w, 1.f))));
          }
          g.x *= z.x * s.x; g.y *= z.y * s.y; g.z *= z.z * s.z; g.w *= z.w * s.w;
        }
        if (!in) d = g = zero4;  // a row behind the piece: pole 1, no drive, no gradient
        float4 x;
        if constexpr (STAGE) x = quad_floats<kFp32>(sm.rows[now][0][tid], 0);
        else x = LOCAL ? zero4 : quad_floats<ACC>(rx[i], p.bf16);
        sd[t][2 * eq] = make_float4(d.x, d.y, d.x * x.x, d.y * x.y);
        sd[t][2 * eq + 1] = make_float4(d.z, d.w, d.z * x.z, d.w * x.w);
        *reinterpret_cast<float4*>(&sv[t][2 * eq]) = g;
        if (!LOCAL) {
          if (!STAGE) kx[i] = rx[i];
          sg[i][tid] = slope;
        } else {
          float4 s = sums[1][tid];
          s.x += d.x; s.y += d.y; s.z += d.z; s.w += d.w;
          sums[1][tid] = s;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < EB; ++i) {
      if (tb0 + i * ML < kBlock) {
        if (!LOCAL) sB[tb0 + i * ML][bl] = quad_floats<ACC>(rB[i], p.bf16);
        sC[tb0 + i * ML][bl] = quad_floats<ACC>(rC[i], p.bf16);
      }
    }
    if (!LOCAL && !STAGE) {
#pragma unroll
      for (int i = 0; i < kCPT; ++i) sh[0][i][tid] = hn[i];
    }
    __syncthreads();
    if (t0 - kBlock >= q.t0) fetch(t0 - kBlock, kBlock);

    // The later half of the block first: its entry state is a run over the earlier half,
    // whose poles and states are rebuilt afterwards. A whole block's values would take every
    // register of two CTAs per SM (4 x 2047 x 2048 bf16: 365 us against 346).
#pragma unroll 1
    for (int tb = HALF; tb >= 0; tb -= HALF) {
      f2 a[HALF][kCPT][2], h[HALF + 1][kCPT][2];
      if (!LOCAL) {
#pragma unroll
        for (int i = 0; i < kCPT; ++i) {
          const ulonglong2 e = *reinterpret_cast<const ulonglong2*>(&sh[now][i][tid]);
          h[0][i][0] = e.x;
          h[0][i][1] = e.y;
        }
        if (tb > 0) {
#pragma unroll
          for (int t = 0; t < HALF; ++t) {
            const float4 d = sd[t][cp];
            const ulonglong2 B = *reinterpret_cast<const ulonglong2*>(&sB[t][lm]);
#pragma unroll
            for (int i = 0; i < kCPT; ++i) {
              const float dd = i == 0 ? d.x : d.y, dx = i == 0 ? d.z : d.w;
              h[0][i][0] = fma2(poles(dd, A2[i][0]), h[0][i][0], drive(dx, B.x));
              h[0][i][1] = fma2(poles(dd, A2[i][1]), h[0][i][1], drive(dx, B.y));
            }
          }
        }
      }
#pragma unroll
      for (int t = 0; t < HALF; ++t) {
        const float4 d = sd[tb + t][cp];
#pragma unroll
        for (int i = 0; i < kCPT; ++i) {
          const float dd = i == 0 ? d.x : d.y;
          a[t][i][0] = poles(dd, A2[i][0]);
          a[t][i][1] = poles(dd, A2[i][1]);
        }
        if (!LOCAL) {
          const ulonglong2 B = *reinterpret_cast<const ulonglong2*>(&sB[tb + t][lm]);
#pragma unroll
          for (int i = 0; i < kCPT; ++i) {
            const float dx = i == 0 ? d.z : d.w;
            h[t + 1][i][0] = fma2(a[t][i][0], h[t][i][0], drive(dx, B.x));
            h[t + 1][i][1] = fma2(a[t][i][1], h[t][i][1], drive(dx, B.y));
          }
        }
      }
#pragma unroll
      for (int t = HALF - 1; t >= 0; --t) {
        // The compiler would load all steps' operands ahead and spill.
        asm volatile("" ::: "memory");
        const ulonglong2 C = *reinterpret_cast<const ulonglong2*>(&sC[tb + t][lm]);
        const float2 vv = sv[tb + t][cp];
        if (LOCAL) {
#pragma unroll
          for (int i = 0; i < kCPT; ++i) {
            const f2 v = i == 0 ? pack2(vv.x, vv.x) : pack2(vv.y, vv.y);
            carry[i][0] = mul2(a[t][i][0], fma2(C.x, v, carry[i][0]));
            carry[i][1] = mul2(a[t][i][1], fma2(C.y, v, carry[i][1]));
          }
        } else {
          const float4 d4 = sd[tb + t][cp];
          const ulonglong2 B = *reinterpret_cast<const ulonglong2*>(&sB[tb + t][lm]);
          float v1[NV1], v2[8];
          f2 b0 = 0ull, b1 = 0ull, c0 = 0ull, c1 = 0ull;
#pragma unroll
          for (int i = 0; i < kCPT; ++i) {
            const f2 v = i == 0 ? pack2(vv.x, vv.x) : pack2(vv.y, vv.y);
            const f2 d = i == 0 ? pack2(d4.x, d4.x) : pack2(d4.y, d4.y);
            const f2 dx = i == 0 ? pack2(d4.z, d4.z) : pack2(d4.w, d4.w);
            const f2 g0 = fma2(C.x, v, carry[i][0]), g1 = fma2(C.y, v, carry[i][1]);
            carry[i][0] = mul2(a[t][i][0], g0);
            carry[i][1] = mul2(a[t][i][1], g1);
            const f2 u0 = mul2(carry[i][0], h[t][i][0]), u1 = mul2(carry[i][1], h[t][i][1]);
            const float2 gB = unpack2(fma2(g1, B.y, mul2(g0, B.x)));
            const float2 uA = unpack2(fma2(u1, A2[i][1], mul2(u0, A2[i][0])));
            v1[2 * i] = gB.x + gB.y;
            v1[2 * i + 1] = uA.x + uA.y;
            dA[i][0] = fma2(u0, d, dA[i][0]);
            dA[i][1] = fma2(u1, d, dA[i][1]);
            b0 = i == 0 ? mul2(g0, dx) : fma2(g0, dx, b0);
            b1 = i == 0 ? mul2(g1, dx) : fma2(g1, dx, b1);
            c0 = i == 0 ? mul2(h[t + 1][i][0], v) : fma2(h[t + 1][i][0], v, c0);
            c1 = i == 0 ? mul2(h[t + 1][i][1], v) : fma2(h[t + 1][i][1], v, c1);
          }
          const float2 e0 = unpack2(b0), e1 = unpack2(b1), e2 = unpack2(c0), e3 = unpack2(c1);
          v2[0] = e0.x; v2[1] = e0.y; v2[2] = e1.x; v2[3] = e1.y;
          v2[4] = e2.x; v2[5] = e2.y; v2[6] = e3.x; v2[7] = e3.y;
          halve_sum<NV1, GM, 1>(v1, lane);
          halve_sum<8, CL, GM>(v2, lane);
          // Value k of (channel, {gB, uA}) is float 2 sc + k of the step's row.
          constexpr int SPARE1 = GM > NV1 ? GM / NV1 : 1;
          if (lm % SPARE1 == 0) {
#pragma unroll
            for (int k = 0; k < NO1; ++k) so[tb + t][2 * sc + lm / SPARE1 * NO1 + k] = v1[k];
          }
          constexpr int SPARE2 = CL > 8 ? CL / 8 : 1;
          if (cl % SPARE2 == 0) {
            float* w = reinterpret_cast<float*>(sw[warp][tb + t]);
#pragma unroll
            for (int k = 0; k < NO2; ++k) {
              const int id = cl / SPARE2 * NO2 + k;  // (dB, dC) x 4 modes
              w[(id / 4) * NP + n0 + id % 4] = v2[k];
            }
          }
        }
      }
    }
    __syncthreads();
    if (!LOCAL) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int t = et + i * TS;
        if (t < nt && en > 0) {
          const int64_t o = (q.row0 + t0 + t) * p.C + ech;
          const float4 s0 = *reinterpret_cast<const float4*>(&so[t][2 * ec]);
          const float4 s1 = *reinterpret_cast<const float4*>(&so[t][2 * ec + 4]);
          // d and dv as this thread put them there.
          float4 x;
          if constexpr (STAGE) x = quad_floats<kFp32>(sm.rows[now][0][tid], 0);
          else x = quad_floats<ACC>(kx[i], p.bf16);
          const float4 k = sg[i][tid], D = spar[1][eq];
          const float4 g = *reinterpret_cast<const float4*>(&sv[t][2 * eq]);
          const float2 d01 = *reinterpret_cast<const float2*>(&sd[t][2 * eq]);
          const float2 d23 = *reinterpret_cast<const float2*>(&sd[t][2 * eq + 1]);
          store_quad<ACC>(p.dx, o, p.bf16, en,
                          make_float4(fmaf(d01.x, s0.x, D.x * g.x), fmaf(d01.y, s0.z, D.y * g.y),
                                      fmaf(d23.x, s1.x, D.z * g.z), fmaf(d23.y, s1.z, D.w * g.w)));
          const float4 ddt = make_float4(fmaf(s0.y, kLn2, x.x * s0.x) * k.x, fmaf(s0.w, kLn2, x.y * s0.z) * k.y,
                                         fmaf(s1.y, kLn2, x.z * s1.x) * k.z, fmaf(s1.w, kLn2, x.w * s1.z) * k.w);
          store_quad<ACC>(p.ddt, o, p.dt_bf16, en, ddt);
          float4 sD = sums[0][tid], sb = sums[1][tid];
          sD.x = fmaf(g.x, x.x, sD.x); sD.y = fmaf(g.y, x.y, sD.y);
          sD.z = fmaf(g.z, x.z, sD.z); sD.w = fmaf(g.w, x.w, sD.w);
          sb.x += ddt.x; sb.y += ddt.y; sb.z += ddt.z; sb.w += ddt.w;
          sums[0][tid] = sD;
          sums[1][tid] = sb;
        }
      }
      // dB | dC of the CTA's channels: the warps' sums in order.
      for (int e = tid; e < nt * 2 * GM; e += kThreads) {
        const int t = e / (2 * GM), v = e % (2 * GM), n = v % GM * 4;
        float4 s = sw[0][t][v];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
          const float4 o = sw[w][t][v];
          s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w;
        }
        const int64_t o = ((int64_t)ct * p.m.T + q.row0 + t0 + t) * 2 * p.N + (v / GM) * p.N + n;
        if (bc_quads) {
          if (n < p.N) *reinterpret_cast<float4*>(p.pBC + o) = s;
        } else {
          store_quad<kAny>(p.pBC, o, 0, min(4, p.N - n), s);
        }
      }
    }
  }
  float* out = LOCAL ? p.entry + j * p.C * p.N : p.part != nullptr ? p.part + j * ((int64_t)p.C * (p.N + 2)) : nullptr;
  if (out == nullptr) return;
  // Without LOCAL every piece index writes its row, zeros where there is no such piece.
#pragma unroll
  for (int i = 0; i < kCPT; ++i) {
    const float2 v0 = unpack2(LOCAL ? carry[i][0] : dA[i][0]), v1 = unpack2(LOCAL ? carry[i][1] : dA[i][1]);
    store_quad<kAny>(out, at0 + i * p.N, 0, nn[i], make_float4(v0.x, v0.y, v1.x, v1.y));
  }
  // The threads of four channels in order of their rows.
  __syncthreads();
  if (et == 0) {
#pragma unroll
    for (int k = LOCAL ? 1 : 0; k < 2; ++k) {
      float4 s = sums[k][tid];
      for (int i = 1; i < TS; ++i) {
        const float4 d = sums[k][i * (CH / 4) + tid];
        s.x += d.x; s.y += d.y; s.z += d.z; s.w += d.w;
      }
      if (LOCAL) store_quad<kAny>(p.dsum, j * p.C + ech, 0, en, s);
      else store_quad<kAny>(out, (int64_t)p.C * (p.N + k) + ech, 0, en, s);
    }
  }
}

// Joins the carries of the pieces of the sequences that have more than one, from the last
// piece: entry[j] becomes the gradient of the state behind piece j. Threads as in the forward.
__global__ void __launch_bounds__(kThreads) state_scan_join_back_kernel(const ScanParams p) {
  const int64_t per = (int64_t)p.C * p.N;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (!any_split(p.m)) return;
  if (i >= per) return;
  const int64_t c = i / p.N;
  const float A2 = log2_rate(p.A[i]);
  for (int64_t s = blockIdx.y; s < p.m.S; s += gridDim.y) {
    const int64_t row0 = seq_start(p.m, s);
    const int64_t len = p.m.cu == nullptr ? p.m.L : max(seq_start(p.m, s + 1), row0) - row0;
    if (len <= p.m.Q) continue;
    const int64_t base = piece_base(p.m, s, p.m.Q), n = (len + p.m.Q - 1) / p.m.Q;
    float carry = 0.f;
    constexpr int U = 8;  // loads ahead of the chain: entry is written where it was read
    for (int64_t k = n - 1; k >= 0; k -= U) {
      float local[U], decay[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t j = base + k - u;
        local[u] = k - u >= 0 ? p.entry[j * per + i] : 0.f;
        decay[u] = k - u >= 0 ? p.dsum[j * p.C + c] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (k - u >= 0) {
          p.entry[(base + k - u) * per + i] = carry;
          carry = fmaf(semx::ex2_approx(decay[u] * A2), carry, local[u]);
        }
      }
    }
  }
}

// dB and dC: the channel tiles' sums in tile order. A thread takes four neighbouring modes of
// one (row, group, kind); a CTA a run of rows, so that a thread's place in the row is found once.
constexpr int kBcRows = 32;
template <int ACC>
__global__ void __launch_bounds__(256) state_scan_bc_kernel(const ScanParams p, void* dB, void* dC) {
  const int nq = (p.N + 3) / 4, per = 2 * p.G * nq;  // fours of a row: (kind, group, modes)
  const int64_t r0 = (int64_t)blockIdx.x * kBcRows;
  const int rows = (int)min((int64_t)kBcRows, p.m.T - r0);
  const int64_t begin = rows_begin(p.m), end = rows_end(p.m);
  const int64_t tile = p.m.T * 2 * p.N;
  for (int e = threadIdx.x; e < rows * per; e += blockDim.x) {
    const int t = e / per, f = e % per, kind = f / (p.G * nq), g = f / nq % p.G, n = f % nq * 4;
    const int64_t r = r0 + t;
    const int cnt = min(4, p.N - n);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r >= begin && r < end) {
      const float* src = p.pBC + (int64_t)g * p.tpg * tile + r * 2 * p.N + kind * p.N + n;
#pragma unroll 4
      for (int i = 0; i < p.tpg; ++i, src += tile) {
        float4 v;
        if (ACC != kAny) v = *reinterpret_cast<const float4*>(src);
        else v = load_params(src, 0, cnt);
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
      }
    }
    store_quad<ACC>(kind == 0 ? dB : dC, r * p.G * p.N + (int64_t)g * p.N + n, p.bf16, cnt, s);
  }
}

// At least two lanes per channel: with one, a thread would hold four rows of every operand of a tile
// beside a CTA's 60 KB of shared memory. So up to 4 modes leave half of the lanes without any.
int mode_lanes(int N) { return lanes_for(N, 4) < 2 ? 2 : lanes_for(N, 4); }
int tile_channels(int N) { return kThreads / mode_lanes(N) * kCPT; }

void set_tiles(ScanParams& p) {
  p.tpg = (int)semx::cdiv(p.cpg, (int64_t)tile_channels(p.N));
  p.ctiles = p.G * p.tpg;
}

// Rows per piece (0: whole sequences): as in the forward, with three resident CTAs per SM and
// about five waves (4 x 2047 x 2048: whole 590 us, one wave 475 us, five 408 us). One sequence
// of 100 rows and 256 channels, training pass: whole 56.5 us, in pieces 45.9; of 512 rows:
// whole 177 us, pieces of at least 64 rows 63.3, of 32 rows 52.1. The forward's exception holds here too, at
// 64 rows a sequence (training pass of 63 sequences of 4 rows and one of 4000: 602 us; that one alone 102).
constexpr int64_t kResident = 148 * 3;
int64_t bwd_rows_per_piece(const ScanParams& p) {
  const int64_t ctas = (int64_t)p.m.S * p.ctiles;
  const int64_t rows = p.m.S > 0 ? semx::cdiv(p.m.T, p.m.S) : 0;
  if (2 * ctas > kResident) return p.m.cu != nullptr && p.m.S > 1 ? outlier_rows(rows) : 0;
  if (rows <= 64) return 0;
  const int64_t Q = semx::cdiv(semx::cdiv(rows, 5 * kResident / ctas), kBlock) * kBlock;
  return Q < 32 ? 32 : Q;
}

struct Layout {
  size_t entry, dsum, pbc, part, total;
};
Layout layout(const ScanParams& p, int64_t Q) {
  Layout l = {};
  const size_t pieces = (size_t)p.m.pieces;
  size_t at = 0;
  // Every part starts on 16 bytes of the workspace.
  auto up = [](size_t n) { return (n + 3) / 4 * 4; };
  l.entry = at;
  at += Q > 0 ? up(pieces * p.C * p.N) : 0;
  l.dsum = at;
  at += Q > 0 ? up(pieces * p.C) : 0;
  l.pbc = at;
  at += up((size_t)p.ctiles * p.m.T * 2 * p.N);
  l.part = at;
  at += up(pieces * p.C * (p.N + 2));
  l.total = at;
  return l;
}

template <int GM, bool LOCAL, int ACC>
int launch_one(const ScanParams& p, unsigned grid, cudaStream_t st) {
  constexpr size_t bytes = sizeof(BwdShared<GM, LOCAL, ACC>);
  if (!semx::allow_smem(state_scan_bwd_kernel<GM, LOCAL, ACC>, bytes)) return SEMX_ERR_LAUNCH;
  state_scan_bwd_kernel<GM, LOCAL, ACC><<<grid, kThreads, bytes, st>>>(p);
  return semx::check_launch("state_scan_bwd_kernel");
}

template <bool LOCAL>
int launch_bwd(const ScanParams& p, cudaStream_t st) {
  const int64_t grid = p.m.pieces * p.ctiles;
  if (grid == 0) return SEMX_OK;
  if (grid >= ((int64_t)1 << 31)) return semx::fail(SEMX_ERR_SHAPE, "state_scan bwd: too many pieces");
  switch (mode_lanes(p.N)) {
#define SEMX_GM(V)                                                                        \
  case V:                                                                                 \
    if (p.access == kBf16) return launch_one<V, LOCAL, kBf16>(p, (unsigned)grid, st);     \
    if (p.access == kFp32) return launch_one<V, LOCAL, kFp32>(p, (unsigned)grid, st);     \
    return launch_one<V, LOCAL, kAny>(p, (unsigned)grid, st);
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
  if (!semx::aligned(a->ckpt, 16)) p.access = kAny;  // the states are read four at a time, too
  const bool params = a->dA != nullptr || a->dD != nullptr || a->ddt_bias != nullptr;
  p.part = params ? ws + l.part : nullptr;
  if (p.m.T > 0) {
    if (Q > 0 && p.m.S > 0) {
      p.entry = ws + l.entry;
      p.dsum = ws + l.dsum;
      rc = launch_bwd<true>(p, st);
      if (rc != SEMX_OK) return rc;
      state_scan_join_back_kernel<<<join_grid(p), kThreads, 0, st>>>(p);
      rc = semx::check_launch("state_scan_join_back_kernel");
      if (rc != SEMX_OK) return rc;
    }
    rc = launch_bwd<false>(p, st);
    if (rc != SEMX_OK) return rc;
    const unsigned grid = (unsigned)semx::cdiv(p.m.T, (int64_t)kBcRows);
    const uintptr_t align = a->bf16 ? 8 : 16;
    const bool fours = p.N % 4 == 0 && semx::aligned(p.pBC, 16) && semx::aligned(a->dB, align) && semx::aligned(a->dC, align);
    if (!fours) state_scan_bc_kernel<kAny><<<grid, 256, 0, st>>>(p, a->dB, a->dC);
    else if (a->bf16) state_scan_bc_kernel<kBf16><<<grid, 256, 0, st>>>(p, a->dB, a->dC);
    else state_scan_bc_kernel<kFp32><<<grid, 256, 0, st>>>(p, a->dB, a->dC);
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
  return semx::colsum_once(ws + l.part, p.m.T > 0 ? p.m.pieces : 0, a->C * (a->N + 2), seg, st);
}

}  // extern "C"
