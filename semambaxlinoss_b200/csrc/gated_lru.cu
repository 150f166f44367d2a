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
// Bound: HBM (5 values per element forward, 9 backward); the special-function unit (6 operations per
// element forward, 11 backward) comes next. Measured (device time): many sequences, 404 x 321 x 256 fp32 forward
// 113 us (5.9 TB/s) and backward 210 (5.7), bf16 84 and 183 (no unit is full: issue slots 58 %, special functions 56 and
// 47 %, memory 43 and 33 %, 28 and 24 % of the warps; they wait for one another at the barriers and for results); linked,
// 8191 x 2048 bf16 54 (3.1 TB/s: the links' way to L2 and back on top) and backward 123, fp32 72 and 144, 4 x 2047 x 2048
// bf16 backward 123 (2.5). These have decays above 0.883 (kNear); one below among four neighbouring channels takes
// their thread through decay2's other branch: 404 x 321 x 256 fp32 131 and 257, bf16 118 and 257, 8191 x 2048 bf16 70
// and 158, fp32 86 and 175.
//
// Split: a tile is 64 steps (backward 32) of one sequence by 32 channels; a CTA of four warps reads
// it once. A thread has a segment of 4 (2) neighbouring steps of four neighbouring channels: it folds
// them into one map h -> A h + B, one warp (a lane per channel) folds the 16 segments' maps and finds
// the tile's entry state, and each thread runs its steps again from its segment's entry state, on
// registers. CTAs stay and take tile after tile; the next tile's rows are on their way while this
// one's entry state is looked for.
// Many sequences: a CTA walks one after another, the state stays in registers. Few or packed ones:
// tiles are linked through global memory inside the one launch: each leaves its map (A, B) and the
// state behind it, and takes the maps of the tiles in front of it in its group of 16 and the state that
// the group before left. Which maps are folded in which order depends on the numbers alone, so
// results do not change from run to run. Tickets number the tiles in the order in which CTAs take
// them, one count for each 32 channels, so a tile only waits for tiles that are under way. The backward runs the
// same from the last tile on.
#include "semx_reduce.cuh"
#include "state_scan.cuh"

namespace {

using namespace semx_scan;

constexpr int kSms = 148;
constexpr int kT = 128;
constexpr int kCh = 32;             // channels of a tile: eight lanes of four
constexpr int kSegs = kT * 4 / kCh; // segments of a tile
constexpr int kFwdCtas = 5, kBwdCtas = 4;  // per SM
constexpr int kGroup = 16;          // tiles between two states handed on
constexpr float kLeastGain = 1e-3f;  // sqrt(1e-6), as the gamma gain of the selective-LRU scans has it
constexpr float kNear = 0.125f;     // -la up to which the polynomials below hold
constexpr long long kPatience = 4000000000ll;  // cycles that a wait takes at most

// Steps of a segment. The backward has more to keep per step, and its unrolled steps leave the
// instruction cache (404 x 321 x 256 bf16, two or four steps: forward 100 and 84 us, backward 186 and 229).
constexpr int kFwdSeg = 4, kBwdSeg = 2;
constexpr int kUnit = kSegs * kBwdSeg;  // steps between two states that a training forward keeps

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
  float* ckpt;  // (units, C) state in front of every 32nd step
  const void* dy;
  void* dx;
  void* dr;
  void* di;
  void* dz;
  float* part;     // (tiles, or sequences where a CTA walks them; 3, C) partial drate | dr_bias | di_bias
  int* ticket;     // linked: the number of each channel tile's next piece
  ulonglong2* maps;         // linked: (tiles, C) map (A, B) of each tile, kHere in the upper half of both
  unsigned long long* left; // linked: (tiles, C) state behind each tile, kHere in the upper half
};

// Special-function results in pairs.
__device__ __forceinline__ f2 ex2_2(f2 v) {
  const float2 t = unpack2(v);
  return pack2(semx::ex2_approx(t.x), semx::ex2_approx(t.y));
}
__device__ __forceinline__ f2 rcp_2(f2 v) {
  const float2 t = unpack2(v);
  return pack2(semx::rcp_approx(t.x), semx::rcp_approx(t.y));
}
__device__ __forceinline__ f2 rsqrt_2(f2 v) {
  const float2 t = unpack2(v);
  return pack2(semx::rsqrt_approx(t.x), semx::rsqrt_approx(t.y));
}
__device__ __forceinline__ f2 both(float c) { return pack2(c, c); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// With m = -la in [0, 0.125], polynomials of degree 3 in m (fewer coefficients matter because a pair of equal constants
// takes two instructions to make):
//   exp(-m), at most 3.7e-9 of it off, and sqrt((1 - exp(-2 m)) / (2 m)), fitted to the least largest relative error with
//   1 at m = 0: at most 3.1e-8 to either side. Their roundings come on top.
__device__ __forceinline__ f2 horner3(f2 m, float c0, float c1, float c2, float c3) {
  f2 v = fma2(both(c3), m, both(c2));
  v = fma2(v, m, both(c1));
  return fma2(v, m, both(c0));
}
__device__ __forceinline__ f2 decay_near(f2 m) {
  return fma2(horner3(m, -1.0f, 0.4999960958957672f, -0.16650986671447754f, 0.03964177519083023f), m, both(1.f));
}
__device__ __forceinline__ f2 root_near(f2 m) {
  return horner3(m, 1.0f, -0.49999523162841797f, 0.20810209214687347f, -0.05929150432348251f);
}
// What a channel's rates come to, one float per channel of the tile.
struct Rates {
  float speed[kCh], minus[kCh];  // rate_scale softplus(rate), and its negative
  float root[kCh];   // sqrt(2 speed)
  float slope[kCh];  // d speed / d rate
  float r2[kCh], i2[kCh];  // biases, times -log2(e)
};
__device__ __forceinline__ void load_rates(const GlParams& p, int c0, int lane, Rates* to) {
  const int c = min(c0 + lane, p.C - 1);
  const float rate = p.rate[c];
  float e, s = p.scale * softplus(rate, &e);
  to->slope[lane] = p.scale * softplus_slope(rate, e);
  s = s > 1e37f ? 1e37f : s;  // an infinite one times a closed gate is no number
  to->speed[lane] = s;
  to->minus[lane] = -s;
  to->root[lane] = sqrtf(2.f * s);  // (not by the reciprocal root, which takes a speed below the normal numbers for 0)
  to->r2[lane] = p.r_bias != nullptr ? -kLog2e * p.r_bias[c] : 0.f;
  to->i2[lane] = p.i_bias != nullptr ? -kLog2e * p.i_bias[c] : 0.f;
}
__device__ __forceinline__ f2 shared_pair(const float* row, int c) {
  return *reinterpret_cast<const f2*>(row + c);
}

// Channels 2 h and 2 h + 1 of four.
template <int ACC>
__device__ __forceinline__ f2 pair_of(const typename RawQuad<ACC>::type& q, int h, int bf16) {
  if constexpr (ACC == kBf16) {
    const uint32_t w = h ? q.y : q.x;
    return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    const uint32_t a = h ? q.z : q.x, b = h ? q.w : q.y;
    return ACC == kFp32 ? pack2(__uint_as_float(a), __uint_as_float(b)) : pack2(as_float(a, bf16), as_float(b, bf16));
  }
}

// Decay and gain of a pair of channels. The decay gate's reciprocal root q gives both the gate
// rho = q^2 and the gain: with m = -la = speed rho, sqrt(1 - exp(-2 m)) = sqrt(2 speed) q root(m).
// Near m = 0 the decay is exact to its rounding (a state multiplies hundreds of them) and nothing
// cancels; far from it the special-function exponential is 2 steps off, which a decay below 0.89
// forgets in tens of steps. gain: not yet at its least value. SLOW: no channel gets far.
template <bool SLOW>
__device__ __forceinline__ void decay2(f2 q, f2 speed, f2 root, f2* rho, f2* m, f2* a, f2* gain) {
  *rho = mul2(q, q);
  *m = mul2(*rho, speed);
  *a = decay_near(*m);
  *gain = mul2(mul2(q, root), root_near(*m));
  if constexpr (!SLOW) {
    const float2 mm = unpack2(*m);
    float2 aa = unpack2(*a), gg = unpack2(*gain);
    if (mm.x > kNear) {
      aa.x = semx::ex2_approx(-kLog2e * mm.x);
      gg.x = sqrtf(fmaf(-aa.x, aa.x, 1.f));
    }
    if (mm.y > kNear) {
      aa.y = semx::ex2_approx(-kLog2e * mm.y);
      gg.y = sqrtf(fmaf(-aa.y, aa.y, 1.f));
    }
    *a = pack2(aa.x, aa.y);
    *gain = pack2(gg.x, gg.y);
  }
}
// The gain, its least value at least. (A NaN stays: the gradient of x has no other trace of it.)
__device__ __forceinline__ f2 least2(f2 gain) {
  float2 g = unpack2(gain);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(g.x) : "f"(kLeastGain));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(g.y) : "f"(kLeastGain));
  return pack2(g.x, g.y);
}
// 1 - s of a sigmoid s = 1 / (1 + e): e s, which nothing cancels in, and 1 where e is infinite (a shut gate: s is 0,
// and so is what it multiplies, however large the rest is; the gradient of a gate that is no number has s in it too).
__device__ __forceinline__ f2 rest2(f2 e, f2 s) {
  const float2 t = unpack2(mul2(e, s));
  return pack2(fminf(t.x, 1.f), fminf(t.y, 1.f));
}
__device__ __forceinline__ f2 gate_arg(f2 v, f2 bias) { return fma2(v, both(-kLog2e), bias); }

// -- links between the tiles of a sequence --------------------------------------------------------

constexpr unsigned long long kHere = 1ull << 32;

// Where tile number `at` in the order of the recurrence is among the pieces: j0 + dir at.
struct Chain {
  int j0, dir, at;
};

__device__ __forceinline__ ulonglong2 peek_map(const ulonglong2* p) {
  ulonglong2 v;
  asm volatile("ld.relaxed.gpu.global.v2.u64 {%0, %1}, [%2];" : "=l"(v.x), "=l"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long peek(const unsigned long long* p) {
  unsigned long long v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
// Every number comes with the mark that it is there (64 bits are one access), so that no fence
// stands between a tile and the next.
__device__ __forceinline__ unsigned long long marked(float v) { return kHere | __float_as_uint(v); }
__device__ __forceinline__ void leave_map(const GlParams& p, int64_t j, int c, float A, float B) {
  asm volatile("st.relaxed.gpu.global.v2.u64 [%0], {%1, %2};" ::"l"(&p.maps[j * p.C + c]), "l"(marked(A)), "l"(marked(B)) : "memory");
}
__device__ __forceinline__ void leave_state(const GlParams& p, int64_t j, int c, float h) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(&p.left[j * p.C + c]), "l"(marked(h)) : "memory");
}

// State in front of the tile for channel c (a lane each; ok false: none): the maps of the tiles in
// front in its group, folded in their order, applied to the state that the group before left. Three warps fetch
// five of the maps each while the fourth waits for the state, so that a link is one way to L2 and back
// (4 x 2047 x 2048 bf16, the fourth warp alone: forward 59 us, backward 135; so: 54 and 126, with a tile's sums as
// they are added now 123). The first tile of a sequence has its entry state in its map (A = 0).
constexpr int kAhead = (kGroup - 1) / 3;  // maps of a warp
static_assert(3 * kAhead == kGroup - 1, "maps in front");
typedef float Links[3][2][kCh];
__device__ __forceinline__ float link_failed() {
  atomicAdd(&g_link_timeouts, 1u);
  return __int_as_float(0x7fffffff);
}
// Warps 1 to 3: the fold of their maps.
__device__ __forceinline__ void link_maps(const GlParams& p, const Chain& q, int c, bool ok, Links& to) {
  const int part = threadIdx.x / 32 - 1, e0 = q.at / kGroup * kGroup + part * kAhead, j = q.j0 + q.dir * e0;
  // Offsets that decrease can name pieces that are none.
  const int there = j < 0 || j >= (int)p.m.pieces ? 0 : q.dir > 0 ? (int)p.m.pieces - j : j + 1;
  const int n = ok ? min(q.at - e0, there) : 0;
  float a = 1.f, b = 0.f;
  if (n > 0) {
    const long long from = clock64();
    const ulonglong2* at = p.maps + (int64_t)j * p.C + c;
    const int64_t step = (int64_t)q.dir * p.C;
    ulonglong2 m[kAhead];
    bool done, given_up;
    do {
      done = true;
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        m[e] = make_ulonglong2(marked(1.f), marked(0.f));
        if (e < n) m[e] = peek_map(at + e * step);
      }
#pragma unroll
      for (int e = 0; e < kAhead; ++e) done = done && (m[e].x & kHere) != 0 && (m[e].y & kHere) != 0;
      given_up = !done && clock64() - from > kPatience;
    } while (!done && !given_up);
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const float A = __uint_as_float((unsigned)m[e].x), B = __uint_as_float((unsigned)m[e].y);
      b = fmaf(A, b, B);
      a *= A;
    }
    if (given_up) b = link_failed();
  }
  to[part][0][threadIdx.x & 31] = a;
  to[part][1][threadIdx.x & 31] = b;
}
// Warp 0: the state that the group before left.
__device__ __forceinline__ float link_state(const GlParams& p, const Chain& q, int c, bool ok) {
  const int g0 = q.at / kGroup * kGroup, jb = q.j0 + q.dir * (g0 - 1);
  if (!ok || g0 == 0 || jb < 0 || jb >= (int)p.m.pieces) return 0.f;
  const long long from = clock64();
  const unsigned long long* at = &p.left[(int64_t)jb * p.C + c];
  unsigned long long before;
  do {
    before = peek(at);
    if ((before & kHere) == 0 && clock64() - from > kPatience) return link_failed();
  } while ((before & kHere) == 0);
  return __uint_as_float((unsigned)before);
}
__device__ __forceinline__ float link_all(const Links& from, float h) {
#pragma unroll
  for (int k = 0; k < 3; ++k) h = fmaf(from[k][0][threadIdx.x & 31], h, from[k][1][threadIdx.x & 31]);
  return h;
}
// Warps 1 to 3 have left their folds; warp 0 waits for them.
__device__ __forceinline__ void links_left() { asm volatile("bar.arrive 1, %0;" ::"n"(kT) : "memory"); }
__device__ __forceinline__ void links_await() { asm volatile("bar.sync 1, %0;" ::"n"(kT) : "memory"); }

// -- the order of a CTA's tiles -------------------------------------------------------------------

// A tile: rows [row, row + n) of the batch, number k of `tiles` of sequence s, piece j of the batch; the
// state in front of its first step is kept as number `unit`.
struct Tile {
  int row, n, k, tiles, s, j, unit;
  bool any, live;  // any: there is one; live: it is a part of a sequence (one without rows has tile 0)
};

__device__ __forceinline__ int start_of(const semx::SeqMap& m, int s) {
  return m.cu == nullptr ? s * (int)m.L : min(max(m.cu[s], 0), (int)m.T);
}
// Piece j of Q rows, as semx::find_piece has it, in 32 bits with Q known.
template <int Q>
__device__ __forceinline__ void find_tile(const semx::SeqMap& m, int j, Tile* t) {
  int start, len;
  if (m.cu == nullptr) {
    t->s = (int)((unsigned)j / (unsigned)m.per);
    t->k = j - t->s * (int)m.per;
    start = t->s * (int)m.L;
    len = (int)m.L;
  } else {
    int lo = 0, n = (int)m.S;
    const int lane = threadIdx.x & 31;
    while (n > 1) {
      const int step = (n + 31) / 32;
      const int at = lo + lane * step;
      const bool ok = lane * step < n && start_of(m, at) / Q + at <= j;
      const unsigned hit = __ballot_sync(0xffffffffu, ok);
      const int w = hit == 0u ? 0 : 31 - __clz((int)hit);
      lo += w * step;
      n = min(step, n - w * step);
    }
    t->s = lo;
    start = start_of(m, lo);
    len = max(start_of(m, lo + 1), start) - start;
    t->k = j - (start / Q + lo);
  }
  t->tiles = (len + Q - 1) / Q;
  t->live = t->k >= 0 && (t->k == 0 || t->k < t->tiles);
  t->row = start + (t->live ? t->k * Q : 0);
  t->unit = (m.cu == nullptr ? t->s * ((int)(m.L + kUnit - 1) / kUnit) : start / kUnit + t->s) + t->k * (Q / kUnit);
  t->n = t->live ? min(len - t->k * Q, Q) : 0;
}

// LINK: piece number n of the batch, the ticket of the CTA's channel tile. Else tile number `step` of
// sequence n of equal lengths. BACK: from the last one on.
template <bool LINK, bool BACK, int Q>
__device__ __forceinline__ Tile tile_at(const GlParams& p, int n, int step) {
  Tile t;
  t.any = n < (int)(LINK ? p.m.pieces : p.m.S);
  t.live = false;
  t.j = t.k = t.n = t.s = t.tiles = t.row = t.unit = 0;
  if (!t.any) return t;
  if (LINK) {
    t.j = BACK ? (int)p.m.pieces - 1 - n : n;
    if (p.m.S > 0) find_tile<Q>(p.m, t.j, &t);
  } else {
    t.s = n;
    t.tiles = (int)p.m.per;
    t.k = BACK ? t.tiles - 1 - step : step;
    t.j = n * t.tiles + t.k;
    t.row = n * (int)p.m.L + t.k * Q;
    t.n = min((int)p.m.L - t.k * Q, Q);
    t.unit = n * ((int)(p.m.L + kUnit - 1) / kUnit) + t.k * (Q / kUnit);
    t.live = true;
  }
  return t;
}

// The rows that belong to no sequence, shared out over all threads: f(row, channel, channels).
template <class F>
__device__ __forceinline__ void unused_rows(const GlParams& p, F f) {
  if (p.m.cu == nullptr) return;
  const int64_t front = rows_begin(p.m), count = front + p.m.T - rows_end(p.m);
  const int quads = (p.C + 3) / 4;
  for (int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x; i < count * quads; i += (int64_t)gridDim.x * kT) {
    const int64_t r = i / quads;
    const int c = (int)(i - r * quads) * 4;
    f(r < front ? r : p.m.T - count + r, c, min(4, p.C - c));
  }
}

// Bytes of an element of a row.
__device__ __forceinline__ int element(int acc, int bf16) { return acc == kBf16 || (acc == kAny && bf16) ? 2 : 4; }

// Four elements into shared memory, zeros where there are none; on their way until copies_done(). Only
// the thread that asked for them reads them. (from may lie anywhere where `any` is false.)
template <int ACC>
__device__ __forceinline__ void bring_quad(typename RawQuad<ACC>::type* to, const char* from, bool any) {
  const unsigned at = (unsigned)__cvta_generic_to_shared(to);
  if constexpr (ACC == kBf16)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(at), "l"(from), "r"(any ? 8 : 0) : "memory");
  else
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(from), "r"(any ? 16 : 0) : "memory");
}

template <int ACC, int SEG, int OPS>
struct Stage {
  typename RawQuad<ACC>::type v[OPS][SEG][kT];
};

// What both kernels' CTAs have: their channel tile, and the order of their tiles. LINK: the tickets of the
// channel tile. Else they walk sequences, every (CTAs per channel tile)-th.
struct Place {
  int ct, c0, nn, lc, seg;  // channel tile, its first channel; the thread's channels, first of them in the tile, segment
  int walk;                 // sequences between two of the CTA's
};
__device__ __forceinline__ Place place_of(const GlParams& p) {
  Place at;
  at.ct = blockIdx.x % (unsigned)p.ctiles;
  at.c0 = at.ct * kCh;
  at.lc = threadIdx.x % (kCh / 4) * 4;
  at.seg = threadIdx.x / (kCh / 4);
  at.nn = max(0, min(p.C - at.c0 - at.lc, 4));
  at.walk = gridDim.x / (unsigned)p.ctiles;
  return at;
}

// The thread's rows of one operand, on their way into its own places.
template <int ACC, int SEG, int OPS>
__device__ __forceinline__ void bring(const GlParams& p, const Place& at, const Tile& w, Stage<ACC, SEG, OPS>& st, int op,
                                      const void* from, int64_t ld) {
  const int most = at.nn > 0 ? w.n - at.seg * SEG : 0;
  const int row = most > 0 ? w.row + at.seg * SEG : 0, ch = at.nn > 0 ? at.c0 + at.lc : 0;
  const int size = element(ACC, p.bf16);
  const char* src = reinterpret_cast<const char*>(from) + ((int64_t)row * (int)ld + ch) * size;
  const int64_t step = ld * size;
#pragma unroll
  for (int u = 0; u < SEG; ++u, src += step) {
    if constexpr (ACC == kAny) st.v[op][u][threadIdx.x] = load_quad<ACC>(src, 0, p.bf16, u < most ? at.nn : 0);
    else bring_quad<ACC>(&st.v[op][u][threadIdx.x], src, u < most);
  }
}

// The exponentials exp(-(r + r_bias)) and exp(-(i + i_bias)) of a thread's steps, which the backward takes twice.
template <int SEG>
struct Exps {
  float4 r[SEG][kT], i[SEG][kT];
};

// Decay a and input b = gain iota x of the thread's steps; the exponentials into `exps` where it is given.
template <int ACC, int SEG, bool SLOW, int OPS>
__device__ __forceinline__ void gate_steps(const GlParams& p, const Rates& rt, int lc, const Stage<ACC, SEG, OPS>& st, f2 (&a)[SEG][2],
                                           f2 (&b)[SEG][2], Exps<SEG>* exps) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int u = 0; u < SEG; ++u) {
    const typename RawQuad<ACC>::type rx = st.v[0][u][tid], rr = st.v[1][u][tid], ri = st.v[2][u][tid];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = lc + 2 * h;
      const f2 ar = gate_arg(pair_of<ACC>(rr, h, p.bf16), shared_pair(rt.r2, c));
      const f2 ai = gate_arg(pair_of<ACC>(ri, h, p.bf16), shared_pair(rt.i2, c));
      const f2 er = ex2_2(ar), ei = ex2_2(ai);
      f2 rho, m, gain;
      decay2<SLOW>(rsqrt_2(add2(er, both(1.f))), shared_pair(rt.speed, c), shared_pair(rt.root, c), &rho, &m, &a[u][h], &gain);
      const f2 iota = rcp_2(add2(ei, both(1.f)));
      if (exps != nullptr) {
        reinterpret_cast<f2*>(&exps->r[u][tid])[h] = er;
        reinterpret_cast<f2*>(&exps->i[u][tid])[h] = ei;
      }
      b[u][h] = mul2(mul2(iota, pair_of<ACC>(rx, h, p.bf16)), least2(gain));
    }
  }
}

// LINK: tiles linked through global memory. Else: sequences walked. Two barriers a tile: the maps are
// there; the segments' entry states are there.
template <int ACC, int SEG, bool LINK>
__global__ void __launch_bounds__(kT, kFwdCtas) gated_lru_fwd_kernel(const GlParams p) {
  typedef typename RawQuad<ACC>::type Raw;
  constexpr int Q = kSegs * SEG;
  extern __shared__ __align__(16) unsigned char raw[];
  Stage<ACC, SEG, 4>& st = *reinterpret_cast<Stage<ACC, SEG, 4>*>(raw);
  __shared__ __align__(16) float maps[2][2][kSegs][kCh];  // this tile's and the one's before: A, B
  __shared__ __align__(16) float entries[2][kCh];          // linked: state in front of the tile
  __shared__ Links links;
  __shared__ __align__(16) Rates rt;
  __shared__ int ticket;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  const Place at = place_of(p);
  const bool gated = p.z != nullptr;
  if (LINK && tid == 0) ticket = atomicAdd(&p.ticket[at.ct], 1);
  if (warp == 1) load_rates(p, at.c0, lane, &rt);
  unused_rows(p, [&](int64_t row, int c, int k) {
    store_quad<ACC>(p.y, row * p.C + c, p.bf16, k, make_float4(0.f, 0.f, 0.f, 0.f));
  });
  __syncthreads();
  int n = LINK ? ticket : (int)(blockIdx.x / (unsigned)p.ctiles), step = 0, buf = 0;
  __syncthreads();
  auto fetch = [&](const Tile& w) {
    bring(p, at, w, st, 0, p.x, p.ldx);
    bring(p, at, w, st, 1, p.r, p.ldr);
    bring(p, at, w, st, 2, p.i, p.ldi);
    if (gated) bring(p, at, w, st, 3, p.z, p.ldz);
  };
  const float4 sp = *reinterpret_cast<const float4*>(&rt.speed[at.lc]);
  const bool slow = fmaxf(fmaxf(sp.x, sp.y), fmaxf(sp.z, sp.w)) <= kNear;
  const int c = at.c0 + lane;  // warp 0: a lane per channel
  const bool ok = c < p.C;
  Tile w = tile_at<LINK, false, Q>(p, n, 0);
  fetch(w);
  float carry = 0.f;  // warp 0: the walked sequence's state
  while (w.any) {
    const bool first = w.k == 0, last = w.k + 1 >= w.tiles;
    int64_t slot = semx::kNone;
    if (p.m.n_slots > 0 && w.live && (first || last)) slot = find_slot(p.m, w.s);
    int drawn = 0;  // on its way while the tile's steps are folded
    if (LINK && tid == 0) drawn = atomicAdd(&p.ticket[at.ct], 1);
    float(*mA)[kCh] = maps[buf][0], (*mB)[kCh] = maps[buf][1];
    f2 a[SEG][2], b[SEG][2];
    f2 A[2] = {both(1.f), both(1.f)}, B[2] = {both(0.f), both(0.f)};
    Raw rz[SEG];
    copies_done();
    const int most = w.n - at.seg * SEG;  // steps of the thread that exist
    if (warp * (kSegs / 4) * SEG < w.n) {
      if (slow) gate_steps<ACC, SEG, true>(p, rt, at.lc, st, a, b, static_cast<Exps<SEG>*>(nullptr));
      else gate_steps<ACC, SEG, false>(p, rt, at.lc, st, a, b, static_cast<Exps<SEG>*>(nullptr));
      if (gated) {
#pragma unroll
        for (int u = 0; u < SEG; ++u) rz[u] = st.v[3][u][tid];
      }
    }
    if (most < SEG) {  // rows behind the last one keep the state
#pragma unroll
      for (int u = 0; u < SEG; ++u)
        if (u >= most) a[u][0] = a[u][1] = both(1.f), b[u][0] = b[u][1] = both(0.f);
    }
#pragma unroll
    for (int u = 0; u < SEG; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        A[h] = mul2(A[h], a[u][h]);
        B[h] = fma2(a[u][h], B[h], b[u][h]);
      }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      *reinterpret_cast<f2*>(&mA[at.seg][at.lc + 2 * h]) = A[h];
      *reinterpret_cast<f2*>(&mB[at.seg][at.lc + 2 * h]) = B[h];
    }
    if (LINK && tid == 0) ticket = drawn;
    __syncthreads();
    if (LINK) {
      n = ticket;
    } else if (++step == w.tiles) {
      step = 0;
      n += at.walk;
    }
    float h = 0.f;
    if (warp == 0 && first && ok && slot != semx::kNone) {
      const bool fresh = p.m.fresh != nullptr && p.m.fresh[w.s] != 0;
      h = slot == semx::kRefused ? __int_as_float(0x7fffffff) : fresh ? 0.f : p.state[slot * p.C + c];
    }
    const bool keeps = p.ckpt != nullptr && ok && w.live;
    float fA = 1.f, fB = 0.f, uA[Q / kUnit], uB[Q / kUnit];
    if (LINK && warp == 0) {
      // Behind this the maps of the steps in front of each segment stand in the segments' places.
#pragma unroll
      for (int s = 0; s < kSegs; ++s) {
        const float A = mA[s][lane], B = mB[s][lane];
        mA[s][lane] = fA;
        mB[s][lane] = fB;
        if (s % (kUnit / SEG) == 0) uA[s * SEG / kUnit] = fA, uB[s * SEG / kUnit] = fB;
        fA *= A;
        fB = fmaf(A, fB, B);
      }
      if (ok) leave_map(p, w.j, c, first ? 0.f : fA, first ? fmaf(fA, h, fB) : fB);
    }
    // The next tile's rows set out while this one's state is on its way; a walked sequence's warp 0 has the state to
    // find first.
    const Tile next = tile_at<LINK, false, Q>(p, n, step);
    if (LINK || warp != 0) fetch(next);
    if (LINK) {
      const bool waits = !first && w.live;  // of the whole CTA
      const Chain chain{w.j - w.k, 1, w.k};
      if (warp != 0) {
        if (waits) link_maps(p, chain, c, ok, links);
        links_left();
      }
      if (warp == 0) {
        if (waits) h = link_state(p, chain, c, ok);
        links_await();
        if (waits) h = link_all(links, h);
        entries[buf][lane] = h;
        // Every tile leaves its state, so that nothing waits for long whatever the offsets are.
        const float after = fmaf(fA, h, fB);
        if (ok) leave_state(p, w.j, c, after);
#pragma unroll
        for (int u = 0; u < Q / kUnit; ++u)
          if (keeps && (u == 0 || u * kUnit < w.n)) p.ckpt[((int64_t)w.unit + u) * p.C + c] = fmaf(uA[u], h, uB[u]);
        if (w.live && last && ok && slot >= 0) p.state[slot * p.C + c] = after;
      }
    } else if (warp == 0) {
      if (!first) h = carry;
#pragma unroll
      for (int s = 0; s < kSegs; ++s) {
        if (s % (kUnit / SEG) == 0 && keeps && (s == 0 || s * SEG < w.n)) p.ckpt[((int64_t)w.unit + s * SEG / kUnit) * p.C + c] = h;
        const float after = fmaf(mA[s][lane], h, mB[s][lane]);
        mB[s][lane] = h;  // from here on the segment's entry state
        h = after;
      }
      carry = h;
      if (last && ok && slot >= 0) p.state[slot * p.C + c] = h;
    }
    __syncthreads();
    if (!LINK && warp == 0) fetch(next);
    f2 hs[2] = {shared_pair(mB[at.seg], at.lc), shared_pair(mB[at.seg], at.lc + 2)};
    if (LINK) {
#pragma unroll
      for (int k = 0; k < 2; ++k) hs[k] = fma2(shared_pair(mA[at.seg], at.lc + 2 * k), shared_pair(entries[buf], at.lc + 2 * k), hs[k]);
    }
    char* out = reinterpret_cast<char*>(p.y) + ((int64_t)(w.row + at.seg * SEG) * p.C + at.c0 + at.lc) * element(ACC, p.bf16);
    const int64_t row = (int64_t)p.C * element(ACC, p.bf16);
    const int end = at.nn > 0 ? most : 0;
#pragma unroll
    for (int u = 0; u < SEG; ++u) {
      if (u >= end) break;
      f2 y[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        hs[k] = fma2(a[u][k], hs[k], b[u][k]);
        y[k] = hs[k];
        if (gated) {
          const f2 z = pair_of<ACC>(rz[u], k, p.bf16);
          y[k] = mul2(y[k], mul2(z, rcp_2(add2(ex2_2(mul2(z, both(-kLog2e))), both(1.f)))));
        }
      }
      const float2 lo = unpack2(y[0]), hi = unpack2(y[1]);
      store_quad<ACC>(out + u * row, 0, p.bf16, at.nn, make_float4(lo.x, lo.y, hi.x, hi.y));
    }
    w = next;
    buf ^= 1;
  }
}

// The gradients of the thread's steps, from the last one on. a: decays, b: the states in front, d: the
// gradients that reach h from y; gs: what reaches the last step from behind; sums over the steps of
// rho dla, dr and di are added to `sum`.
template <int ACC, int SEG, bool SLOW>
__device__ __forceinline__ void gradient_steps(const GlParams& p, const Rates& rt, const Place& at, const Stage<ACC, SEG, 5>& st,
                                               const Exps<SEG>& exps, int most, int row0, const f2 (&a)[SEG][2], const f2 (&b)[SEG][2], const f2 (&d)[SEG][2],
                                               f2 (&gs)[2], f2 (&sum)[3][2]) {
  typedef typename RawQuad<ACC>::type Raw;
  const int tid = threadIdx.x;
  const bool gated = p.z != nullptr;
  const int64_t out = ((int64_t)(row0 + at.seg * SEG) * p.C + at.c0 + at.lc) * element(ACC, p.bf16);
  const int64_t row = (int64_t)p.C * element(ACC, p.bf16);
#pragma unroll
  for (int u = SEG - 1; u >= 0; --u) {
    if (u >= most) continue;
    const Raw rx = st.v[0][u][tid], rg = st.v[4][u][tid];
    const f2* er_of = reinterpret_cast<const f2*>(&exps.r[u][tid]);
    const f2* ei_of = reinterpret_cast<const f2*>(&exps.i[u][tid]);
    f2 dx[2], dr[2], di[2], dz[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = at.lc + 2 * k;
      const f2 x = pair_of<ACC>(rx, k, p.bf16), speed = shared_pair(rt.speed, c);
      const f2 gt = add2(d[u][k], gs[k]);
      const f2 er = er_of[k], ei = ei_of[k];
      f2 rho, m, same, gain;
      decay2<SLOW>(rsqrt_2(add2(er, both(1.f))), speed, shared_pair(rt.root, c), &rho, &m, &same, &gain);
      const float2 gg = unpack2(gain);
      // -1 / gain; at its least value no gradient goes through the gain
      const f2 inv = pack2(gg.x > kLeastGain ? semx::rcp_approx(-gg.x) : 0.f, gg.y > kLeastGain ? semx::rcp_approx(-gg.y) : 0.f);
      gain = least2(gain);
      const f2 iota = rcp_2(add2(ei, both(1.f)));
      const f2 ah = mul2(a[u][k], b[u][k]);
      if (gated) {
        const f2 z = pair_of<ACC>(st.v[3][u][tid], k, p.bf16);
        const f2 ez = ex2_2(mul2(z, both(-kLog2e))), s = rcp_2(add2(ez, both(1.f)));
        const f2 h = fma2(mul2(gain, iota), x, ah);
        // silu'(z) = s (1 + z (1 - s))
        dz[k] = mul2(mul2(pair_of<ACC>(rg, k, p.bf16), h), mul2(s, fma2(z, rest2(ez, s), both(1.f))));
      }
      const f2 gi = mul2(gt, iota);
      dx[k] = mul2(gi, gain);
      di[k] = mul2(mul2(dx[k], x), rest2(ei, iota));
      const f2 dla = fma2(gt, ah, mul2(mul2(gi, x), mul2(mul2(a[u][k], a[u][k]), inv)));
      const f2 rd = mul2(rho, dla);
      dr[k] = mul2(mul2(rd, rest2(er, rho)), shared_pair(rt.minus, c));
      gs[k] = mul2(a[u][k], gt);
      sum[0][k] = add2(sum[0][k], rd);
      sum[1][k] = add2(sum[1][k], dr[k]);
      sum[2][k] = add2(sum[2][k], di[k]);
    }
    if (at.nn > 0) {
      const int64_t o = out + u * row;
      auto put = [&](void* to, const f2 (&v)[2]) {
        const float2 lo = unpack2(v[0]), hi = unpack2(v[1]);
        store_quad<ACC>(reinterpret_cast<char*>(to) + o, 0, p.bf16, at.nn, make_float4(lo.x, lo.y, hi.x, hi.y));
      };
      put(p.dx, dx);
      put(p.dr, dr);
      put(p.di, di);
      if (gated) put(p.dz, dz);
    }
  }
}

template <int ACC, int SEG, bool LINK>
__global__ void __launch_bounds__(kT, kBwdCtas) gated_lru_bwd_kernel(const GlParams p) {
  typedef typename RawQuad<ACC>::type Raw;
  constexpr int Q = kSegs * SEG;
  extern __shared__ __align__(16) unsigned char raw[];
  Stage<ACC, SEG, 5>* stages = reinterpret_cast<Stage<ACC, SEG, 5>*>(raw);  // this tile's and the next one's
  __shared__ __align__(16) float maps[2][3][kSegs][kCh];  // A, B, and B of the adjoint's map
  __shared__ __align__(16) float entries[2][kCh];         // linked: what reaches the tile's last step from behind
  __shared__ Links links;
  __shared__ __align__(16) Rates rt;
  __shared__ int ticket;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  const Place at = place_of(p);
  const bool gated = p.z != nullptr;
  if (LINK && tid == 0) ticket = atomicAdd(&p.ticket[at.ct], 1);
  if (warp == 1) load_rates(p, at.c0, lane, &rt);
  unused_rows(p, [&](int64_t row, int c, int k) {
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    store_quad<ACC>(p.dx, row * p.C + c, p.bf16, k, zero);
    store_quad<ACC>(p.dr, row * p.C + c, p.bf16, k, zero);
    store_quad<ACC>(p.di, row * p.C + c, p.bf16, k, zero);
    if (gated) store_quad<ACC>(p.dz, row * p.C + c, p.bf16, k, zero);
  });
  __syncthreads();
  int n = LINK ? ticket : (int)(blockIdx.x / (unsigned)p.ctiles), step = 0, buf = 0;
  __syncthreads();
  auto fetch = [&](const Tile& w, Stage<ACC, SEG, 5>& st) {
    bring(p, at, w, st, 0, p.x, p.ldx);
    bring(p, at, w, st, 1, p.r, p.ldr);
    bring(p, at, w, st, 2, p.i, p.ldi);
    bring(p, at, w, st, 4, p.dy, p.C);
    if (gated) bring(p, at, w, st, 3, p.z, p.ldz);
  };
  const float4 sp = *reinterpret_cast<const float4*>(&rt.speed[at.lc]);
  const bool slow = fmaxf(fmaxf(sp.x, sp.y), fmaxf(sp.z, sp.w)) <= kNear;
  const int c = at.c0 + lane;  // warp 0: a lane per channel
  const bool ok = c < p.C;
  Tile w = tile_at<LINK, true, Q>(p, n, 0);
  fetch(w, stages[0]);
  float carry = 0.f;  // warp 0: what reaches the walked sequence's tile from behind
  int summed = -1;    // row of partial sums that waits in shared memory
  auto write_sums = [&]() {
    if (summed < 0 || warp == 0 || !ok) return;
    const int k = warp - 1;
    float v = 0.f;
#pragma unroll
    for (int s = 0; s < kSegs; ++s) v += maps[buf ^ 1][k][s][lane];
    p.part[((int64_t)summed * 3 + k) * p.C + c] = k == 0 ? -rt.slope[lane] * v : v;
  };
  f2 sum[3][2];
#pragma unroll
  for (int k = 0; k < 3; ++k) sum[k][0] = sum[k][1] = both(0.f);
  while (w.any) {
    const bool end = w.k + 1 >= w.tiles;  // nothing behind it
    const int most = w.n - at.seg * SEG;  // steps of the thread that exist
    const bool busy = warp * (kSegs / 4) * SEG < w.n;
    int drawn = 0;  // on its way while the tile's steps are folded
    if (LINK && tid == 0) drawn = atomicAdd(&p.ticket[at.ct], 1);
    const float entry = warp == 0 && w.live && ok ? p.ckpt[(int64_t)w.unit * p.C + c] : 0.f;
    const Stage<ACC, SEG, 5>& st = stages[buf];
    // Wide rows' exponentials take the places of the gates that they are made of.
    static_assert(ACC == kBf16 || sizeof(Exps<SEG>) == 2 * sizeof(st.v[0]), "places");
    Exps<SEG>& exps = *reinterpret_cast<Exps<SEG>*>(ACC == kBf16 ? raw + 2 * sizeof(Stage<ACC, SEG, 5>) : reinterpret_cast<unsigned char*>(stages[buf].v[1]));
    float(*mA)[kCh] = maps[buf][0], (*mB)[kCh] = maps[buf][1], (*mG)[kCh] = maps[buf][2];
    // b: gain iota x, later the state in front of the step; d: the gradient that reaches h from y.
    f2 a[SEG][2], b[SEG][2], d[SEG][2];
    f2 A[2] = {both(1.f), both(1.f)}, B[2] = {both(0.f), both(0.f)}, G[2] = {both(0.f), both(0.f)};
    copies_done();
    if (busy) {
      if (slow) gate_steps<ACC, SEG, true>(p, rt, at.lc, st, a, b, &exps);
      else gate_steps<ACC, SEG, false>(p, rt, at.lc, st, a, b, &exps);
#pragma unroll
      for (int u = 0; u < SEG; ++u) {
        const Raw rg = st.v[4][u][tid];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          d[u][h] = pair_of<ACC>(rg, h, p.bf16);
          if (gated) {
            const f2 z = pair_of<ACC>(st.v[3][u][tid], h, p.bf16);
            d[u][h] = mul2(d[u][h], mul2(z, rcp_2(add2(ex2_2(mul2(z, both(-kLog2e))), both(1.f)))));
          }
        }
      }
    }
    if (most < SEG) {  // rows behind the last one keep the state
#pragma unroll
      for (int u = 0; u < SEG; ++u)
        if (u >= most) {
          a[u][0] = a[u][1] = both(1.f);
          b[u][0] = b[u][1] = d[u][0] = d[u][1] = both(0.f);
        }
    }
#pragma unroll
    for (int u = 0; u < SEG; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        A[h] = mul2(A[h], a[u][h]);
        B[h] = fma2(a[u][h], B[h], b[u][h]);
      }
    // What reaches the step in front of the segment: a_t (d_t + what reaches step t from behind).
#pragma unroll
    for (int u = SEG - 1; u >= 0; --u)
#pragma unroll
      for (int h = 0; h < 2; ++h) G[h] = mul2(a[u][h], add2(d[u][h], G[h]));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      *reinterpret_cast<f2*>(&mA[at.seg][at.lc + 2 * h]) = A[h];
      *reinterpret_cast<f2*>(&mB[at.seg][at.lc + 2 * h]) = B[h];
      *reinterpret_cast<f2*>(&mG[at.seg][at.lc + 2 * h]) = G[h];
    }
    if (LINK && tid == 0) ticket = drawn;
    __syncthreads();
    write_sums();  // of the tile before
    summed = -1;
    if (LINK) {
      n = ticket;
    } else if (++step == w.tiles) {
      step = 0;
      n += at.walk;
    }
    float fA = 1.f, fG = 0.f, behind[kSegs];
    if (LINK && warp == 0) {
#pragma unroll
      for (int s = kSegs - 1; s >= 0; --s) {
        const float A = mA[s][lane], G = mG[s][lane];
        behind[s] = fA;
        mG[s][lane] = fG;  // from here on the map of the steps behind the segment, A's part still to come
        fA *= A;
        fG = fmaf(A, fG, G);
      }
      if (ok) leave_map(p, w.j, c, end ? 0.f : fA, fG);
    }
    const Tile next = tile_at<LINK, true, Q>(p, n, step);
    if (LINK || warp != 0) fetch(next, stages[buf ^ 1]);
    const bool waits = LINK && !end && w.live;  // of the whole CTA
    const Chain chain{w.j - w.k + w.tiles - 1, -1, w.tiles - 1 - w.k};
    if (LINK && warp != 0) {
      if (waits) link_maps(p, chain, c, ok, links);
      links_left();
    }
    if (warp == 0) {
      float h = entry;
#pragma unroll
      for (int s = 0; s < kSegs; ++s) {
        const float after = fmaf(mA[s][lane], h, mB[s][lane]);
        mB[s][lane] = h;
        if (LINK) mA[s][lane] = behind[s];
        h = after;
      }
      float g = 0.f;
      if (LINK) {
        if (waits) g = link_state(p, chain, c, ok);
        links_await();
        if (waits) g = link_all(links, g);
        entries[buf][lane] = g;
        if (ok) leave_state(p, w.j, c, fmaf(fA, g, fG));
      } else {
        if (!end) g = carry;
#pragma unroll
        for (int s = kSegs - 1; s >= 0; --s) {
          const float before = fmaf(mA[s][lane], g, mG[s][lane]);
          mG[s][lane] = g;  // from here on what reaches the segment's last step from behind
          g = before;
        }
        carry = g;
      }
    }
    __syncthreads();
    if (!LINK && warp == 0) fetch(next, stages[buf ^ 1]);
    if (busy) {
      f2 hs[2] = {shared_pair(mB[at.seg], at.lc), shared_pair(mB[at.seg], at.lc + 2)};
#pragma unroll
      for (int u = 0; u < SEG; ++u)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const f2 after = fma2(a[u][k], hs[k], b[u][k]);
          b[u][k] = hs[k];
          hs[k] = after;
        }
      f2 gs[2] = {shared_pair(mG[at.seg], at.lc), shared_pair(mG[at.seg], at.lc + 2)};
      if (LINK) {
#pragma unroll
        for (int k = 0; k < 2; ++k) gs[k] = fma2(shared_pair(mA[at.seg], at.lc + 2 * k), shared_pair(entries[buf], at.lc + 2 * k), gs[k]);
      }
      if (slow) gradient_steps<ACC, SEG, true>(p, rt, at, st, exps, most, w.row, a, b, d, gs, sum);
      else gradient_steps<ACC, SEG, false>(p, rt, at, st, exps, most, w.row, a, b, d, gs, sum);
    }
    if (p.part != nullptr && (LINK || w.k == 0)) {
      // Into the segment's places among the maps, which only this thread has read since the barrier; behind the next
      // one the segments are added (exchanged between lanes first, 4 x 2047 x 2048 bf16 took 126 us, so 123).
#pragma unroll
      for (int k = 0; k < 3; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          *reinterpret_cast<f2*>(&maps[buf][k][at.seg][at.lc + 2 * h]) = sum[k][h];
          sum[k][h] = both(0.f);
        }
      summed = LINK ? w.j : w.s;
    }
    w = next;
    buf ^= 1;
  }
  __syncthreads();
  write_sums();
}

// One token per sequence: a thread has four channels of one, a CTA a run of sequences (their slots
// are looked up together, the parameters read once). Bound by its chain of slots, rows and state: 192 x 4096 fp32
// 6.2 us (22 MB), one row of 2048 3.5.
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
  float speed[4] = {}, root[4] = {}, r2[4] = {}, i2[4] = {};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < nn) {
      const float s = p.scale * semx::softplus(p.rate[c + k]);
      speed[k] = s > 1e37f ? 1e37f : s;
      root[k] = sqrtf(2.f * speed[k]);
      if (p.r_bias != nullptr) r2[k] = -kLog2e * p.r_bias[c + k];
      if (p.i_bias != nullptr) i2[k] = -kLog2e * p.i_bias[c + k];
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
        const float4 o = old[u];
        f2 hs[2] = {pack2(o.x, o.y), pack2(o.z, o.w)}, ys[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const f2 q = rsqrt_2(add2(ex2_2(gate_arg(pair_of<ACC>(rr[u], k, p.bf16), pack2(r2[2 * k], r2[2 * k + 1]))), both(1.f)));
          f2 rho, m, a, gain;
          decay2<false>(q, pack2(speed[2 * k], speed[2 * k + 1]), pack2(root[2 * k], root[2 * k + 1]), &rho, &m, &a, &gain);
          const f2 iota = rcp_2(add2(ex2_2(gate_arg(pair_of<ACC>(ri[u], k, p.bf16), pack2(i2[2 * k], i2[2 * k + 1]))), both(1.f)));
          hs[k] = fma2(a, hs[k], mul2(mul2(iota, pair_of<ACC>(rx[u], k, p.bf16)), least2(gain)));
          if (slot == semx::kRefused) hs[k] = both(__int_as_float(0x7fffffff));
          ys[k] = hs[k];
          if (p.z != nullptr) {
            const f2 z = pair_of<ACC>(rz[u], k, p.bf16);
            ys[k] = mul2(ys[k], mul2(z, rcp_2(add2(ex2_2(mul2(z, both(-kLog2e))), both(1.f)))));
          }
        }
        const float2 h0 = unpack2(hs[0]), h1 = unpack2(hs[1]), y0 = unpack2(ys[0]), y1 = unpack2(ys[1]);
        if (slot >= 0)
          store_quad<F>(p.state, slot * p.C + c, 0, nn, make_float4(h0.x, h0.y, h1.x, h1.y));
        store_quad<ACC>(p.y, s * p.C + c, p.bf16, nn, make_float4(y0.x, y0.y, y1.x, y1.y));
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
                   semx::aligned(a->workspace, 16),
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
  semx::set_pieces(&p->m, kSegs * (bwd ? kBwdSeg : kFwdSeg));
  return SEMX_OK;
}

// Whether tiles are linked: packed sequences, whose lengths the host does not know, and sequences too
// few to give each SM four CTAs that walk them. Sequences of 1000 steps, linked (with the clearing) and walked, us:
//   pairs of a sequence and a channel tile      128          256          384          512          768         3232 (321 steps)
//   forward bf16                             21 and 30    34 and 39    46 and 44    59 and 49    83 and 80    115 and 86
//   backward bf16                            39 and 55    72 and 67   105 and 84   138 and 103  205 and 176   281 and 186
// fp32 is alike. (By these figures a walk would pay from 384 pairs on, in the backward from 256.)
bool gl_linked(const GlParams& p) {
  if (p.m.cu != nullptr) return true;
  return p.m.per > 1 && p.m.S * p.ctiles < kSms * 4;
}

size_t link_bytes(const GlParams& p) {
  const size_t tickets = ((size_t)p.ctiles * sizeof(int) + 15) / 16 * 16;
  return gl_linked(p) ? tickets + (size_t)p.m.pieces * p.C * (sizeof(ulonglong2) + sizeof(unsigned long long)) : 0;
}
int64_t part_rows(const GlParams& p) { return gl_linked(p) ? p.m.pieces : p.m.S; }

// Lays the links into the workspace and clears them.
int set_links(GlParams* p, void* workspace, cudaStream_t st) {
  const size_t bytes = link_bytes(*p);
  if (bytes == 0) return SEMX_OK;
  SEMX_REQUIRE(workspace != nullptr, SEMX_ERR_WORKSPACE, "gated_lru: workspace is NULL");
  p->maps = reinterpret_cast<ulonglong2*>(workspace);
  p->left = reinterpret_cast<unsigned long long*>(p->maps + (size_t)p->m.pieces * p->C);
  p->ticket = reinterpret_cast<int*>(p->left + (size_t)p->m.pieces * p->C);
  const cudaError_t e = cudaMemsetAsync(workspace, 0, bytes, st);
  SEMX_REQUIRE(e == cudaSuccess, SEMX_ERR_LAUNCH, "gated_lru: cudaMemsetAsync: %s", cudaGetErrorString(e));
  return SEMX_OK;
}

template <int ACC>
int launch_gl(bool bwd, const GlParams& p, cudaStream_t st) {
  const bool linked = p.ticket != nullptr;
  const int64_t works = linked ? p.m.pieces : p.m.S;  // of each channel tile
  if (works == 0) return SEMX_OK;
  // As many CTAs as run at once, the same number for each channel tile: each takes tile after tile, and
  // fetches the next one's rows early.
  int64_t each = kSms * (bwd ? kBwdCtas : kFwdCtas) / p.ctiles;
  if (each > works) each = works;
  if (each < 1) each = 1;
  const unsigned n = (unsigned)(each * p.ctiles);
  constexpr size_t kStatic = 16 * 1024;  // shared memory of fixed size, at most
#define SEMX_GL(KERNEL, STAGES)                                      \
  do {                                                               \
    if ((STAGES) + kStatic > 48 * 1024 && !semx::allow_smem(KERNEL, (STAGES) + 48 * 1024)) return SEMX_ERR_LAUNCH; \
    KERNEL<<<n, kT, STAGES, st>>>(p);                                \
    return semx::check_launch("gated_lru kernel");                   \
  } while (0)
  constexpr size_t fwd = sizeof(Stage<ACC, kFwdSeg, 4>), back = 2 * sizeof(Stage<ACC, kBwdSeg, 5>) + (ACC == kBf16 ? sizeof(Exps<kBwdSeg>) : 0);
  if (!bwd && linked) SEMX_GL((gated_lru_fwd_kernel<ACC, kFwdSeg, true>), fwd);
  if (!bwd) SEMX_GL((gated_lru_fwd_kernel<ACC, kFwdSeg, false>), fwd);
  if (linked) SEMX_GL((gated_lru_bwd_kernel<ACC, kBwdSeg, true>), back);
  SEMX_GL((gated_lru_bwd_kernel<ACC, kBwdSeg, false>), back);
#undef SEMX_GL
}

int dispatch_gl(bool bwd, const GlParams& p, cudaStream_t st) {
  if (p.access == kBf16) return launch_gl<kBf16>(bwd, p, st);
  if (p.access == kFp32) return launch_gl<kFp32>(bwd, p, st);
  return launch_gl<kAny>(bwd, p, st);
}

// (The sizes do not depend on addresses.)
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
  if (p.m.S == 0 && p.m.T > 0 && p.m.pieces == 0) p.m.pieces = 1;
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
  GlParams p = gl_sizes(a, false, &rc);
  semx::set_pieces(&p.m, kUnit);
  return rc == SEMX_OK ? (size_t)p.m.pieces * p.C * sizeof(float) : 0;
}

size_t semx_gated_lru_workspace_bytes(const SemxGatedLruArgs* a, int32_t backward) {
  if (a == nullptr) return 0;
  int rc;
  const GlParams p = gl_sizes(a, backward != 0, &rc);
  if (rc != SEMX_OK) return 0;
  return link_bytes(p) + (backward != 0 ? (size_t)part_rows(p) * 3 * p.C * sizeof(float) : 0);
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
  // Without a sequence every row is a row behind the last one.
  if (p.m.S == 0 && p.m.T > 0 && p.m.pieces == 0) p.m.pieces = 1;
  rc = set_links(&p, a->workspace, st);
  if (rc != SEMX_OK) return rc;
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
  int64_t rows = 0;
  if (p.m.T > 0) {
    if (p.m.S == 0 && p.m.pieces == 0) p.m.pieces = 1;
    rc = set_links(&p, a->workspace, st);
    if (rc != SEMX_OK) return rc;
    if (params) {
      SEMX_REQUIRE(a->workspace != nullptr, SEMX_ERR_WORKSPACE, "gated_lru bwd: workspace is NULL");
      p.part = reinterpret_cast<float*>(reinterpret_cast<char*>(a->workspace) + link_bytes(p));
      rows = part_rows(p);
    }
    rc = dispatch_gl(true, p, st);
    if (rc != SEMX_OK) return rc;
  }
  if (!params) return SEMX_OK;
  semx::Segments seg = {};
  seg.n = 3;
  seg.out[0] = a->drate;
  seg.out[1] = a->dr_bias;
  seg.out[2] = a->di_bias;
  seg.len[0] = seg.len[1] = seg.len[2] = a->C;
  return semx::colsum_once(p.part, rows, 3 * a->C, seg, st);
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
