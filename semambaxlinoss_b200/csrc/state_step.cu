// Selective state scan of a single token per sequence, for sm_100a.
//
//   d = softplus(dt + dt_bias);  h[n] = exp(d A[n]) h[n] + d x B[n]  (in place)
//   v = sum_n C[n] h[n] + D x;   y = v silu(z)
//
// Bound: HBM for large batches (8 N bytes of state against 10 bytes of everything else per
// channel), the launch for small ones. A thread owns one channel and 4 neighbouring modes
// (one 16-byte access of the state where N is a multiple of 4), the lanes of a channel are
// neighbours, so a warp reads and writes consecutive state. A CTA takes a run of sequences:
// A, D and dt_bias are read once for all of them, and kAhead sequences' operands and states
// are loaded before the first is used.
#include "state_scan.cuh"

namespace {

using namespace semx_scan;

constexpr int kAhead = 4;
constexpr int kStepRows = 8;  // sequences per CTA at most

// ACC: how B and C are read; the state is read four modes at a time unless ACC is kAny.
template <int GL, int ACC>
__global__ void __launch_bounds__(kThreads) state_step_kernel(const ScanParams p, int rows) {
  constexpr int CH = kThreads / GL;
  __shared__ int64_t slots[kStepRows];
  const int64_t s0 = (int64_t)(blockIdx.x / p.ctiles) * rows;
  const int n = (int)min((int64_t)rows, p.m.S - s0);
  const int c = (blockIdx.x % p.ctiles) * CH + threadIdx.x / GL;
  const int lm = threadIdx.x % GL, n0 = lm * 4;
  const bool ok = c < p.C;
  const int cc = min(c, p.C - 1), g = cc / p.cpg;
  const int nn = min(4, p.N - n0);
  const float4 a4 = load_params(p.A, (int64_t)cc * p.N + n0, nn);
  const float A2[4] = {log2_rate(a4.x), log2_rate(a4.y), log2_rate(a4.z), log2_rate(a4.w)};
  const float bias = p.dt_bias != nullptr ? p.dt_bias[cc] : 0.f;
  const float D = p.D != nullptr ? p.D[cc] : 0.f;
  semx::find_slots<kStepRows>(p.m, s0, n, slots);
  // Row k R + lm of a batch of kAhead is this lane's for what a channel needs once (the step,
  // the gate, the store): the lanes of a channel share the rows instead of repeating them.
  constexpr int R = GL < kAhead ? GL : kAhead, PER = kAhead / R;
  const int first = (threadIdx.x & 31) - lm, own = lm % R;
  const int64_t cn = (int64_t)p.C * p.N;
  float* st0 = p.state + (int64_t)cc * p.N + n0;
  for (int i0 = 0; i0 < n; i0 += kAhead) {
    float4 h[kAhead];
    typename RawQuad<ACC>::type rB[kAhead], rC[kAhead];
    float d[PER], dx[PER], gate[PER], skip[PER];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      h[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      rB[u] = rC[u] = typename RawQuad<ACC>::type{};
      if (i0 + u < n && nn > 0) {
        const int64_t s = s0 + i0 + u, slot = slots[i0 + u];
        const bool cold = slot < 0 || (p.m.fresh != nullptr && p.m.fresh[s] != 0);
        if (!cold) {
          const float* st = st0 + slot * cn;
          if (ACC != kAny) h[u] = *reinterpret_cast<const float4*>(st);
          else h[u] = load_params(st, 0, nn);
        }
        rB[u] = load_quad<ACC>(p.B, s * p.ldb + (int64_t)g * p.N + n0, p.bf16, nn);
        rC[u] = load_quad<ACC>(p.Cm, s * p.ldc + (int64_t)g * p.N + n0, p.bf16, nn);
      }
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      d[k] = dx[k] = skip[k] = 0.f;
      gate[k] = 1.f;
      const int u = i0 + k * R + own;
      if (u < n) {
        const int64_t s = s0 + u;
        const float x = load(p.x, s * p.ldx + cc, p.bf16);
        d[k] = load(p.dt, s * p.lddt + cc, p.dt_bf16) + bias;
        if (p.softplus) d[k] = softplus(d[k]);
        dx[k] = d[k] * x;
        skip[k] = D * x;
        if (p.z != nullptr) {
          const float z = load(p.z, s * p.ldz + cc, p.bf16);
          gate[k] = z * sigmoid(z);
        }
        if (slots[u] == semx::kRefused) gate[k] = __int_as_float(0x7fffffff);
      }
    }
    float acc[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float du = __shfl_sync(0xffffffffu, d[u / R], first + u % R);
      const float xu = __shfl_sync(0xffffffffu, dx[u / R], first + u % R);
      const float4 B = quad_floats<ACC>(rB[u], p.bf16), C = quad_floats<ACC>(rC[u], p.bf16);
      float4 e = h[u];
      e.x = fmaf(pole(du, A2[0]), e.x, xu * B.x);
      e.y = fmaf(pole(du, A2[1]), e.y, xu * B.y);
      e.z = fmaf(pole(du, A2[2]), e.z, xu * B.z);
      e.w = fmaf(pole(du, A2[3]), e.w, xu * B.w);
      acc[u] = fmaf(e.x, C.x, fmaf(e.y, C.y, fmaf(e.z, C.z, e.w * C.w)));
      if (i0 + u < n && ok && nn > 0) {
        const int64_t slot = slots[i0 + u];
        if (slot >= 0) {
          float* st = st0 + slot * cn;
          if (ACC != kAny) *reinterpret_cast<float4*>(st) = e;
          else store_quad<kAny>(st, 0, 0, nn, e);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      float part[R];
#pragma unroll
      for (int r = 0; r < R; ++r) part[r] = acc[k * R + r];
      const float v = (lanes_scatter_sum<GL, R>(part, lm) + skip[k]) * gate[k];
      const int u = i0 + k * R + own;
      if (ok && lm < R && u < n) store(p.y, (s0 + u) * p.C + cc, p.bf16, v);
    }
  }
}

}  // namespace

extern "C" {

int semx_state_step(const SemxStateScanArgs* a, semx_stream_t stream) {
  SEMX_CHECK_ARGS(a, SemxStateScanArgs);
  ScanParams p = {};
  int rc = scan_validate(a, false, &p);
  if (rc != SEMX_OK) return rc;
  SEMX_REQUIRE(a->cu_seqlens == nullptr && (a->L == 1 || a->S == 0), SEMX_ERR_SHAPE, "state_step: one row per sequence");
  SEMX_REQUIRE(a->state != nullptr, SEMX_ERR_NULL, "state_step: state is NULL");
  if (p.m.S == 0) return SEMX_OK;
  semx::DeviceScope scope;
  rc = scope.bind({a->y});
  if (rc != SEMX_OK) return rc;
  cudaStream_t st = semx::as_stream(stream);
  const int gl = lanes_for(p.N, 4);
  p.ctiles = (int)semx::cdiv(p.C, (int64_t)(kThreads / gl));
  // Sequences per CTA: as many as leave eight CTAs per SM (192 x 4096, cold state: at most 4
  // 31.7 us, 8 28.6, 16 31.7).
  int rows = kStepRows;
  while (rows > 1 && semx::cdiv(p.m.S, rows) * p.ctiles < 148 * 8) rows /= 2;
  const int64_t grid = semx::cdiv(p.m.S, rows) * p.ctiles;
  if (grid >= ((int64_t)1 << 31)) return semx::fail(SEMX_ERR_SHAPE, "state_step: too many sequences");
  const int access = semx::aligned(p.state, 16) ? p.access : kAny;
  switch (gl) {
#define SEMX_GL(V)                                                                                       \
  case V:                                                                                                \
    if (access == kBf16) state_step_kernel<V, kBf16><<<(unsigned)grid, kThreads, 0, st>>>(p, rows);      \
    else if (access == kFp32) state_step_kernel<V, kFp32><<<(unsigned)grid, kThreads, 0, st>>>(p, rows); \
    else state_step_kernel<V, kAny><<<(unsigned)grid, kThreads, 0, st>>>(p, rows);                       \
    return semx::check_launch("state_step_kernel");
    SEMX_GL(1)
    SEMX_GL(2)
    SEMX_GL(4)
    SEMX_GL(8)
    SEMX_GL(16)
    SEMX_GL(32)
#undef SEMX_GL
  }
  return semx::fail(SEMX_ERR_UNSUPPORTED, "state_step: %d modes", p.N);
}

}  // extern "C"
