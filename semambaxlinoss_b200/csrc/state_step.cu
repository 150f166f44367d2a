// Selective state scan of a single token per sequence, for sm_100a.
//
//   d = softplus(dt + dt_bias);  h[n] = exp(d A[n]) h[n] + d x B[n]  (in place)
//   v = sum_n C[n] h[n] + D x;   y = v silu(z)
//
// Bound: HBM for large batches (8 N bytes of state against 10 bytes of everything else per
// channel), the launch for small ones. A thread owns one channel and 4 neighbouring modes
// (one 16-byte access of the state where N is a multiple of 4), the lanes of a channel are
// neighbours, so a warp reads and writes consecutive state. A row's operands are a few
// elements per thread and stay in L1.
#include "state_scan.cuh"

namespace {

using namespace semx_scan;

template <int GL, bool VEC>
__global__ void __launch_bounds__(kThreads) state_step_kernel(const ScanParams p) {
  constexpr int CH = kThreads / GL;
  const int64_t s = blockIdx.x / p.ctiles;
  const int c = (blockIdx.x % p.ctiles) * CH + threadIdx.x / GL;
  const int lm = threadIdx.x % GL, n0 = lm * 4;
  const bool ok = c < p.C;
  const int cc = min(c, p.C - 1), g = cc / p.cpg;
  // Everything that does not depend on the slot first.
  float A2[4], Bn[4], Cn[4], h[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const bool in = n0 + n < p.N;
    A2[n] = in ? p.A[(int64_t)cc * p.N + n0 + n] * kLog2e : 0.f;
    Bn[n] = in ? load(p.B, s * p.ldb + (int64_t)g * p.N + n0 + n, p.bf16) : 0.f;
    Cn[n] = in ? load(p.Cm, s * p.ldc + (int64_t)g * p.N + n0 + n, p.bf16) : 0.f;
  }
  const float x = load(p.x, s * p.ldx + cc, p.bf16);
  float d = load(p.dt, s * p.lddt + cc, p.dt_bf16) + (p.dt_bias != nullptr ? p.dt_bias[cc] : 0.f);
  const float z = p.z != nullptr ? load(p.z, s * p.ldz + cc, p.bf16) : 0.f;
  const float Dc = p.D != nullptr ? p.D[cc] : 0.f;
  const int64_t slot = find_slot(p.m, s);
  const bool cold = slot < 0 || (p.m.fresh != nullptr && p.m.fresh[s] != 0);
  float* st = p.state + (max(slot, (int64_t)0) * p.C + cc) * p.N + n0;
  if (VEC) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!cold && n0 < p.N) v = *reinterpret_cast<const float4*>(st);
    h[0] = v.x; h[1] = v.y; h[2] = v.z; h[3] = v.w;
  } else {
#pragma unroll
    for (int n = 0; n < 4; ++n) h[n] = !cold && n0 + n < p.N ? st[n] : 0.f;
  }
  if (p.softplus) d = softplus(d);
  float v = 0.f;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    h[n] = fmaf(pole(d, A2[n]), h[n], d * x * Bn[n]);
    v = fmaf(h[n], Cn[n], v);
  }
#pragma unroll
  for (int m = 1; m < GL; m *= 2) v += __shfl_xor_sync(0xffffffffu, v, m);
  if (!ok) return;
  if (slot >= 0) {
    if (VEC) {
      if (n0 < p.N) *reinterpret_cast<float4*>(st) = make_float4(h[0], h[1], h[2], h[3]);
    } else {
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (n0 + n < p.N) st[n] = h[n];
    }
  }
  if (lm == 0) {
    v = fmaf(Dc, x, v);
    if (p.z != nullptr) v *= z * sigmoid(z);
    if (slot == semx::kRefused) v = __int_as_float(0x7fffffff);
    store(p.y, s * p.C + cc, p.bf16, v);
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
  const int64_t grid = p.m.S * p.ctiles;
  if (grid >= ((int64_t)1 << 31)) return semx::fail(SEMX_ERR_SHAPE, "state_step: too many sequences");
  const bool vec = p.N % 4 == 0 && semx::aligned(p.state, 16);
  switch (gl) {
#define SEMX_GL(V)                                                                              \
  case V:                                                                                       \
    if (vec) state_step_kernel<V, true><<<(unsigned)grid, kThreads, 0, st>>>(p);                \
    else state_step_kernel<V, false><<<(unsigned)grid, kThreads, 0, st>>>(p);                   \
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
