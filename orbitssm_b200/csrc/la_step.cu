// One token of linear attention with a constant decay for each head (decode), one launch:
//   S' = a S + v k^T,    y = scale S' q        a = exp(log_decay[head]),  S [B, H, Dv, Dk] float32
// A group of LPR lanes owns a row of the state (a value channel): the row is read and written once in float4 accesses, the dot
// product with q is a shuffle sum.  ROWS rows a group keep that many 16-byte loads a thread in flight.  S' may be S itself:
// every element is read and written by the same thread, read first.
// HBM-bound: 8 bytes a state element and token.
#include "common.cuh"
#include "../../include/orbit_b200.h"

namespace orbit {

constexpr int LS_THREADS = 128;

struct LaStepArgs {
  const void *q, *k, *v;
  int64_t q_bs, q_hs, k_bs, k_hs, v_bs, v_hs;
  const float *log_decay, *s0;
  float* s1;
  void* y;
  int H, Dk, Dv;
  float scale;
};

// VEC elements an access (4, or 1 where Dk or the pointers do not allow it)
template <typename IO, int LPR, int ROWS, int VEC>
__global__ void __launch_bounds__(LS_THREADS) la_step_kernel(const LaStepArgs a) {
  constexpr int GROUPS = LS_THREADS / LPR;
  const int sub = threadIdx.x % LPR, grp = threadIdx.x / LPR, Dk = a.Dk, Dv = a.Dv;
  const int tiles = (Dv + GROUPS * ROWS - 1) / (GROUPS * ROWS);
  const int64_t head = blockIdx.x / tiles;
  const int h = (int)(head % a.H);
  const int64_t b = head / a.H;
  const int e0 = (int)(blockIdx.x % tiles) * (GROUPS * ROWS) + grp;   // rows e0, e0 + GROUPS, ...
  const IO* q = (const IO*)a.q + b * a.q_bs + h * a.q_hs;
  const IO* k = (const IO*)a.k + b * a.k_bs + h * a.k_hs;
  const IO* v = (const IO*)a.v + b * a.v_bs + h * a.v_hs;
  const float* s0 = a.s0 + head * Dv * Dk;
  float* s1 = a.s1 + head * Dv * Dk;
  float dot[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) dot[r] = 0.f;
  for (int x = sub * VEC; x < Dk; x += LPR * VEC) {
    float s[ROWS][VEC];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int e = e0 + r * GROUPS;
      if (e < Dv) {
        if constexpr (VEC == 4) {
          const float4 t = *reinterpret_cast<const float4*>(s0 + (int64_t)e * Dk + x);
          s[r][0] = t.x; s[r][1] = t.y; s[r][2] = t.z; s[r][3] = t.w;
        } else {
          s[r][0] = s0[(int64_t)e * Dk + x];
        }
      }
    }
    const float dec = expf(a.log_decay[h]);
    float kk[VEC], qq[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) { kk[i] = ldf(k + x + i); qq[i] = ldf(q + x + i); }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int e = e0 + r * GROUPS;
      if (e < Dv) {
        const float vv = ldf(v + e);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          s[r][i] = fmaf(dec, s[r][i], vv * kk[i]);
          dot[r] = fmaf(s[r][i], qq[i], dot[r]);
        }
        if constexpr (VEC == 4) *reinterpret_cast<float4*>(s1 + (int64_t)e * Dk + x) = make_float4(s[r][0], s[r][1], s[r][2], s[r][3]);
        else s1[(int64_t)e * Dk + x] = s[r][0];
      }
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) dot[r] += __shfl_xor_sync(0xffffffffu, dot[r], o);
    const int e = e0 + r * GROUPS;
    if (sub == 0 && e < Dv) stf((IO*)a.y + head * Dv + e, a.scale * dot[r]);
  }
}

template <typename IO, int LPR, int VEC>
static int step_launch(const LaStepArgs& a, int64_t heads, cudaStream_t st) {
  constexpr int ROWS = 4, GROUPS = LS_THREADS / LPR;
  const int64_t grid = heads * ((a.Dv + GROUPS * ROWS - 1) / (GROUPS * ROWS));
  ORBIT_REQUIRE(grid <= 0x7fffffffLL, ERR_UNSUPPORTED, "orbit_la_step: %lld (batch, head) states are too many for one call", (long long)heads);
  la_step_kernel<IO, LPR, ROWS, VEC><<<(unsigned)grid, LS_THREADS, 0, st>>>(a);
  ORBIT_CHECK_LAUNCH("la_step_kernel");
  return OK;
}

// lanes a row: as many as its float4s, a power of two from 8 to 32
template <typename IO>
static int step_t(const LaStepArgs& a, int64_t heads, cudaStream_t st) {
  if (a.Dk % 4 == 0 && aligned16(a.s0) && aligned16(a.s1)) {
    if (a.Dk <= 32) return step_launch<IO, 8, 4>(a, heads, st);
    if (a.Dk <= 64) return step_launch<IO, 16, 4>(a, heads, st);
    return step_launch<IO, 32, 4>(a, heads, st);
  }
  return step_launch<IO, 32, 1>(a, heads, st);
}

}  // namespace orbit

using namespace orbit;

extern "C" int orbit_la_step(const void* q, int64_t q_bs, int64_t q_hs, const void* k, int64_t k_bs, int64_t k_hs, const void* v,
                             int64_t v_bs, int64_t v_hs, const float* log_decay, const float* state0, float* state1, void* y,
                             int B, int H, int Dk, int Dv, float scale, int dtype, void* stream) {
  ORBIT_REQUIRE(B >= 0 && H > 0 && Dk > 0 && Dv > 0, ERR_BAD_ARG, "orbit_la_step: bad sizes B=%d H=%d Dk=%d Dv=%d", B, H, Dk, Dv);
  ORBIT_REQUIRE(dtype == BF16 || dtype == F32, ERR_BAD_ARG, "orbit_la_step: unknown dtype code %d", dtype);
  if (B == 0) return OK;
  ORBIT_REQUIRE(q && k && v && log_decay && state0 && state1 && y, ERR_BAD_ARG, "orbit_la_step: null pointer");
  LaStepArgs a = {q, k, v, q_bs, q_hs, k_bs, k_hs, v_bs, v_hs, log_decay, state0, state1, y, H, Dk, Dv, scale};
  const int64_t heads = (int64_t)B * H;
  return dtype == BF16 ? step_t<__nv_bfloat16>(a, heads, (cudaStream_t)stream) : step_t<float>(a, heads, (cudaStream_t)stream);
}
