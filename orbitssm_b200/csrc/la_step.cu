// One token of linear attention with a constant decay for each head (decode), one launch:
//   S' = a S + v k^T,    y = scale S' q        a = exp(log_decay[head]),  S [B, H, Dv, Dk] float32
// A group of LPR lanes owns a row of the state (a value channel): the row is read and written once in float4 accesses, the dot
// product with q is a shuffle sum.  ROWS rows a group keep that many 16-byte loads a thread in flight.  S' may be S itself:
// every element is read and written by the same thread, read first.
// HBM-bound: 8 bytes a state element and token.  2048 states of 128 x 128, bfloat16 operands, from memory: 49 us (5.5 TB/s), 8192 of
// them 174 us (6.2 TB/s, 94% of the measured copy); 2048 states of 96 x 128: 41 us (5.0 TB/s).  With clean lines in L2 before the call 42
// us for the first of these, 45 with float32 operands.
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

// VEC elements an access of the state (4, or 1 where Dk or the pointers do not allow it); QK4: q and k are read in fours as well
template <typename IO, int LPR, int ROWS, int VEC, bool QK4>
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
    if constexpr (QK4) {
      const uint2 ku = *reinterpret_cast<const uint2*>(k + x), qu = *reinterpret_cast<const uint2*>(q + x);
      unpack_bf16(ku.x, kk[0], kk[1]);
      unpack_bf16(ku.y, kk[2], kk[3]);
      unpack_bf16(qu.x, qq[0], qq[1]);
      unpack_bf16(qu.y, qq[2], qq[3]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) { kk[i] = ldf(k + x + i); qq[i] = ldf(q + x + i); }
    }
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

template <typename IO, int LPR, int VEC, bool QK4>
static int step_launch(const LaStepArgs& a, int64_t heads, cudaStream_t st) {
  constexpr int ROWS = 4, GROUPS = LS_THREADS / LPR;
  const int64_t grid = heads * ((a.Dv + GROUPS * ROWS - 1) / (GROUPS * ROWS));
  ORBIT_REQUIRE(grid <= 0x7fffffffLL, ERR_UNSUPPORTED, "orbit_la_step: %lld (batch, head) states are too many for one call", (long long)heads);
  la_step_kernel<IO, LPR, ROWS, VEC, QK4><<<(unsigned)grid, LS_THREADS, 0, st>>>(a);
  ORBIT_CHECK_LAUNCH("la_step_kernel");
  return OK;
}

// Lanes a row: 8, 16 or 32, what leaves the fewest of them without a float4 in the row's last access, the larger of equals
// (2048 states of 128 x 72: 35 us with 8 lanes, 45 with 32; of 128 x 128: 49 us with 32 lanes).
template <typename IO, bool QK4>
static int step_rows(const LaStepArgs& a, int64_t heads, cudaStream_t st) {
  const int n4 = a.Dk / 4, by8 = (n4 + 7) / 8 * 8, by16 = (n4 + 15) / 16 * 16, by32 = (n4 + 31) / 32 * 32;
  if (by32 <= by8) return step_launch<IO, 32, 4, QK4>(a, heads, st);
  if (by16 <= by8) return step_launch<IO, 16, 4, QK4>(a, heads, st);
  return step_launch<IO, 8, 4, QK4>(a, heads, st);
}
template <typename IO>
static int step_t(const LaStepArgs& a, int64_t heads, cudaStream_t st) {
  if (a.Dk % 4 == 0 && aligned16(a.s0) && aligned16(a.s1)) {
    // bfloat16 q and k in 8-byte reads where they lie so (8192 states of 128 x 128: 182 -> 174 us; wider reads of float32 ones
    // gained nothing)
    if constexpr (sizeof(IO) == 2) {
      if ((a.q_bs | a.q_hs | a.k_bs | a.k_hs) % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k)) & 7) == 0)
        return step_rows<IO, true>(a, heads, st);
    }
    return step_rows<IO, false>(a, heads, st);
  }
  return step_launch<IO, 32, 1, false>(a, heads, st);
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
