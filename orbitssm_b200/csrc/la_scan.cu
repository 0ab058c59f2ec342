// Linear attention with a constant decay for each head, float32 kernels (any head widths up to 256, either IO dtype) and the
// entry points.
//
//   S_t = a S_{t-1} + v_t k_t^T,   y_t = scale S_t q_t,   a = exp(log_decay[head]),   S [Dv, Dk] float32
//
// In chunks of T tokens, entering state Z = S^T:
//   P[t,s] = a^{t-s} (q_t . k_s) for s <= t;   y = scale (P V + a^{t+1} Q Z);   Z' = a^T Z + sum_s a^{T-1-s} k_s v_s^T
// All four directions (y, dq, dk, dv) are this pass with the operands in other roles, forwards or backwards in time: see
// LaJob.  Backwards in time the factors are counted from the chunk's other end; the carry is the gradient of the state after
// the chunk, so the row factor is a^{T-1-t} and the write factor a^{s+1}.
//
// Few (batch, head) pairs and a long sequence: the sequence is split into segments.  A first launch forms what each segment
// alone adds to the state, a second joins these shares into the states that enter the segments, and each CTA of the third walks
// its segment from there.  No CTA waits on another.
//
// One CTA of 256 threads owns a head's segment and 64 output channels; 4 x 4 register tiles (float4 reads of operands that
// are kept transposed in shared memory).  The FP32 pipe bounds it: a chunk of 64 tokens of a 128 x 64 tile is 14000 cycles of FMAs,
// and the chunks take 1.9 times that (half of the scores are masked work, and the reads of a chunk are not hidden).  Measured in
// float32: [8, 4096, 16, 128, 128] 2771 us, [2, 777, 8, 64, 64] forward 53 us and backward 99.
#include "common.cuh"
#include "la_args.h"
#include <math.h>

namespace orbit {

constexpr int LG_THREADS = 256, LG_E = 64;

// smem floats of a chunk size
static int64_t lg_floats(int T, int X) {
  const int64_t X4 = (X + 3) / 4 * 4, TS = T + 4;
  return 2 * X4 * TS + (int64_t)T * LG_E + X4 * LG_E + (int64_t)T * TS + 2 * (T + 4) + 8;
}

template <typename IO, int T>
__global__ void __launch_bounds__(LG_THREADS) la_generic_kernel(const __grid_constant__ LaPlan p, const int local) {
  constexpr int TS = T + 4, TM = T / 16;              // padded row of the transposed operands; rows of a thread's tile
  extern __shared__ float4 sm4[];
  const LaJob& J = p.job[blockIdx.y];
  const int X = J.X, E = J.E, X4 = (X + 3) / 4 * 4, rev = J.reverse;
  const int etiles = (E + LG_E - 1) / LG_E;
  int64_t id = blockIdx.x;
  const int64_t units = (int64_t)p.B * p.H * p.nseg * etiles;
  if (id >= units) return;
  const int et = (int)(id % etiles);
  id /= etiles;
  const int seg = (int)(id % p.nseg);
  id /= p.nseg;
  const int h = (int)(id % p.H), b = (int)(id / p.H), e0 = et * LG_E;
  if (local && seg == (rev ? 0 : p.nseg - 1)) return;  // nobody reads the last segment's share

  float* QT = reinterpret_cast<float*>(sm4);           // [X4][TS]
  float* KT = QT + (int64_t)X4 * TS;                   // [X4][TS]
  float* Vs = KT + (int64_t)X4 * TS;                   // [T][64]
  float* Z = Vs + T * LG_E;                            // [X4][64]
  float* PT = Z + (int64_t)X4 * LG_E;                  // [s][t], row TS
  float* pw = PT + T * TS;                             // a^0 .. a^T
  float* fw = pw + T + 4;                              // write factor of each token of the chunk
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, lane = tid & 31, warp = tid >> 5;
  const double ld = (double)p.log_decay[h];
  if (tid <= T) pw[tid] = tid == 0 ? 1.f : (float)exp(ld * tid);

  const int s0 = seg * p.seg_len, s1 = min(p.L, s0 + p.seg_len);
  const int64_t head = (int64_t)b * p.H + h;
  // the state that enters the segment (joined from the segments' shares, or the carried one)
  const float* enter = local ? nullptr : J.part ? J.part + (head * p.nseg + seg) * p.S : J.z0 ? J.z0 + head * p.S : nullptr;
  // (the axis that lies dense goes along the lanes; eight reads in flight)
  auto z_in = [&](int x, int e) { return enter && x < X && e0 + e < E ? enter[x * J.xs + (e0 + e) * J.es] : 0.f; };
  if (J.xs == 1) {
    for (int x = lane; x < X4; x += 32) {
      float r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = z_in(x, warp * 8 + i);
      float4* d = reinterpret_cast<float4*>(Z + x * LG_E + warp * 8);
      d[0] = make_float4(r[0], r[1], r[2], r[3]);
      d[1] = make_float4(r[4], r[5], r[6], r[7]);
    }
  } else {
    for (int x = warp; x < X4; x += 32) {
      float r[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) { r[i][0] = z_in(x + 8 * i, lane); r[i][1] = z_in(x + 8 * i, lane + 32); }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (x + 8 * i < X4) { Z[(x + 8 * i) * LG_E + lane] = r[i][0]; Z[(x + 8 * i) * LG_E + lane + 32] = r[i][1]; }
    }
  }

  const IO* q = (const IO*)J.q + b * J.q_bs + h * J.q_hs;
  const IO* k = (const IO*)J.k + b * J.k_bs + h * J.k_hs;
  const IO* v = (const IO*)J.v + b * J.v_bs + h * J.v_hs + e0;
  IO* y = (IO*)J.y + b * J.y_bs + h * J.y_hs + e0;
  const int nch = (s1 - s0 + T - 1) / T;
  for (int ci = 0; ci < nch; ++ci) {
    const int t0 = s0 + (rev ? nch - 1 - ci : ci) * T, Tv = min(T, s1 - t0);
    __syncthreads();
    // a warp owns RT tokens: its lanes read along the rows, RT reads a lane and operand in flight, and store the tokens side by
    // side (float4, eight lanes on 32 different banks)
    constexpr int RT = T / 8;
#pragma unroll 2
    for (int x = lane; x < X4; x += 32) {
      float rk[RT], rq[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int t = warp * RT + i;
        const bool in = t < Tv && x < X;
        rk[i] = in ? ldf(k + (int64_t)(t0 + t) * J.k_ls + x) : 0.f;
        rq[i] = in && !local ? ldf(q + (int64_t)(t0 + t) * J.q_ls + x) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < RT; i += 4) {
        *reinterpret_cast<float4*>(KT + x * TS + warp * RT + i) = make_float4(rk[i], rk[i + 1], rk[i + 2], rk[i + 3]);
        if (!local) *reinterpret_cast<float4*>(QT + x * TS + warp * RT + i) = make_float4(rq[i], rq[i + 1], rq[i + 2], rq[i + 3]);
      }
    }
    {
      float rv[RT][2];
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int t = warp * RT + i;
#pragma unroll
        for (int j = 0; j < 2; ++j) rv[i][j] = t < Tv && e0 + lane + 32 * j < E ? ldf(v + (int64_t)(t0 + t) * J.v_ls + lane + 32 * j) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) Vs[(warp * RT + i) * LG_E + lane + 32 * j] = rv[i][j];
    }
    if (tid < T) fw[tid] = tid < Tv ? J.s_state * pw[rev ? tid + 1 : Tv - 1 - tid] : 0.f;
    __syncthreads();
    if (!local) {
      // scores, decayed, transposed: thread (ty, tx) owns rows t = ty TM.., columns s = tx TM..
      float acc[TM][TM];
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = 0.f;
#pragma unroll 4
      for (int x = 0; x < X; ++x) {
        float a[TM], c[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) { a[i] = QT[x * TS + ty * TM + i]; c[i] = KT[x * TS + tx * TM + i]; }
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TM; ++j) acc[i][j] = fmaf(a[i], c[j], acc[i][j]);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          const int t = ty * TM + i, s = tx * TM + j, d = rev ? s - t : t - s;
          PT[s * TS + t] = d >= 0 ? acc[i][j] * pw[d] : 0.f;
        }
      // what the entering state gives, rows t = ty TM.., channels e = tx 4..
      float o[TM][4];
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
#pragma unroll 4
      for (int x = 0; x < X; ++x) {
        const float4 z = *reinterpret_cast<const float4*>(Z + x * LG_E + tx * 4);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const float a = QT[x * TS + ty * TM + i];
          o[i][0] = fmaf(a, z.x, o[i][0]);
          o[i][1] = fmaf(a, z.y, o[i][1]);
          o[i][2] = fmaf(a, z.z, o[i][2]);
          o[i][3] = fmaf(a, z.w, o[i][3]);
        }
      }
      const float ratio = J.s_in / J.s_out;            // s_in is s_out or 1: folded so that one product by s_out ends the sum
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int t = ty * TM + i;
        const float f = t < Tv ? pw[rev ? Tv - 1 - t : t + 1] * ratio : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] *= f;
      }
      __syncthreads();
      // (only the tokens that a row of this tile sees)
      const int sa = rev ? ty * TM : 0, sb = rev ? T : ty * TM + TM;
#pragma unroll 4
      for (int s = sa; s < sb; ++s) {
        const float4 w = *reinterpret_cast<const float4*>(Vs + s * LG_E + tx * 4);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const float a = PT[s * TS + ty * TM + i];
          o[i][0] = fmaf(a, w.x, o[i][0]);
          o[i][1] = fmaf(a, w.y, o[i][1]);
          o[i][2] = fmaf(a, w.z, o[i][2]);
          o[i][3] = fmaf(a, w.w, o[i][3]);
        }
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int t = ty * TM + i;
        if (t < Tv)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (e0 + tx * 4 + j < E) stf(y + (int64_t)(t0 + t) * J.y_ls + tx * 4 + j, J.s_out * o[i][j]);
      }
    }
    // state: rows x = ty 4 + 64 r.., channels e = tx 4..; every thread reads and writes its own elements of Z only, and the
    // reads of Z above lie before the barrier that preceded the second product
    const float aT = pw[Tv];
    if (local) __syncthreads();
    for (int xb = ty * 4; xb < X4; xb += 64) {
      float z[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) z[i][j] = 0.f;
#pragma unroll 2
      for (int s = 0; s < T; s += 4) {
        float4 kk[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) kk[i] = *reinterpret_cast<const float4*>(KT + (xb + i) * TS + s);
        const float4 f = make_float4(fw[s], fw[s + 1], fw[s + 2], fw[s + 3]);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float4 w = *reinterpret_cast<const float4*>(Vs + (s + u) * LG_E + tx * 4);
          const float fu = reinterpret_cast<const float*>(&f)[u];
          w.x *= fu; w.y *= fu; w.z *= fu; w.w *= fu;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float ku = reinterpret_cast<const float*>(&kk[i])[u];
            z[i][0] = fmaf(ku, w.x, z[i][0]);
            z[i][1] = fmaf(ku, w.y, z[i][1]);
            z[i][2] = fmaf(ku, w.z, z[i][2]);
            z[i][3] = fmaf(ku, w.w, z[i][3]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float4* dst = reinterpret_cast<float4*>(Z + (xb + i) * LG_E + tx * 4);
        float4 c = *dst;
        c.x = fmaf(aT, c.x, z[i][0]);
        c.y = fmaf(aT, c.y, z[i][1]);
        c.z = fmaf(aT, c.z, z[i][2]);
        c.w = fmaf(aT, c.w, z[i][3]);
        *dst = c;
      }
    }
  }
  float* out = local ? J.part + (head * p.nseg + seg) * p.S
                     : (J.z1 && seg == (rev ? 0 : p.nseg - 1) ? J.z1 + head * p.S : nullptr);
  if (!out) return;
  __syncthreads();
  if (J.xs == 1) {
    for (int x = lane; x < X; x += 32)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e0 + warp * 8 + i < E) out[x + (e0 + warp * 8 + i) * J.es] = Z[x * LG_E + warp * 8 + i];
  } else {
    for (int i = tid; i < X * LG_E; i += LG_THREADS) {
      const int e = i % LG_E, x = i / LG_E;
      if (e0 + e < E) out[x * J.xs + (e0 + e) * J.es] = Z[i];
    }
  }
}

// One thread an element of a head's state: walks the segments in the direction's order, in place, eight reads in flight.
__global__ void __launch_bounds__(256) la_join_kernel(const __grid_constant__ LaPlan p) {
  constexpr int AHEAD = 8;
  const LaJob& J = p.job[blockIdx.y];
  const int blocks = (p.S + 255) / 256, rev = J.reverse, n = p.nseg;
  const int i = (int)(blockIdx.x % blocks) * 256 + threadIdx.x;
  const int64_t head = blockIdx.x / blocks;
  if (i >= p.S) return;
  float* part = J.part + head * n * p.S + i;
  float z = J.z0 ? J.z0[head * p.S + i] : 0.f;
  const double ld = (double)p.log_decay[head % p.H];
  const float full = (float)exp(ld * p.seg_len), last = (float)exp(ld * (p.L - (n - 1) * p.seg_len));
  for (int k0 = 0; k0 < n; k0 += AHEAD) {
    float share[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int k = k0 + j;
      share[j] = k < n - 1 ? part[(int64_t)(rev ? n - 1 - k : k) * p.S] : 0.f;      // nobody formed the last one's
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int k = k0 + j, s = rev ? n - 1 - k : k;
      if (k < n) {
        part[(int64_t)s * p.S] = z;
        z = fmaf(s == n - 1 ? last : full, z, share[j]);
      }
    }
  }
}

int la_join(const LaPlan& p, cudaStream_t st) {
  const int64_t grid = (int64_t)p.B * p.H * ((p.S + 255) / 256);
  ORBIT_REQUIRE(grid <= 0x7fffffffLL, ERR_UNSUPPORTED, "orbit_la: %lld (batch, head) states are too many for one call", (long long)p.B * p.H);
  la_join_kernel<<<dim3((unsigned)grid, p.njobs), 256, 0, st>>>(p);
  ORBIT_CHECK_LAUNCH("la_join_kernel");
  return OK;
}

int la_plan(const LaArgs& a, bool bwd, int nseg, int seg_len, bool local, LaPlan* p) {
  *p = LaPlan{};
  p->B = a.B; p->L = a.L; p->H = a.H; p->S = a.Dk * a.Dv;
  p->nseg = nseg; p->seg_len = seg_len;
  p->log_decay = a.log_decay; p->status = a.status;
  const int64_t share = (int64_t)a.B * a.H * nseg * p->S;
  float* pf = nseg > 1 ? (float*)a.workspace : nullptr;                 // shares forwards in time
  float* pr = nseg > 1 ? (float*)a.workspace + (bwd ? share : 0) : nullptr;   // and backwards
  auto in = [](LaJob& j, char role, const void* ptr, int64_t bs, int64_t ls, int64_t hs) {
    if (role == 'q') { j.q = ptr; j.q_bs = bs; j.q_ls = ls; j.q_hs = hs; }
    if (role == 'k') { j.k = ptr; j.k_bs = bs; j.k_ls = ls; j.k_hs = hs; }
    if (role == 'v') { j.v = ptr; j.v_bs = bs; j.v_ls = ls; j.v_hs = hs; }
  };
  auto q = [&](LaJob& j, char r) { in(j, r, a.q, a.q_bs, a.q_ls, a.q_hs); };
  auto k = [&](LaJob& j, char r) { in(j, r, a.k, a.k_bs, a.k_ls, a.k_hs); };
  auto v = [&](LaJob& j, char r) { in(j, r, a.v, a.v_bs, a.v_ls, a.v_hs); };
  auto g = [&](LaJob& j, char r) { in(j, r, a.dy, a.dy_bs, a.dy_ls, a.dy_hs); };
  auto out = [](LaJob& j, void* ptr, int64_t bs, int64_t ls, int64_t hs) { j.y = ptr; j.y_bs = bs; j.y_ls = ls; j.y_hs = hs; };
  auto kv = [&](LaJob& j, bool x_is_k, int rev, float so, float si, float sz) {
    j.X = x_is_k ? a.Dk : a.Dv; j.E = x_is_k ? a.Dv : a.Dk;
    j.xs = x_is_k ? 1 : a.Dk;   j.es = x_is_k ? a.Dk : 1;
    j.reverse = rev; j.s_out = so; j.s_in = si; j.s_state = sz;
    j.part = rev ? pr : pf;
  };
  const float sc = a.scale;
  int n = 0;
  if (!bwd || local) {                                  // y; and the forward shares of either direction
    LaJob& j = p->job[n++];
    kv(j, true, 0, sc, sc, 1.f);
    q(j, 'q'); k(j, 'k'); v(j, 'v');
    out(j, a.y, a.y_bs, a.y_ls, a.y_hs);
    j.z0 = a.state0; j.z1 = a.state1;
  }
  if (bwd && !local) {                                  // dq = scale S^T dy
    LaJob& j = p->job[n++];
    kv(j, false, 0, sc, sc, 1.f);
    g(j, 'q'); v(j, 'k'); k(j, 'v');
    out(j, a.dq, a.dq_bs, a.dq_ls, a.dq_hs);
    j.z0 = a.state0;
  }
  if (bwd && !local) {                                  // dk = dS^T v
    LaJob& j = p->job[n++];
    kv(j, false, 1, sc, 1.f, sc);
    v(j, 'q'); g(j, 'k'); q(j, 'v');
    out(j, a.dk, a.dk_bs, a.dk_ls, a.dk_hs);
    j.z0 = a.dstate1;
  }
  if (bwd) {                                            // dv = dS k; and the backward shares
    LaJob& j = p->job[n++];
    kv(j, true, 1, sc, 1.f, sc);
    k(j, 'q'); q(j, 'k'); g(j, 'v');
    out(j, a.dv, a.dv_bs, a.dv_ls, a.dv_hs);
    j.z0 = a.dstate1; j.z1 = a.dstate0;
  }
  p->njobs = n;
  return OK;
}

// The split that takes the fewest chunk steps on 148 SMs: rounds of CTAs times the chunks of a segment and `setup` steps' worth of
// prologue and state; for more than one segment also the first launch, which reads half of the operands and costs about half a step
// for each, and `join` steps for the launch between the two.  At most 32 segments: `join` is a constant, and the joining launch walks a
// head's segments one after another.  A call of few heads then leaves SMs idle ([1, 65536, H, 128, 128] bfloat16: H = 1 104 us on 32
// CTAs, H = 2 113, H = 4 125, H = 16 340).
// (Tensor-core tiles, 16 heads of 128 x 128, one segment against the split taken: 2048 tokens 51 us and 47, 8192 tokens 167 and 76,
// 65536 tokens 1233 and 341.  Float32, [2, 777, 8, 64, 64]: 156 and 53.)
int la_segments(int64_t units, int L, int chunk, double setup, double join, int* seg_len, double* cost_out) {
  const int nch = (L + chunk - 1) / chunk;
  int best = 1, best_len = nch;
  double best_cost = 0.;
  for (int n = 1; n <= 32 && n <= nch; ++n) {
    const int per = (nch + n - 1) / n, ns = (nch + per - 1) / per;
    if (ns != n) continue;
    const int64_t rounds = (units * n + 147) / 148, first = (units * (n - 1) + 147) / 148;
    const double cost = (double)rounds * (per + setup) + (n > 1 ? 0.5 * (double)first * (per + setup) + join : 0.);
    if (n == 1 || cost < 0.95 * best_cost) { best = n; best_len = per; best_cost = cost; }
  }
  *seg_len = best_len * chunk;
  if (cost_out) *cost_out = best_cost;
  return best;
}

static int lg_chunk(const LaArgs& a) { return a.Dk <= 128 && a.Dv <= 128 ? 64 : 32; }
static int lg_segments(const LaArgs& a, bool bwd, int* seg_len) {
  const int64_t ev = (a.Dv + LG_E - 1) / LG_E, ek = (a.Dk + LG_E - 1) / LG_E;
  return la_segments((int64_t)a.B * a.H * (bwd ? 2 * ek + ev : ev), a.L, lg_chunk(a), 1., 1., seg_len);
}

template <typename IO, int T>
static int lg_launch(const LaPlan& p, int local, cudaStream_t st) {
  int X = 0, E = 0;
  for (int i = 0; i < p.njobs; ++i) {
    X = p.job[i].X > X ? p.job[i].X : X;
    E = p.job[i].E > E ? p.job[i].E : E;
  }
  const int64_t smem = lg_floats(T, X) * 4, grid = (int64_t)p.B * p.H * p.nseg * ((E + LG_E - 1) / LG_E);
  ORBIT_REQUIRE(grid <= 0x7fffffffLL, ERR_UNSUPPORTED, "orbit_la: %lld (batch, head, segment) tiles are too many for one call", (long long)grid);
  ORBIT_CHECK_CUDA(cudaFuncSetAttribute(la_generic_kernel<IO, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  la_generic_kernel<IO, T><<<dim3((unsigned)grid, p.njobs), LG_THREADS, smem, st>>>(p, local);
  ORBIT_CHECK_LAUNCH("la_generic_kernel");
  return OK;
}

static int lg_run(const LaArgs& a, bool bwd, int dtype, cudaStream_t st) {
  int seg_len = 0, rc;
  const int nseg = lg_segments(a, bwd, &seg_len), T = lg_chunk(a);
  LaPlan p;
  for (int local = nseg > 1 ? 1 : 0; local >= 0; --local) {
    if ((rc = la_plan(a, bwd, nseg, seg_len, local != 0, &p)) != OK) return rc;
    if (dtype == BF16) rc = T == 64 ? lg_launch<__nv_bfloat16, 64>(p, local, st) : lg_launch<__nv_bfloat16, 32>(p, local, st);
    else rc = T == 64 ? lg_launch<float, 64>(p, local, st) : lg_launch<float, 32>(p, local, st);
    if (rc == OK && local) rc = la_join(p, st);
    if (rc != OK) return rc;
  }
  return OK;
}

static int la_check(const LaArgs* a, int dtype, const char* who) {
  ORBIT_REQUIRE(a != nullptr, ERR_BAD_ARG, "%s: null argument block", who);
  ORBIT_REQUIRE(dtype == BF16 || dtype == F32, ERR_BAD_ARG, "%s: unknown dtype code %d", who, dtype);
  ORBIT_REQUIRE(a->B >= 0 && a->L >= 0 && a->H > 0 && a->Dk > 0 && a->Dv > 0, ERR_BAD_ARG, "%s: bad sizes B=%d L=%d H=%d Dk=%d Dv=%d",
                who, a->B, a->L, a->H, a->Dk, a->Dv);
  ORBIT_REQUIRE(a->Dk <= 256 && a->Dv <= 256, ERR_UNSUPPORTED, "%s: head widths Dk=%d Dv=%d: the kernels serve 1..256", who, a->Dk, a->Dv);
  ORBIT_REQUIRE(a->L <= (1 << 30), ERR_UNSUPPORTED, "%s: sequences up to 2^30 tokens, got %d", who, a->L);
  ORBIT_REQUIRE(a->scale != 0.f && isfinite(a->scale), ERR_BAD_ARG, "%s: scale must be finite and not zero", who);
  return OK;
}

}  // namespace orbit

using namespace orbit;

extern "C" int64_t orbit_la_workspace_bytes(const orbit_la_args* a, int backward, int dtype) {
  if (a == nullptr || a->B <= 0 || a->L <= 0 || a->H <= 0) return 0;
  int seg_len = 0;
  const int nseg = la_tc_serves(*a, backward != 0, dtype) ? la_tc_segments(*a, backward != 0, &seg_len) : lg_segments(*a, backward != 0, &seg_len);
  return nseg > 1 ? (int64_t)a->B * a->H * nseg * a->Dk * a->Dv * 4 * (backward ? 2 : 1) : 0;
}

static int la_run(const orbit_la_args* a, bool bwd, int dtype, void* stream, const char* who) {
  const int64_t need = orbit_la_workspace_bytes(a, bwd, dtype);
  ORBIT_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need && aligned16(a->workspace)), ERR_WORKSPACE,
                "%s: a 16-byte aligned workspace of %lld bytes is needed", who, (long long)need);
  return la_tc_serves(*a, bwd, dtype) ? la_tc_launch(*a, bwd, (cudaStream_t)stream) : lg_run(*a, bwd, dtype, (cudaStream_t)stream);
}

extern "C" int orbit_la_fwd(const orbit_la_args* a, int dtype, void* stream) {
  int rc = la_check(a, dtype, "orbit_la_fwd");
  if (rc != OK) return rc;
  const int64_t n = (int64_t)a->B * a->H * a->Dk * a->Dv;
  if (a->B == 0) return OK;
  if (a->L == 0) {                                      // no token: the state goes through
    if (a->state1 && a->state0) ORBIT_CHECK_CUDA(cudaMemcpyAsync(a->state1, a->state0, n * 4, cudaMemcpyDeviceToDevice, (cudaStream_t)stream));
    else if (a->state1) ORBIT_CHECK_CUDA(cudaMemsetAsync(a->state1, 0, n * 4, (cudaStream_t)stream));
    return OK;
  }
  ORBIT_REQUIRE(a->q && a->k && a->v && a->y && a->log_decay, ERR_BAD_ARG, "orbit_la_fwd: null q/k/v/y/log_decay");
  // One token with a state on either side is the decode step (16 heads of 128 x 128: 9 us a call against 14 of a tile with one
  // row).
  if (a->L == 1 && a->state0 && a->state1 && (a->H == 1 || a->y_hs == a->Dv) && (a->B == 1 || a->y_bs == (int64_t)a->H * a->Dv))
    return orbit_la_step(a->q, a->q_bs, a->q_hs, a->k, a->k_bs, a->k_hs, a->v, a->v_bs, a->v_hs, a->log_decay, a->state0, a->state1, a->y,
                         a->B, a->H, a->Dk, a->Dv, a->scale, dtype, stream);
  return la_run(a, false, dtype, stream, "orbit_la_fwd");
}

extern "C" int orbit_la_bwd(const orbit_la_args* a, int dtype, void* stream) {
  int rc = la_check(a, dtype, "orbit_la_bwd");
  if (rc != OK) return rc;
  const int64_t n = (int64_t)a->B * a->H * a->Dk * a->Dv;
  if (a->B == 0) return OK;
  if (a->L == 0) {
    if (a->dstate0 && a->dstate1) ORBIT_CHECK_CUDA(cudaMemcpyAsync(a->dstate0, a->dstate1, n * 4, cudaMemcpyDeviceToDevice, (cudaStream_t)stream));
    else if (a->dstate0) ORBIT_CHECK_CUDA(cudaMemsetAsync(a->dstate0, 0, n * 4, (cudaStream_t)stream));
    return OK;
  }
  ORBIT_REQUIRE(a->q && a->k && a->v && a->dy && a->dq && a->dk && a->dv && a->log_decay, ERR_BAD_ARG,
                "orbit_la_bwd: null q/k/v/dy/dq/dk/dv/log_decay");
  return la_run(a, true, dtype, stream, "orbit_la_bwd");
}
