// The norms around a block in one pass: post-norm, gate, residual scale, residual add, pre-norm of what follows.
//
//   u = h rstd_h w_post      rstd_h = rsqrt(mean(h^2) + eps)          (u = h without a post-norm)
//   m = u sigmoid(g)                                                  (m = u without a gate)
//   r = x + s m                                                       (s = 1 without a scale)
//   n = r rstd_r w_pre       rstd_r = rsqrt(mean(r^2) + eps)          (not formed without a pre-norm)
//
// n is formed from the unrounded r, and everything is held in float32 between the loads and the two stores.  Separate norm,
// gate, add and norm kernels would read or write a row ten times; this reads x, h, g and writes r, n: five.
//
// Backward, from x, h, g, the two rstd and the gradients of r and n (r itself is formed again, unrounded), j = s m:
//   dr' = dr + rstd_r (w_pre dn - rh c1),       rh = r rstd_r,  c1 = mean(w_pre dn rh)
//   dx  = dr'
//   dg  = s dr' u sigmoid'(g)
//   t   = w_post s dr' sigmoid(g),   dh = rstd_h (t - hh c2),   hh = h rstd_h,  c2 = mean(t hh) = mean(dr' j)
// c2 depends on dr' and so on c1, but its sum splits into two that do not:
//   sum(dr' j) = sum((dr + rstd_r w_pre dn) j) - rstd_r c1 sum(rh j)
// so that ONE barrier serves all three row sums.  Column sums: with a = dr' sigmoid(g) hh, ds = w_post sum(a), dw_post =
// s sum(a), dw_pre = sum(dn rh): two accumulators a column in registers over the rows of a CTA, then fixed-order partial sums
// (no atomics: reproducible).
//
// HBM-bound: forward (2 + gate) reads and 2 writes of es bytes an element, backward (4 + gate) reads and (2 + gate) writes.
// Measured at [65536, 2048] with every factor: bfloat16 forward 227 us (5.9 TB/s, 90 % of the copy bandwidth), backward 419 us
// (5.1 TB/s, 78 %: one barrier a row at two CTAs of 256 threads an SM, registers allow no third); float32 497 us (5.4 TB/s) and 716
// (6.0 TB/s).
#include "common.cuh"
#include "../../include/orbit_b200.h"

namespace orbit {

constexpr int BN_THREADS = 256;                              // of the scalar kernels
__host__ __device__ constexpr int bn_threads(int tpr) { return tpr > 256 ? tpr : 256; }   // a CTA: one wide row, or several narrow ones

struct BnArgs {
  const void *x, *h, *g;
  int64_t xrs, hrs, grs;
  const float *scale, *wpost, *wpre;
  void *r, *n;
  float *rstd_h, *rstd_r;
  const void *dr, *dn;
  void *dx, *dh, *dg;
  float* part;
  int64_t M;
  int D;
  float eps;
};

// float32 sigmoids: the column sums they enter are float32 results (the single-MUFU tanh form is good to 2^-11 only)
__device__ __forceinline__ float bn_sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }
// __fdividef returns 0 for a divisor above 2^126, which is the sigmoid's value there to float32's last digit

// Sums of K values over the TPR threads of a row, by TPR consecutive threads; every thread of the row gets them.  `red`
// holds K values for each warp of the CTA; callers alternate two buffers so that one barrier a call is enough.
template <int TPR, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float (*red)[bn_threads(TPR) / 32]) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  if constexpr (TPR > 32) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) red[k][wid] = v[k];
    }
    __syncthreads();
    const int w0 = (threadIdx.x / TPR) * (TPR / 32);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float t = red[k][w0];
#pragma unroll
      for (int w = 1; w < TPR / 32; ++w) t += red[k][w0 + w];
      v[k] = t;
    }
  }
}


// The weights of this thread's columns, kept in registers over the rows of a CTA: js = scale w_post and w_pre.  (Read for every
// row they were the kernel's bound: eight floats a lane, 32 bytes apart, are eight wavefronts a load.)
template <int V, int TPR, int NV>
__device__ __forceinline__ void load_weights(const BnArgs& a, int lt, float (&js)[NV][V], float (&wp)[NV][V]) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * TPR + lt) * V;
    if (c < a.D) {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 one = make_float4(1.f, 1.f, 1.f, 1.f);
        const float4 u = a.scale ? *reinterpret_cast<const float4*>(a.scale + c + i) : one;
        const float4 w = a.wpost ? *reinterpret_cast<const float4*>(a.wpost + c + i) : one;
        const float4 p = a.wpre ? *reinterpret_cast<const float4*>(a.wpre + c + i) : one;
        js[k][i] = u.x * w.x; js[k][i + 1] = u.y * w.y; js[k][i + 2] = u.z * w.z; js[k][i + 3] = u.w * w.w;
        wp[k][i] = p.x; wp[k][i + 1] = p.y; wp[k][i + 2] = p.z; wp[k][i + 3] = p.w;
      }
    }
  }
}

// Forward.  TPR threads a row, NV 16-byte vectors a thread and tensor, 256 / TPR rows at a time; a CTA walks row groups
// blockIdx.x, blockIdx.x + gridDim.x, ..., the loads of the next one in flight over the sums and stores of the current one.
template <typename T, int TPR, int NV, bool GATE>
__global__ void __launch_bounds__(bn_threads(TPR), NV > 1 || TPR > 256 ? 1 : 3) block_norm_fwd_kernel(const BnArgs a) {
  constexpr int V = Vec16<T>::N, ROWS = bn_threads(TPR) / TPR;
  __shared__ float red[4][1][bn_threads(TPR) / 32];               // two sums a row group, two groups
  const int lt = threadIdx.x % TPR, sub = threadIdx.x / TPR, D = a.D;
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + sub;
  Vec16<T> nx[NV], nh[NV], ng[GATE ? NV : 1];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + lt) * V;
      if (r < a.M && c < D) {
        nh[k].load((const T*)a.h + r * a.hrs + c);
        if (GATE) ng[GATE ? k : 0].load((const T*)a.g + r * a.grs + c);
        nx[k].load((const T*)a.x + r * a.xrs + c);
      }
    }
  };
  fetch(row);
  float js[NV][V], wp[NV][V];
  load_weights<V, TPR, NV>(a, lt, js, wp);
  const float invD = 1.f / (float)D;
  int par = 0;
#pragma unroll 1
  for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < a.M; row0 += stride, row += stride, par ^= 2) {
    const bool live = row < a.M;
    float m[NV][V], r[NV][V], ss[1] = {0.f}, s2[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (live && (k * TPR + lt) * V < D) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float hv = nh[k].get(i);
          ss[0] = fmaf(hv, hv, ss[0]);
          m[k][i] = hv * js[k][i];
          if (GATE) m[k][i] *= bn_sigmoid(ng[GATE ? k : 0].get(i));
          r[k][i] = nx[k].get(i);
        }
      }
    }
    fetch(row + stride);
    float rs_h = 1.f;
    if (a.wpost) {
      row_sum<TPR, 1>(ss, red[par]);
      rs_h = rsqrtf(fmaf(ss[0], invD, a.eps));
      if (live && lt == 0 && a.rstd_h) a.rstd_h[row] = rs_h;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + lt) * V;
      if (live && c < D) {
        Vec16<T> o;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          r[k][i] = fmaf(rs_h, m[k][i], r[k][i]);
          s2[0] = fmaf(r[k][i], r[k][i], s2[0]);
          o.set(i, r[k][i]);
        }
        o.store((T*)a.r + row * (int64_t)D + c);
      }
    }
    if (!a.wpre) continue;
    row_sum<TPR, 1>(s2, red[par + 1]);
    const float rs_r = rsqrtf(fmaf(s2[0], invD, a.eps));
    if (live && lt == 0 && a.rstd_r) a.rstd_r[row] = rs_r;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + lt) * V;
      if (live && c < D) {
        Vec16<T> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.set(i, r[k][i] * rs_r * wp[k][i]);
        o.store((T*)a.n + row * (int64_t)D + c);
      }
    }
  }
}

// Backward.  A CTA walks row groups blockIdx.x, blockIdx.x + gridDim.x, ...; the next group's loads are issued before the
// barrier of the current one.
template <typename T, int TPR, int NV, bool GATE>
__global__ void __launch_bounds__(bn_threads(TPR), NV > 1 || TPR > 256 ? 1 : 2) block_norm_bwd_kernel(const BnArgs a) {
  constexpr int V = Vec16<T>::N, ROWS = bn_threads(TPR) / TPR;
  __shared__ float red[2][3][bn_threads(TPR) / 32];
  __shared__ float cols[ROWS > 1 ? 2 * ROWS * TPR * V : 1];  // column sums of the CTA's row groups (narrow rows)
  const int lt = threadIdx.x % TPR, D = a.D;
  const float invD = 1.f / (float)D;
  float acc_a[NV][V], acc_p[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) acc_a[k][i] = acc_p[k][i] = 0.f;
  Vec16<T> rx[NV], rh[NV], rg[GATE ? NV : 1], rdr[NV], rdn[NV];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + lt) * V;
      if (row < a.M && c < D) {
        rx[k].load((const T*)a.x + row * a.xrs + c);
        rh[k].load((const T*)a.h + row * a.hrs + c);
        if (GATE) rg[GATE ? k : 0].load((const T*)a.g + row * a.grs + c);
        if (a.dr) rdr[k].load((const T*)a.dr + row * (int64_t)D + c);
        if (a.dn) rdn[k].load((const T*)a.dn + row * (int64_t)D + c);
      }
    }
  };
  const int64_t first = (int64_t)blockIdx.x * ROWS, stride = (int64_t)gridDim.x * ROWS;
  const int sub = threadIdx.x / TPR;
  int par = 0;
  if (first < a.M) fetch(first + sub);
  float js[NV][V], wp[NV][V];
  load_weights<V, TPR, NV>(a, lt, js, wp);
  for (int64_t row0 = first; row0 < a.M; row0 += stride, par ^= 1) {
    const int64_t row = row0 + sub;
    const bool live = row < a.M;
    const float rs_h = a.wpost && live ? a.rstd_h[row] : 1.f, rs_r = a.dn && live ? a.rstd_r[row] : 1.f;
    // what survives the barrier: the gradient of r before the norm's projection, r / rms, h / rms and sigmoid(g)
    float e[NV][V], q[NV][V], hh[NV][V], sg[GATE ? NV : 1][V];
    float sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + lt) * V;
      if (live && c < D) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          hh[k][i] = rh[k].get(i) * rs_h;
          float j = hh[k][i] * js[k][i];
          if (GATE) {
            sg[GATE ? k : 0][i] = bn_sigmoid(rg[GATE ? k : 0].get(i));
            j *= sg[GATE ? k : 0][i];
          }
          e[k][i] = a.dr ? rdr[k].get(i) : 0.f;
          q[k][i] = 0.f;
          if (a.dn) {
            q[k][i] = (rx[k].get(i) + j) * rs_r;
            const float dn = rdn[k].get(i), w = dn * wp[k][i];
            acc_p[k][i] = fmaf(dn, q[k][i], acc_p[k][i]);
            sum[0] = fmaf(w, q[k][i], sum[0]);
            sum[2] = fmaf(q[k][i], j, sum[2]);
            e[k][i] = fmaf(rs_r, w, e[k][i]);
          }
          sum[1] = fmaf(e[k][i], j, sum[1]);
        }
      }
    }
    if (row0 + stride < a.M) fetch(row + stride);
    row_sum<TPR, 3>(sum, red[par]);
    const float c1 = sum[0] * invD * rs_r, c2 = (sum[1] - c1 * sum[2]) * invD;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + lt) * V;
      if (live && c < D) {
        Vec16<T> ox, oh, og;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = fmaf(-c1, q[k][i], e[k][i]);
          const float sig = GATE ? sg[GATE ? k : 0][i] : 1.f;
          const float t = d * sig;                               // gradient of r through the gate
          acc_a[k][i] = fmaf(t, hh[k][i], acc_a[k][i]);
          ox.set(i, d);
          const float dm = t * js[k][i];
          if (GATE) og.set(i, dm * hh[k][i] * (1.f - sig));
          oh.set(i, a.wpost ? rs_h * (dm - hh[k][i] * c2) : dm);
        }
        ox.store((T*)a.dx + row * (int64_t)D + c);
        oh.store((T*)a.dh + row * (int64_t)D + c);
        if (GATE) og.store((T*)a.dg + row * (int64_t)D + c);
      }
    }
  }
  // partial column sums [slot][2][D], a slot for each CTA; its row groups are added in order
  if (a.part == nullptr) return;
  float* part = a.part + (int64_t)blockIdx.x * 2 * D;
  if constexpr (ROWS > 1) {
    static_assert(NV == 1, "several rows a CTA hold one vector a thread");
#pragma unroll
    for (int i = 0; i < V; ++i) {
      cols[(sub * 2) * TPR * V + lt * V + i] = acc_a[0][i];
      cols[(sub * 2 + 1) * TPR * V + lt * V + i] = acc_p[0][i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * D; c += bn_threads(TPR)) {
      const int which = c >= D, col = c - which * D;
      float t = 0.f;
      for (int r = 0; r < ROWS; ++r) t += cols[(r * 2 + which) * TPR * V + col];
      part[c] = t;
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + lt) * V;
      if (c < D) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          part[c + i] = acc_a[k][i];
          part[D + c + i] = acc_p[k][i];
        }
      }
    }
  }
}

// Rows that 16-byte vectors do not divide, or wider than the registers hold: one CTA a row, element by element, the row read
// again for each sum.  bfloat16 [65536, 1001] forward 600 us and backward 1353 (rows of 1000: 117 and 249), [16384, 9000] 990 us and
// 2960; float32 669 and 1502, 1305 and 4119.
template <typename T>
__global__ void __launch_bounds__(BN_THREADS) block_norm_fwd_scalar_kernel(const BnArgs a) {
  __shared__ float red[32];
  const int D = a.D;
  const T *x = (const T*)a.x, *h = (const T*)a.h, *g = (const T*)a.g;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    float rs_h = 1.f;
    if (a.wpost) {
      float ss = 0.f;
      for (int c = threadIdx.x; c < D; c += BN_THREADS) {
        const float v = ldf(h + row * a.hrs + c);
        ss = fmaf(v, v, ss);
      }
      rs_h = rsqrtf(block_sum(ss, red) / (float)D + a.eps);
      if (threadIdx.x == 0 && a.rstd_h) a.rstd_h[row] = rs_h;
    }
    auto value = [&](int c) {
      float m = ldf(h + row * a.hrs + c);
      if (a.wpost) m = m * rs_h * a.wpost[c];
      if (g) m *= bn_sigmoid(ldf(g + row * a.grs + c));
      return fmaf(a.scale ? a.scale[c] : 1.f, m, ldf(x + row * a.xrs + c));
    };
    float s2 = 0.f;
    for (int c = threadIdx.x; c < D; c += BN_THREADS) {
      const float r = value(c);
      stf((T*)a.r + row * (int64_t)D + c, r);
      s2 = fmaf(r, r, s2);
    }
    if (a.wpre) {
      const float rs_r = rsqrtf(block_sum(s2, red) / (float)D + a.eps);
      if (threadIdx.x == 0 && a.rstd_r) a.rstd_r[row] = rs_r;
      for (int c = threadIdx.x; c < D; c += BN_THREADS) stf((T*)a.n + row * (int64_t)D + c, value(c) * rs_r * a.wpre[c]);
    }
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(BN_THREADS) block_norm_bwd_scalar_kernel(const BnArgs a) {
  __shared__ float red[32];
  const int D = a.D;
  const T *x = (const T*)a.x, *h = (const T*)a.h, *g = (const T*)a.g, *dr = (const T*)a.dr, *dn = (const T*)a.dn;
  bool first = true;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const float rs_h = a.wpost ? a.rstd_h[row] : 1.f, rs_r = dn ? a.rstd_r[row] : 1.f;
    struct At { float hh, sig, j, q, w, e, dn; };
    auto at = [&](int c) {
      At o;
      o.hh = ldf(h + row * a.hrs + c) * rs_h;
      o.sig = g ? bn_sigmoid(ldf(g + row * a.grs + c)) : 1.f;
      o.j = o.hh * (a.scale ? a.scale[c] : 1.f) * (a.wpost ? a.wpost[c] : 1.f) * o.sig;
      o.e = dr ? ldf(dr + row * (int64_t)D + c) : 0.f;
      o.q = o.w = o.dn = 0.f;
      if (dn) {
        o.q = (ldf(x + row * a.xrs + c) + o.j) * rs_r;
        o.dn = ldf(dn + row * (int64_t)D + c);
        o.w = o.dn * a.wpre[c];
        o.e = fmaf(rs_r, o.w, o.e);
      }
      return o;
    };
    float s0 = 0.f, s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < D; c += BN_THREADS) {
      const At o = at(c);
      s0 = fmaf(o.w, o.q, s0);
      s1 = fmaf(o.e, o.j, s1);
      s2 = fmaf(o.q, o.j, s2);
    }
    const float c1 = block_sum(s0, red) / (float)D * rs_r;
    const float b1 = block_sum(s1, red);
    const float c2 = (b1 - c1 * block_sum(s2, red)) / (float)D;
    for (int c = threadIdx.x; c < D; c += BN_THREADS) {
      const At o = at(c);
      const float d = fmaf(-c1, o.q, o.e), t = d * o.sig;
      const float dm = t * (a.scale ? a.scale[c] : 1.f) * (a.wpost ? a.wpost[c] : 1.f);
      stf((T*)a.dx + row * (int64_t)D + c, d);
      stf((T*)a.dh + row * (int64_t)D + c, a.wpost ? rs_h * (dm - o.hh * c2) : dm);
      if (g) stf((T*)a.dg + row * (int64_t)D + c, dm * o.hh * (1.f - o.sig));
      if (a.part) {
        float* p = a.part + (int64_t)blockIdx.x * 2 * D + c;     // this thread's own columns: no other thread touches them
        p[0] = (first ? 0.f : p[0]) + t * o.hh;
        p[D] = (first ? 0.f : p[D]) + o.dn * o.q;
      }
    }
    first = false;
    __syncthreads();
  }
}

// Column sums over the partial slots in a fixed order (a CTA owns 32 columns; warp w sums the slots congruent to w modulo 8,
// then the eight sums are added in order), handed out as dscale = w_post sum(a), dw_post = scale sum(a), dw_pre.
__global__ void __launch_bounds__(256) block_norm_colsum_kernel(const float* __restrict__ part, int64_t nslots, int D,
                                                                const float* __restrict__ scale, const float* __restrict__ wpost,
                                                                float* __restrict__ dscale, float* __restrict__ dwpost,
                                                                float* __restrict__ dwpre) {
  __shared__ float red[8][33];
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, which = blockIdx.y;
  float acc = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int64_t s = grp; s < nslots; s += 8) acc += part[(s * 2 + which) * D + c];
  }
  red[grp][lane] = acc;
  __syncthreads();
  if (grp != 0 || c >= D) return;
  float v = red[0][lane];
#pragma unroll
  for (int g = 1; g < 8; ++g) v += red[g][lane];
  if (which == 0) {
    if (dscale) dscale[c] = v * (wpost ? wpost[c] : 1.f);
    if (dwpost) dwpost[c] = v * (scale ? scale[c] : 1.f);
  } else if (dwpre) {
    dwpre[c] = v;
  }
}

// 16-byte vectors a row takes -> threads a row and vectors a thread (0: the scalar kernels).  A row keeps to one warp up to 32
// vectors and spreads over up to 512 threads, one vector of each tensor a thread (72 registers forward, 125 to 128 backward), so that
// many rows are in flight.  Rows of 513 to 1024 vectors take four a thread: 217 registers forward ([16384, 8192] bfloat16 with every
// factor: 229 us, 5.9 TB/s), 255 backward with 2312 bytes of spill stores and 1424 of loads, which bound it (1710 us, 1.3 TB/s; [16384, 5120] 175 and 1050 us).
struct BnShape { int tpr, nv; };
static BnShape bn_shape(int vectors) {
  if (vectors <= 32) return {32, 1};
  if (vectors <= 64) return {64, 1};
  if (vectors <= 128) return {128, 1};
  if (vectors <= 256) return {256, 1};
  if (vectors <= 512) return {512, 1};
  if (vectors <= 1024) return {256, 4};
  return {0, 0};
}

template <typename T>
static bool bn_vectors(const BnArgs& a, bool bwd, BnShape* s) {
  constexpr int V = Vec16<T>::N;
  bool ok = a.D % V == 0 && a.xrs % V == 0 && a.hrs % V == 0 && (!a.g || a.grs % V == 0) && aligned16(a.x) && aligned16(a.h) &&
            aligned16(a.g) && aligned16(a.scale) && aligned16(a.wpost) && aligned16(a.wpre);
  if (bwd) ok = ok && aligned16(a.dr) && aligned16(a.dn) && aligned16(a.dx) && aligned16(a.dh) && aligned16(a.dg);
  else ok = ok && aligned16(a.r) && aligned16(a.n);
  *s = bn_shape((a.D + V - 1) / V);
  return ok && s->tpr > 0;
}

// CTAs that walk in the backward pass: two to an SM; every slot is written in full before it is read.
constexpr int BN_SLOTS = 148 * 2;
static int64_t bn_slots(int64_t M) { return M < BN_SLOTS ? (M > 0 ? M : 1) : BN_SLOTS; }

#define BN_DISPATCH(KERNEL, GRID)                                                              \
  do {                                                                                         \
    const int key = s.tpr * 8 + s.nv;                                                          \
    const unsigned grid = (unsigned)(GRID);                                                    \
    if (a.g) {                                                                                 \
      if (key == 32 * 8 + 1) KERNEL<T, 32, 1, true><<<grid, bn_threads(32), 0, st>>>(a);           \
      else if (key == 64 * 8 + 1) KERNEL<T, 64, 1, true><<<grid, bn_threads(64), 0, st>>>(a);      \
      else if (key == 128 * 8 + 1) KERNEL<T, 128, 1, true><<<grid, bn_threads(128), 0, st>>>(a);    \
      else if (key == 256 * 8 + 1) KERNEL<T, 256, 1, true><<<grid, bn_threads(256), 0, st>>>(a);    \
      else if (key == 512 * 8 + 1) KERNEL<T, 512, 1, true><<<grid, bn_threads(512), 0, st>>>(a);    \
      else KERNEL<T, 256, 4, true><<<grid, bn_threads(256), 0, st>>>(a);                            \
    } else {                                                                                   \
      if (key == 32 * 8 + 1) KERNEL<T, 32, 1, false><<<grid, bn_threads(32), 0, st>>>(a);          \
      else if (key == 64 * 8 + 1) KERNEL<T, 64, 1, false><<<grid, bn_threads(64), 0, st>>>(a);     \
      else if (key == 128 * 8 + 1) KERNEL<T, 128, 1, false><<<grid, bn_threads(128), 0, st>>>(a);   \
      else if (key == 256 * 8 + 1) KERNEL<T, 256, 1, false><<<grid, bn_threads(256), 0, st>>>(a);   \
      else if (key == 512 * 8 + 1) KERNEL<T, 512, 1, false><<<grid, bn_threads(512), 0, st>>>(a);   \
      else KERNEL<T, 256, 4, false><<<grid, bn_threads(256), 0, st>>>(a);                           \
    }                                                                                          \
  } while (0)

template <typename T>
static int block_norm_fwd_t(const BnArgs& a, cudaStream_t st) {
  BnShape s;
  if (bn_vectors<T>(a, false, &s)) {
    const int rows = bn_threads(s.tpr) / s.tpr;
    const int64_t groups = (a.M + rows - 1) / rows, most = s.nv > 1 || s.tpr > 256 ? 148 : 148 * 3;   // what the SMs hold at once
    const int64_t blocks = groups < most ? groups : most;
    BN_DISPATCH(block_norm_fwd_kernel, blocks);
    ORBIT_CHECK_LAUNCH("block_norm_fwd_kernel");
    return OK;
  }
  block_norm_fwd_scalar_kernel<T><<<(unsigned)(a.M < 148 * 8 ? a.M : 148 * 8), BN_THREADS, 0, st>>>(a);
  ORBIT_CHECK_LAUNCH("block_norm_fwd_scalar_kernel");
  return OK;
}

template <typename T>
static int block_norm_bwd_t(const BnArgs& a, float* dscale, float* dwpost, float* dwpre, cudaStream_t st) {
  BnShape s;
  int64_t slots;
  if (bn_vectors<T>(a, true, &s)) {
    const int rows = bn_threads(s.tpr) / s.tpr;
    slots = bn_slots((a.M + rows - 1) / rows);
    BN_DISPATCH(block_norm_bwd_kernel, slots);
    ORBIT_CHECK_LAUNCH("block_norm_bwd_kernel");
  } else {
    slots = bn_slots(a.M);
    block_norm_bwd_scalar_kernel<T><<<(unsigned)slots, BN_THREADS, 0, st>>>(a);
    ORBIT_CHECK_LAUNCH("block_norm_bwd_scalar_kernel");
  }
  if (a.part) {
    block_norm_colsum_kernel<<<dim3((a.D + 31) / 32, 2), 256, 0, st>>>(a.part, slots, a.D, a.scale, a.wpost, dscale, dwpost, dwpre);
    ORBIT_CHECK_LAUNCH("block_norm_colsum_kernel");
  }
  return OK;
}

}  // namespace orbit

using namespace orbit;

extern "C" int orbit_block_norm_fwd(const void* x, int64_t x_row_stride, const void* h, int64_t h_row_stride, const void* gate,
                                    int64_t gate_row_stride, const float* scale, const float* w_post, const float* w_pre,
                                    void* r, void* n, float* rstd_h, float* rstd_r, int64_t M, int D, float eps, int dtype,
                                    void* stream) {
  ORBIT_REQUIRE(M >= 0 && D > 0, ERR_BAD_ARG, "orbit_block_norm_fwd: bad sizes M=%lld D=%d", (long long)M, D);
  ORBIT_REQUIRE(dtype == BF16 || dtype == F32, ERR_BAD_ARG, "orbit_block_norm_fwd: unknown dtype code %d", dtype);
  if (M == 0) return OK;
  ORBIT_REQUIRE(x && h && r, ERR_BAD_ARG, "orbit_block_norm_fwd: null x/h/r");
  ORBIT_REQUIRE(w_pre == nullptr || n != nullptr, ERR_BAD_ARG, "orbit_block_norm_fwd: n is required with a pre-norm");
  BnArgs a = {};
  a.x = x; a.h = h; a.g = gate; a.xrs = x_row_stride; a.hrs = h_row_stride; a.grs = gate_row_stride;
  a.scale = scale; a.wpost = w_post; a.wpre = w_pre; a.r = r; a.n = n; a.rstd_h = rstd_h; a.rstd_r = rstd_r;
  a.M = M; a.D = D; a.eps = eps;
  return dtype == BF16 ? block_norm_fwd_t<__nv_bfloat16>(a, (cudaStream_t)stream) : block_norm_fwd_t<float>(a, (cudaStream_t)stream);
}

extern "C" int64_t orbit_block_norm_bwd_workspace_bytes(int64_t M, int D) {
  return bn_slots(M) * 2 * D * (int64_t)sizeof(float);
}

extern "C" int orbit_block_norm_bwd(const void* x, int64_t x_row_stride, const void* h, int64_t h_row_stride, const void* gate,
                                    int64_t gate_row_stride, const float* scale, const float* w_post, const float* w_pre,
                                    const float* rstd_h, const float* rstd_r, const void* dr, const void* dn, void* dx, void* dh,
                                    void* dgate, float* dscale, float* dw_post, float* dw_pre, void* workspace,
                                    int64_t workspace_bytes, int64_t M, int D, int dtype, void* stream) {
  ORBIT_REQUIRE(M >= 0 && D > 0, ERR_BAD_ARG, "orbit_block_norm_bwd: bad sizes M=%lld D=%d", (long long)M, D);
  ORBIT_REQUIRE(dtype == BF16 || dtype == F32, ERR_BAD_ARG, "orbit_block_norm_bwd: unknown dtype code %d", dtype);
  cudaStream_t st = (cudaStream_t)stream;
  const bool sums = dscale || dw_post || dw_pre;
  if (M == 0) {
    if (dscale) ORBIT_CHECK_CUDA(cudaMemsetAsync(dscale, 0, sizeof(float) * D, st));
    if (dw_post) ORBIT_CHECK_CUDA(cudaMemsetAsync(dw_post, 0, sizeof(float) * D, st));
    if (dw_pre) ORBIT_CHECK_CUDA(cudaMemsetAsync(dw_pre, 0, sizeof(float) * D, st));
    return OK;
  }
  ORBIT_REQUIRE(x && h && dx && dh && (dr || dn), ERR_BAD_ARG, "orbit_block_norm_bwd: null x/h/dx/dh, or no gradient at all");
  ORBIT_REQUIRE(gate == nullptr || dgate != nullptr, ERR_BAD_ARG, "orbit_block_norm_bwd: dgate is required with a gate");
  ORBIT_REQUIRE(w_post == nullptr || rstd_h != nullptr, ERR_BAD_ARG, "orbit_block_norm_bwd: rstd_h is required with a post-norm");
  ORBIT_REQUIRE(dn == nullptr || (w_pre != nullptr && rstd_r != nullptr), ERR_BAD_ARG,
                "orbit_block_norm_bwd: a gradient of n needs w_pre and rstd_r");
  ORBIT_REQUIRE(!sums || (workspace && workspace_bytes >= orbit_block_norm_bwd_workspace_bytes(M, D)), ERR_WORKSPACE,
                "orbit_block_norm_bwd: workspace of %lld bytes needed", (long long)orbit_block_norm_bwd_workspace_bytes(M, D));
  BnArgs a = {};
  a.x = x; a.h = h; a.g = gate; a.xrs = x_row_stride; a.hrs = h_row_stride; a.grs = gate_row_stride;
  a.scale = scale; a.wpost = w_post; a.wpre = w_pre; a.rstd_h = const_cast<float*>(rstd_h); a.rstd_r = const_cast<float*>(rstd_r);
  a.dr = dr; a.dn = dn; a.dx = dx; a.dh = dh; a.dg = dgate; a.part = sums ? (float*)workspace : nullptr;
  a.M = M; a.D = D;
  return dtype == BF16 ? block_norm_bwd_t<__nv_bfloat16>(a, dscale, dw_post, dw_pre, st)
                       : block_norm_bwd_t<float>(a, dscale, dw_post, dw_pre, st);
}
