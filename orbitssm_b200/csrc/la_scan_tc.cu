// Linear attention with a constant decay for each head on tcgen05 tensor cores (bfloat16, head widths that are multiples of 8
// up to 128).  The recurrence, its four roles (y, dq, dk, dv) and the split into segments are those of la_scan.cu; here a chunk
// is 128 tokens and its products are tensor-core tiles with float32 accumulators in TMEM.
//
// One CTA owns (batch, head, segment, 64 channels of v') and walks the chunks of its segment:
//   S1[t,s] = q'_t . k'_s                    128 x 128 x X     both operands as TMA wrote them
//   P       = decay mask o S1 -> bfloat16                      the only rounding of the part inside the chunk
//   O [t,e] = P V'                           128 x 64 x 128    P read from TMEM
//   O2[t,e] = q'_t . Zb                      128 x 64 x X      Zb: the state rounded to bfloat16, the only rounding of that part
//   dZ[x,e] = sum_s k'_s[x] (f_s v'_s[e])    128 x 192 x 128   f_s v' in three bfloat16 parts (hi + mid + lo hold all 24 bits of
//                                                              the float32 product) side by side, so that the float32 state and
//                                                              the state's gradient lose nothing to the operands' type
//   out = s_out O + s_in a^{..} O2;   Z = a^T Z + dZ           Z in registers, float32
// Row factors are applied to the accumulators, not to the operands: scaling q' or k' first would round them once more.
//
// Warp-specialised, 18 warps that meet only through mbarriers (every wait bounded):
//   warps 0..3   decay mask: S1 -> P (TMEM to TMEM; the slabs beyond the diagonal are zero and written once)
//   warps 4..7   state: Z in registers (thread = state row), writes Zb, adds dZ
//   warps 8..11  scaled v': three bfloat16 tiles (thread = token)
//   warps 12..15 read-out: O, O2 -> output tile in the place of the v' tile -> TMA store
//   warp 16      one lane issues the TMA loads (two stages), warp 17 one lane issues the MMAs
// 64 channels a CTA (two CTAs for a 128-wide head, adjacent so that q' and k' come from L2 the second time): the state then
// leaves room in shared memory for two stages of operands, and short batches fill twice the SMs.
#include "common.cuh"
#include "la_args.h"
#include "tc_common.cuh"
#include "tc_scan_common.cuh"

namespace orbit {
using namespace tc;

constexpr int LT_T = 128, LT_E = 64, LT_THREADS = 576;
constexpr uint32_t LT_S1 = 0, LT_P = 128, LT_O = 192, LT_O2 = 256, LT_DZ = 320;   // TMEM columns (512 in all)
constexpr int LT_STAGE = 5;                                  // blocks of 16 KB: q' 2, k' 2, v' 1
constexpr int LT_SMEM = (2 * LT_STAGE + 3 + 1) * (int)BLK + 1024;

struct LaTcArgs {
  CUtensorMap map[3][4];                                     // q', k', v', output of each job
  LaPlan p;
};

struct LtBars {
  uint64_t qk_full[2], qk_empty[2], v_full[2], v_empty[2], s1_full, s1_empty, p_full, p_empty, vd_full, vd_empty, zb_full,
      zb_empty, dz_full, dz_empty, acc_full, acc_empty;
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* m, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* m, const void* src, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}
__device__ __forceinline__ float bf16_round(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }

__global__ void __launch_bounds__(LT_THREADS, 1) la_tc_kernel(const __grid_constant__ LaTcArgs a, const int local) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ LtBars bars;
  __shared__ float pw[LT_T + 1];                             // a^0 .. a^128
  __shared__ uint32_t tmem_slot;
  __shared__ int s_abort;
  const LaPlan& p = a.p;
  // tile index: e tile fastest, then job, segment, head, batch
  int64_t id = blockIdx.x;
  const int ne = p.ne;
  const int et = (int)(id % ne);
  id /= ne;
  const int jb = (int)(id % p.njobs);
  id /= p.njobs;
  const int seg = (int)(id % p.nseg);
  id /= p.nseg;
  const int h = (int)(id % p.H), b = (int)(id / p.H), e0 = et * LT_E;
  const LaJob& J = p.job[jb];
  const int rev = J.reverse, X = J.X, E = J.E;
  if (e0 >= E) return;
  if (local && seg == (rev ? 0 : p.nseg - 1)) return;        // nobody reads the last segment's share
  const CUtensorMap *mq = &a.map[jb][0], *mk = &a.map[jb][1], *mv = &a.map[jb][2], *my = &a.map[jb][3];

  uint8_t* sm = align1024(smem_raw);
  uint8_t* sVd = sm + 2 * LT_STAGE * BLK;                    // scaled v': hi, mid, lo
  uint8_t* sZb = sVd + 3 * BLK;                              // entering state, bfloat16 [128 x][64 e]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q = warp & 3, role = warp >> 2;
  const int s0 = seg * p.seg_len, s1 = min(p.L, s0 + p.seg_len), nch = (s1 - s0 + LT_T - 1) / LT_T;
  const double ld = (double)p.log_decay[h];

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.qk_full[i], 1);
      mbar_init(&bars.qk_empty[i], 1);
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.v_empty[i], 1);
    }
    mbar_init(&bars.s1_full, 1);
    mbar_init(&bars.s1_empty, 4);
    mbar_init(&bars.p_full, 4);
    mbar_init(&bars.p_empty, 1);
    mbar_init(&bars.vd_full, 4);
    mbar_init(&bars.vd_empty, 1);
    mbar_init(&bars.zb_full, 4);
    mbar_init(&bars.zb_empty, 1);
    mbar_init(&bars.dz_full, 1);
    mbar_init(&bars.dz_empty, 4);
    mbar_init(&bars.acc_full, 1);
    mbar_init(&bars.acc_empty, 4);
    mbar_fence_init();
    s_abort = 0;
  }
  if (tid <= LT_T) pw[tid] = tid == 0 ? 1.f : (float)exp(ld * tid);
  if (warp == 0) tmem_alloc(&tmem_slot, 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tbase = tmem_slot;
  volatile int* abort_flag = &s_abort;
  bool dead = false;
  auto chunk_start = [&](int c) { return s0 + (rev ? nch - 1 - c : c) * LT_T; };

  if (warp == 16) {
    if (lane == 0) {
      // ---- producer ----
      int done = 0;
#pragma unroll 1
      for (int c = 0; c < nch; ++c) {
        const int s = c & 1, t0 = chunk_start(c);
        uint8_t* st = sm + s * LT_STAGE * BLK;
        if (c >= 2 && !lane_wait(&bars.qk_empty[s], (uint32_t)(((c >> 1) - 1) & 1), abort_flag, dead)) break;
        const int blocks = X > 64 ? 2 : 1;                   // the second block of a narrow head is never contracted
        mbar_expect_tx(&bars.qk_full[s], (uint32_t)(local ? blocks : 2 * blocks) * BLK);
        for (int i = 0; i < blocks; ++i) {
          if (!local) tma_load_4d(st + i * BLK, mq, &bars.qk_full[s], i * 64, h, t0, b);
          tma_load_4d(st + (2 + i) * BLK, mk, &bars.qk_full[s], i * 64, h, t0, b);
        }
        done = 2 * c + 1;
        if (c >= 2 && !lane_wait(&bars.v_empty[s], (uint32_t)(((c >> 1) - 1) & 1), abort_flag, dead)) break;
        mbar_expect_tx(&bars.v_full[s], BLK);
        tma_load_4d(st + 4 * BLK, mv, &bars.v_full[s], e0, h, t0, b);
        done = 2 * c + 2;
      }
      if (dead) {                                            // wind-down: what was issued has to land before the CTA goes
        for (int k = max(0, done - 4); k < done; ++k)
          mbar_wait((k & 1) ? &bars.v_full[(k >> 1) & 1] : &bars.qk_full[(k >> 1) & 1], (uint32_t)((k >> 2) & 1));
      }
    }
    __syncwarp();
  } else if (warp == 17) {
    if (lane == 0) {
      // ---- MMA issuer ----
      const uint32_t id_s = idesc_bf16(128, 128, 0, 0), id_o = idesc_bf16(128, 64, 0, 1), id_z = idesc_bf16(128, 192, 1, 1);
      const int kx = (X + 15) / 16;
      const uint32_t vd = lo_mn(smem_u32(sVd)), zb = lo_mn(smem_u32(sZb));
      auto base = [&](int c, int blk) { return smem_u32(sm + ((c & 1) * LT_STAGE + blk) * BLK); };
      auto scores = [&](int c) {
        const uint32_t aq = lo_k(base(c, 0)), bk = lo_k(base(c, 2));
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          if (ks < kx) umma_bf16_h(tbase + LT_S1, aq + inc_k(ks), bk + inc_k(ks), id_s, ks > 0 ? 1u : 0u);
        umma_commit(&bars.s1_full);
      };
      if (lane_wait(&bars.qk_full[0], 0, abort_flag, dead) && !local) {
        tc_fence_after_sync();
        scores(0);
      }
#pragma unroll 1
      for (int c = 0; c < nch && !dead; ++c) {
        const uint32_t ph = (uint32_t)(c & 1), prev = (uint32_t)((c - 1) & 1);
        if (local && c > 0 && !lane_wait(&bars.qk_full[c & 1], (uint32_t)((c >> 1) & 1), abort_flag, dead)) break;
        if (!local) {
          if (!lane_wait(&bars.zb_full, ph, abort_flag, dead)) break;
          if (c > 0 && !lane_wait(&bars.acc_empty, prev, abort_flag, dead)) break;
          tc_fence_after_sync();
          const uint32_t aq = lo_k(base(c, 0));
#pragma unroll
          for (int ks = 0; ks < 8; ++ks)
            if (ks < kx) umma_bf16_h(tbase + LT_O2, aq + inc_k(ks), zb + inc_mn(ks), id_o, ks > 0 ? 1u : 0u);
          umma_commit(&bars.zb_empty);
        }
        if (!lane_wait(&bars.vd_full, ph, abort_flag, dead)) break;
        if (c > 0 && !lane_wait(&bars.dz_empty, prev, abort_flag, dead)) break;
        tc_fence_after_sync();
        const uint32_t ak = lo_mn(base(c, 2));
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) umma_bf16_h(tbase + LT_DZ, ak + inc_mn(ks), vd + inc_mn(ks), id_z, ks > 0 ? 1u : 0u);
        umma_commit(&bars.dz_full);
        umma_commit(&bars.vd_empty);
        umma_commit(&bars.qk_empty[c & 1]);                  // q' and k' of this chunk have been read for the last time
        if (local) continue;
        if (c + 1 < nch) {
          if (!lane_wait(&bars.qk_full[(c + 1) & 1], (uint32_t)(((c + 1) >> 1) & 1), abort_flag, dead)) break;
          if (!lane_wait(&bars.s1_empty, ph, abort_flag, dead)) break;
          tc_fence_after_sync();
          scores(c + 1);
        }
        if (!lane_wait(&bars.p_full, ph, abort_flag, dead)) break;
        tc_fence_after_sync();
        const uint32_t bv = lo_mn(base(c, 4));
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          umma_bf16_ta_h(tbase + LT_O, tbase + LT_P + ks * 8, bv + inc_mn(ks), id_o, ks > 0 ? 1u : 0u);
        umma_commit(&bars.p_empty);
        umma_commit(&bars.acc_full);
      }
    }
    __syncwarp();
  } else if (role == 0) {
    if (!local) {
      // ---- decay mask: thread = row t; slab j holds columns 32 j .. 32 j + 31 ----
      {
        uint32_t z[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (rev ? j < q : j > q) tmem_st16(tmem_addr(tbase, q * 32, LT_P + j * 16), z);
        tmem_st_wait();
      }
#pragma unroll 1
      for (int c = 0; c < nch; ++c) {
        bool ok = role_wait(&bars.s1_full, (uint32_t)(c & 1), abort_flag, dead);
        if (c > 0) ok = role_wait(&bars.p_empty, (uint32_t)((c - 1) & 1), abort_flag, dead) && ok;
        if (ok) {
          tc_fence_after_sync();
#pragma unroll 1
          for (int j = rev ? q : 0; j <= (rev ? 3 : q); ++j) {
            uint32_t r[32], o[16];
            tmem_ld32(tmem_addr(tbase, q * 32, LT_S1 + j * 32), r);
            tmem_ld_wait();
            if (j == q) {
              // a^{t-s} on and below the diagonal (reverse: a^{s-t} on and above it); zero beyond, whatever the score
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int d0 = rev ? 2 * i - lane : lane - 2 * i, d1 = rev ? 2 * i + 1 - lane : lane - 2 * i - 1;
                const float f0 = pw[max(d0, 0)], f1 = pw[max(d1, 0)];
                o[i] = pack_bf16(d0 >= 0 ? __uint_as_float(r[2 * i]) * f0 : 0.f, d1 >= 0 ? __uint_as_float(r[2 * i + 1]) * f1 : 0.f);
              }
            } else {
              // a whole slab away the factor splits at the slab's near end: both parts are powers of a that are at least one
              // factor each, so neither grows beyond 1
              const float rf = pw[rev ? 32 * (j - q) - lane : 32 * (q - j) + lane - 31];
              const float2 rf2 = make_float2(rf, rf);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float2 cf = rev ? make_float2(pw[2 * i], pw[2 * i + 1]) : make_float2(pw[31 - 2 * i], pw[30 - 2 * i]);
                const float2 v = mul2(f2(r[2 * i], r[2 * i + 1]), mul2(rf2, cf));
                o[i] = pack_bf16(v.x, v.y);
              }
            }
            tmem_st16(tmem_addr(tbase, q * 32, LT_P + j * 16), o);
          }
          tmem_st_wait();
        }
        warp_arrive(&bars.s1_empty, false);
        if (lane == 0) mbar_arrive(&bars.p_full);
      }
    }
  } else if (role == 1) {
    // ---- state: thread = state row x, its 64 channels in registers ----
    const int x = q * 32 + lane;
    const int64_t head = (int64_t)b * p.H + h;
    float z[LT_E];
#pragma unroll
    for (int e = 0; e < LT_E; ++e) z[e] = 0.f;
    const bool live = x < X;
    if (!local && live) {
      // the carried state and the shares of the segments before this one, each with its decay since
      const int64_t off = x * J.xs + e0 * J.es;
      if (J.z0) {
        const float* src = J.z0 + head * p.S + off;
#pragma unroll
        for (int e = 0; e < LT_E; ++e) if (e0 + e < E) z[e] = src[e * J.es];
      }
      if (J.part) {
        const float full = (float)exp(ld * p.seg_len);
        const int n = rev ? p.nseg - 1 - seg : seg;
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
          const int s = rev ? p.nseg - 1 - i : i;
          const float f = s == p.nseg - 1 ? (float)exp(ld * (p.L - s * p.seg_len)) : full;
          const float* src = J.part + (head * p.nseg + s) * p.S + off;
#pragma unroll
          for (int e = 0; e < LT_E; ++e) if (e0 + e < E) z[e] = fmaf(f, z[e], src[e * J.es]);
        }
      }
    }
#pragma unroll 1
    for (int c = 0; c < nch; ++c) {
      if (!local) {
        bool ok = !dead;
        if (c > 0) ok = role_wait(&bars.zb_empty, (uint32_t)((c - 1) & 1), abort_flag, dead);
        if (ok) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(sZb + sw128_offset(x, j)) =
                make_uint4(pack_bf16(z[8 * j], z[8 * j + 1]), pack_bf16(z[8 * j + 2], z[8 * j + 3]), pack_bf16(z[8 * j + 4], z[8 * j + 5]),
                           pack_bf16(z[8 * j + 6], z[8 * j + 7]));
        }
        warp_arrive(&bars.zb_full, true);
      }
      const float aT = pw[min(LT_T, s1 - chunk_start(c))];
      if (role_wait(&bars.dz_full, (uint32_t)(c & 1), abort_flag, dead)) {
        tc_fence_after_sync();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t hi[8], mi[8], lo[8];
          tmem_ld8(tmem_addr(tbase, q * 32, LT_DZ + j * 8), hi);
          tmem_ld8(tmem_addr(tbase, q * 32, LT_DZ + 64 + j * 8), mi);
          tmem_ld8(tmem_addr(tbase, q * 32, LT_DZ + 128 + j * 8), lo);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i)
            z[8 * j + i] = fmaf(aT, z[8 * j + i], __uint_as_float(hi[i]) + (__uint_as_float(mi[i]) + __uint_as_float(lo[i])));
        }
      }
      warp_arrive(&bars.dz_empty, false);
    }
    float* out = local ? J.part + (head * p.nseg + seg) * p.S : (J.z1 && seg == (rev ? 0 : p.nseg - 1) ? J.z1 + head * p.S : nullptr);
    if (out && live && !dead) {
      out += x * J.xs + e0 * J.es;
#pragma unroll
      for (int e = 0; e < LT_E; ++e) if (e0 + e < E) out[e * J.es] = z[e];
    }
  } else if (role == 2) {
    // ---- scaled v': thread = token s; f v = hi + mid + lo exactly (each difference is exact in float32) ----
    const int s = q * 32 + lane;
#pragma unroll 1
    for (int c = 0; c < nch; ++c) {
      const int Tv = min(LT_T, s1 - chunk_start(c));
      const float f = s < Tv ? J.s_state * pw[rev ? s + 1 : Tv - 1 - s] : 0.f;
      const uint8_t* v = sm + ((c & 1) * LT_STAGE + 4) * BLK;
      bool ok = role_wait(&bars.v_full[c & 1], (uint32_t)((c >> 1) & 1), abort_flag, dead);
      if (c > 0) ok = role_wait(&bars.vd_empty, (uint32_t)((c - 1) & 1), abort_flag, dead) && ok;
      if (ok) {
#pragma unroll 2
        for (int j = 0; j < 8; ++j) {
          const uint32_t off = sw128_offset(s, j);
          const uint4 w = *reinterpret_cast<const uint4*>(v + off);
          const uint32_t in[4] = {w.x, w.y, w.z, w.w};
          uint32_t oh[4], om[4], ol[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float2 y;
            unpack_bf16(in[i], y.x, y.y);
            y = mul2(y, make_float2(f, f));
            oh[i] = pack_bf16(y.x, y.y);
            float2 t;
            unpack_bf16(oh[i], t.x, t.y);
            y = add2(y, make_float2(-t.x, -t.y));
            om[i] = pack_bf16(y.x, y.y);
            unpack_bf16(om[i], t.x, t.y);
            y = add2(y, make_float2(-t.x, -t.y));
            ol[i] = pack_bf16(y.x, y.y);
          }
          *reinterpret_cast<uint4*>(sVd + off) = make_uint4(oh[0], oh[1], oh[2], oh[3]);
          *reinterpret_cast<uint4*>(sVd + BLK + off) = make_uint4(om[0], om[1], om[2], om[3]);
          *reinterpret_cast<uint4*>(sVd + 2 * BLK + off) = make_uint4(ol[0], ol[1], ol[2], ol[3]);
        }
      }
      warp_arrive(&bars.vd_full, true);
      if (local) {                                           // nothing else reads the v' tile: this role gives the stage back
        named_bar_sync(3, 128);
        if (q == 0 && lane == 0) mbar_arrive(&bars.v_empty[c & 1]);
      }
    }
  } else if (!local) {
    // ---- read-out: thread = row t ----
    const int t = q * 32 + lane;
#pragma unroll 1
    for (int c = 0; c < nch; ++c) {
      const int t0 = chunk_start(c), Tv = min(LT_T, s1 - t0);
      uint8_t* out = sm + ((c & 1) * LT_STAGE + 4) * BLK;    // every reader of the v' tile is done once the accumulators are
      const float fi = t < Tv ? J.s_in * pw[rev ? Tv - 1 - t : t + 1] : 0.f, fo = J.s_out;
      const bool ok = role_wait(&bars.acc_full, (uint32_t)(c & 1), abort_flag, dead);
      if (ok) {
        tc_fence_after_sync();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t r[16], w[16];
          tmem_ld16(tmem_addr(tbase, q * 32, LT_O + j * 16), r);
          tmem_ld16(tmem_addr(tbase, q * 32, LT_O2 + j * 16), w);
          tmem_ld_wait();
          uint32_t o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 v = fma2(make_float2(fi, fi), f2(w[2 * i], w[2 * i + 1]), mul2(make_float2(fo, fo), f2(r[2 * i], r[2 * i + 1])));
            o[i] = pack_bf16(v.x, v.y);
          }
          *reinterpret_cast<uint4*>(out + sw128_offset(t, 2 * j)) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(out + sw128_offset(t, 2 * j + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
      }
      warp_arrive(&bars.acc_empty, true);
      named_bar_sync(2, 128);
      if (tid == 12 * 32) {
        if (ok) {
          tma_store_4d(my, out, e0, h, t0, b);
          bulk_commit_group();
          bulk_wait_group_read<0>();
        }
        mbar_arrive(&bars.v_empty[c & 1]);
      }
    }
    if (tid == 12 * 32) bulk_wait_group<0>();
  }
  tc_fence_before_sync();
  __syncthreads();
  if (tid == 0 && *abort_flag && p.status) atomicExch(p.status, 1);
  if (warp == 0) tmem_dealloc(tbase, 512);
}

// ---- host ----------------------------------------------------------------------------------------------------------
static bool tc_operand(const void* ptr, int64_t bs, int64_t ls, int64_t hs) {
  return aligned16(ptr) && bs % 8 == 0 && ls % 8 == 0 && hs % 8 == 0 && bs > 0 && ls > 0 && hs > 0 && bs < (1LL << 38) && ls < (1LL << 38) &&
         hs < (1LL << 38);
}

bool la_tc_serves(const LaArgs& a, bool bwd, int dtype) {
  if (dtype != BF16 || a.Dk % 8 || a.Dv % 8 || a.Dk > 128 || a.Dv > 128) return false;
  bool ok = tc_operand(a.q, a.q_bs, a.q_ls, a.q_hs) && tc_operand(a.k, a.k_bs, a.k_ls, a.k_hs) && tc_operand(a.v, a.v_bs, a.v_ls, a.v_hs);
  if (!bwd) return ok && tc_operand(a.y, a.y_bs, a.y_ls, a.y_hs);
  return ok && tc_operand(a.dy, a.dy_bs, a.dy_ls, a.dy_hs) && tc_operand(a.dq, a.dq_bs, a.dq_ls, a.dq_hs) &&
         tc_operand(a.dk, a.dk_bs, a.dk_ls, a.dk_hs) && tc_operand(a.dv, a.dv_bs, a.dv_ls, a.dv_hs);
}

int la_tc_segments(const LaArgs& a, bool bwd, int* seg_len) {
  const int64_t ev = (a.Dv + LT_E - 1) / LT_E, ek = (a.Dk + LT_E - 1) / LT_E;
  return la_segments((int64_t)a.B * a.H * (bwd ? 2 * ek + ev : ev), a.L, LT_T, seg_len);
}

// [B, L, H, D] with any strides as 128-token boxes of 64 channels of one head; what lies outside reads as zero and is not written
static int tc_map(CUtensorMap* m, const void* base, int D, int64_t bs, int64_t ls, int64_t hs, const LaPlan& p) {
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)p.H, (uint64_t)p.L, (uint64_t)p.B};
  const uint64_t str[3] = {(uint64_t)hs * 2, (uint64_t)ls * 2, (uint64_t)bs * 2};
  const uint32_t box[4] = {64, 1, LT_T, 1};
  return make_tensor_map_bf16(m, base, 4, dims, str, box);
}

int la_tc_launch(const LaArgs& a, bool bwd, cudaStream_t st) {
  int seg_len = 0, rc;
  const int nseg = la_tc_segments(a, bwd, &seg_len);
  ORBIT_CHECK_CUDA(cudaFuncSetAttribute(la_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LT_SMEM));
  for (int local = nseg > 1 ? 1 : 0; local >= 0; --local) {
    LaTcArgs t;
    if ((rc = la_plan(a, bwd, nseg, seg_len, local != 0, &t.p)) != OK) return rc;
    int ne = 1;
    for (int i = 0; i < t.p.njobs; ++i) {
      const LaJob& j = t.p.job[i];
      if ((j.E + LT_E - 1) / LT_E > ne) ne = (j.E + LT_E - 1) / LT_E;
      if ((rc = tc_map(&t.map[i][1], j.k, j.X, j.k_bs, j.k_ls, j.k_hs, t.p)) != OK) return rc;
      if ((rc = tc_map(&t.map[i][2], j.v, j.E, j.v_bs, j.v_ls, j.v_hs, t.p)) != OK) return rc;
      if (!local) {
        if ((rc = tc_map(&t.map[i][0], j.q, j.X, j.q_bs, j.q_ls, j.q_hs, t.p)) != OK) return rc;
        if ((rc = tc_map(&t.map[i][3], j.y, j.E, j.y_bs, j.y_ls, j.y_hs, t.p)) != OK) return rc;
      }
    }
    t.p.ne = ne;
    const int64_t grid = (int64_t)a.B * a.H * nseg * t.p.njobs * ne;
    ORBIT_REQUIRE(grid <= 0x7fffffffLL, ERR_UNSUPPORTED, "orbit_la: %lld (batch, head, segment) tiles are too many for one call", (long long)grid);
    la_tc_kernel<<<(unsigned)grid, LT_THREADS, LT_SMEM, st>>>(t, local);
    ORBIT_CHECK_LAUNCH("la_tc_kernel");
  }
  return OK;
}

}  // namespace orbit
