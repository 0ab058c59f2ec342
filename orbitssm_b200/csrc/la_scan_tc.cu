// Linear attention with a constant decay for each head on tcgen05 tensor cores (bfloat16, head widths that are multiples of 8
// up to 128).  The recurrence, its four roles (y, dq, dk, dv) and the split into segments are those of la_scan.cu; here a chunk
// is 128 tokens and its products are tensor-core tiles with float32 accumulators in TMEM.
//
// One CTA owns (batch, head, segment, 64 channels of v') and walks the chunks of its segment:
//   S1[t,s] = q'_t . k'_s                      128 x 128 x X   both operands as TMA wrote them
//   P[t,s]  = S1[t,s] a^{c-s} (s <= t, else 0) -> bfloat16     the only rounding of the part inside the chunk
//   O[t,e]  = P v' + q' Zb                     128 x 64 x (128 + X)   P read from TMEM; Zb = a^{c+1} s_in / s_out Z rounded to
//                                                              bfloat16, the only rounding of that part
//   dZ[x,e] = sum_s k'_s[x] (f_s v'_s[e])      128 x 192 x 128 f_s v' in three bfloat16 parts (hi + mid + lo hold all 24 bits of
//                                                              the float32 product) side by side, so that the float32 state and
//                                                              the state's gradient lose nothing to the operands' type
//   out = s_out a^{t-c} O;   Z = a^T Z + dZ                    Z in registers, float32
// The decay a^{t-s} is split into a column factor on the scores and a row factor on the float32 accumulator, counted from the
// middle of the chunk (c = 64; backwards in time a^{s-c} and a^{c-t}, c = 63), so that both parts of the output meet in one
// accumulator and no operand is rounded twice.  That needs a^{-64} to stay far from overflow: heads with a < 1/2 (`steep`) keep
// a^{t-s} on the scores, where it is at most 1, and the two parts in accumulators of their own.
//
// Warp-specialised, 27 warps that meet only through mbarriers (every wait bounded):
//   warps 0..3   decay mask: S1 -> P (TMEM to TMEM; the 32-column slabs beyond the diagonal are zero and written once)
//   warps 4..11  state: Z in registers (thread = state row, 32 of its channels), writes Zb, adds dZ
//   warps 12..19 scaled v': three bfloat16 tiles (thread = token, 32 channels)
//   warps 20..23 read-out: O -> output tile in the place of the v' tile -> TMA store
//   warp 24      one lane issues the TMA loads (two stages); warp 25 the MMAs S1 and O, warp 26 those of dZ
// Two issuing warps: the tensor pipe then has work of one queue while the other waits for its operands.
// 64 channels a CTA (two CTAs for a 128-wide head, adjacent so that q' and k' come from L2 the second time): the state then
// leaves room in shared memory for two stages of operands, and short batches fill twice the SMs.
#include "common.cuh"
#include "la_args.h"
#include "tc_common.cuh"
#include "tc_scan_common.cuh"

namespace orbit {
using namespace tc;

constexpr int LT_T = 128, LT_E = 64;
constexpr int LT_ZG = 2, LT_VG = 2;   // groups of four warps for the state and for v'
constexpr int LT_W_V = 4 + 4 * LT_ZG, LT_W_OUT = LT_W_V + 4 * LT_VG, LT_W_LOAD = LT_W_OUT + 4, LT_THREADS = (LT_W_LOAD + 3) * 32;   // first warps of the roles
constexpr uint32_t LT_S1 = 0, LT_P = 128, LT_O = 192, LT_DZ = 320;   // TMEM columns: 128, 64, 2 x 64, 192 (512 in all)
constexpr int LT_SMEM = (2 * 5 + 3 + 1) * (int)BLK + 1024;   // two stages of (q' 2, k' 2, v' 1), scaled v' 3, Zb 1 blocks of 16 KB
constexpr int LT_FWD_C = 64, LT_REV_C = 63;                  // the token that decays are counted from

struct LaTcArgs {
  CUtensorMap map[3][4];                                     // q', k', v', output of each job
  LaPlan p;
};

struct LtBars {
  uint64_t qk_full[2], qk_empty[2], v_full[2], v_empty[2], v_read[2], s1_full, s1_empty, p_full, p_empty, vd_full[2], vd_empty[2], zb_full,
      zb_empty, dz_full[2], dz_empty[2], acc_full[2], acc_empty[2];
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
// a^n for |n| <= 128 from the table of a^0 .. a^128 (n < 0 only where a is at least 1/2)
__device__ __forceinline__ float power(const float* pw, int n) { return n >= 0 ? pw[n] : __fdividef(1.f, pw[-n]); }

// One lane of a converged warp, the same one every time.  Issued under a plain `lane == 0` test the compiler takes the MMA's
// operands for values that differ between lanes: 94 cycles an instruction at N = 64 against 75, and 94 against 42 with the
// operand in TMEM (measured alone; the four products of a chunk 4450 cycles against 2000).
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok));
  return ok != 0;
}

struct LtShared {
  LtBars bars;
  float pw[LT_T + 1];                                        // a^0 .. a^128
  uint32_t tmem_slot;
  int abort_flag;
};

// The walk of one CTA; the compiler's copies for each direction, kind of head and launch keep the loops of the roles short.
template <bool rev, bool steep, bool local>
__device__ __forceinline__ void la_tc_walk(const LaTcArgs& a, LtShared& sh, uint8_t* sm, const int jb, const int b, const int h,
                                           const int seg, const int et, const double ld) {
  const LaPlan& p = a.p;
  const LaJob& J = p.job[jb];
  const int X = J.X, E = J.E, e0 = et * LT_E;
  const CUtensorMap *mq = &a.map[jb][0], *mk = &a.map[jb][1], *mv = &a.map[jb][2], *my = &a.map[jb][3];
  LtBars& bars = sh.bars;
  const float* pw = sh.pw;
  // Blocks of a stage and its k' and v' tiles in it.  The state-only launch loads no q' and has room for two sets of scaled v' and
  // of accumulators, so that scaling, product and state update of three chunks run side by side.
  constexpr int STAGE = local ? 3 : 5, KO = local ? 0 : 2, VO = local ? 2 : 4, SETS = local ? 2 : 1;
  uint8_t* sVd = sm + 2 * STAGE * BLK;                       // scaled v': hi, mid, lo
  uint8_t* sZb = sVd + 3 * BLK;                              // entering state, bfloat16 [128 x][64 e]
  auto set_of = [](int c) { return c % SETS; };
  auto turn_of = [](int c) { return (uint32_t)((c / SETS) & 1); };   // phase of a set's barriers at chunk c
  constexpr uint32_t DZ = local ? 0 : LT_DZ;
  constexpr int VG = local ? 4 : LT_VG;                      // groups that scale v': the mask's and the read-out's warps join there
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, q = warp & 3;
  const int s0 = seg * p.seg_len, s1 = min(p.L, s0 + p.seg_len), nch = (s1 - s0 + LT_T - 1) / LT_T;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.qk_full[i], 1);
      mbar_init(&bars.qk_empty[i], local ? 1 : 2);           // released by both issuing warps
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.v_empty[i], local ? 4 * VG : 1);       // by the read-out, which puts its tile there (local: the scaling warps)
      mbar_init(&bars.v_read[i], 4 * VG);
      mbar_init(&bars.vd_full[i], 4 * VG);
      mbar_init(&bars.vd_empty[i], 1);
      mbar_init(&bars.dz_full[i], 1);
      mbar_init(&bars.dz_empty[i], 4 * LT_ZG);
      mbar_init(&bars.acc_full[i], 1);
      mbar_init(&bars.acc_empty[i], 4);
    }
    mbar_init(&bars.s1_full, 1);
    mbar_init(&bars.s1_empty, 4);
    mbar_init(&bars.p_full, 4);
    mbar_init(&bars.p_empty, 1);
    mbar_init(&bars.zb_full, 4 * LT_ZG);
    mbar_init(&bars.zb_empty, 1);
    mbar_fence_init();
    sh.abort_flag = 0;
  }
  if (tid <= LT_T) sh.pw[tid] = tid == 0 ? 1.f : (float)exp(ld * tid);
  if (warp == 0) tmem_alloc(&sh.tmem_slot, 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tbase = sh.tmem_slot;
  volatile int* abort_flag = &sh.abort_flag;
  bool dead = false;
  // The state is kept times the factor that makes the carried part share the row factor of the other (steep heads and the
  // state-only launch: as it is), so that Zb is one rounding of what the registers hold.
  const float zscale = steep || local ? 1.f : J.s_in / J.s_out * power(pw, rev ? LT_T - 1 - LT_REV_C : LT_FWD_C + 1);
  auto chunk_start = [&](int c) { return s0 + (rev ? nch - 1 - c : c) * LT_T; };

  if (warp == LT_W_LOAD) {
    if (lane == 0) {
      // ---- producer ----
      int done_qk = 0, done_v = 0;                           // loads issued
#pragma unroll 1
      for (int c = 0; c < nch; ++c) {
        const int s = c & 1, t0 = chunk_start(c);
        uint8_t* st = sm + s * STAGE * BLK;
        const int blocks = X > 64 ? 2 : 1;                   // the second block of a narrow head is never contracted
        auto load_v = [&] {
          if (c >= 2 && !lane_wait(&bars.v_empty[s], (uint32_t)(((c >> 1) - 1) & 1), abort_flag, dead)) return false;
          mbar_expect_tx(&bars.v_full[s], BLK);
          tma_load_4d(st + VO * BLK, mv, &bars.v_full[s], e0, h, t0, b);
          ++done_v;
          return true;
        };
        // whichever place is free first: that of v' where the scaling gives it back, that of q' and k' where the read-out does
        if (local && !load_v()) break;
        if (c >= 2 && !lane_wait(&bars.qk_empty[s], (uint32_t)(((c >> 1) - 1) & 1), abort_flag, dead)) break;
        mbar_expect_tx(&bars.qk_full[s], (uint32_t)(local ? blocks : 2 * blocks) * BLK);
        for (int i = 0; i < blocks; ++i) {
          if (!local) tma_load_4d(st + i * BLK, mq, &bars.qk_full[s], i * 64, h, t0, b);
          tma_load_4d(st + (KO + i) * BLK, mk, &bars.qk_full[s], i * 64, h, t0, b);
        }
        ++done_qk;
        if (!local && !load_v()) break;
      }
      if (dead) {                                            // wind-down: what was issued has to land before the CTA goes
        for (int k = max(0, done_qk - 2); k < done_qk; ++k) mbar_wait(&bars.qk_full[k & 1], (uint32_t)((k >> 1) & 1));
        for (int k = max(0, done_v - 2); k < done_v; ++k) mbar_wait(&bars.v_full[k & 1], (uint32_t)((k >> 1) & 1));
      }
    }
    __syncwarp();
  } else if (warp == LT_W_LOAD + 1) {
    // ---- MMA issuer of the scores and the output: the warp waits, one lane issues ----
    if (!local) {
      const uint32_t id_s = idesc_bf16(128, 128, 0, 0), id_o = idesc_bf16(128, 64, 0, 1);
      const int kx = (X + 15) / 16;
      const uint32_t zb = lo_mn(smem_u32(sZb));
      auto base = [&](int c, int blk) { return smem_u32(sm + ((c & 1) * STAGE + blk) * BLK); };
      auto scores = [&](int c) {
        const uint32_t aq = lo_k(base(c, 0)), bk = lo_k(base(c, KO));
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < 8; ++ks)
            if (ks < kx) umma_bf16_h(tbase + LT_S1, aq + inc_k(ks), bk + inc_k(ks), id_s, ks > 0 ? 1u : 0u);
          umma_commit(&bars.s1_full);
        }
      };
      if (role_wait(&bars.qk_full[0], 0, abort_flag, dead)) {
        tc_fence_after_sync();
        scores(0);
      }
#pragma unroll 1
      for (int c = 0; c < nch && !dead; ++c) {
        const uint32_t ph = (uint32_t)(c & 1);
        // accumulators of this chunk: one of two sets; steep heads use both, for the two parts
        const uint32_t acc2 = tbase + LT_O + (steep ? 0u : ph * 64u), acc1 = steep ? tbase + LT_O + 64u : acc2;
        if (!role_wait(&bars.zb_full, ph, abort_flag, dead)) break;
        if (steep && c > 0 && !role_wait(&bars.acc_empty[ph ^ 1u], (uint32_t)(((c - 1) >> 1) & 1), abort_flag, dead)) break;
        if (!steep && c > 1 && !role_wait(&bars.acc_empty[ph], (uint32_t)(((c >> 1) - 1) & 1), abort_flag, dead)) break;
        tc_fence_after_sync();
        const uint32_t aq = lo_k(base(c, 0));
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < 8; ++ks)
            if (ks < kx) umma_bf16_h(acc2, aq + inc_k(ks), zb + inc_mn(ks), id_o, ks > 0 ? 1u : 0u);
          umma_commit(&bars.zb_empty);
          umma_commit(&bars.qk_empty[c & 1]);                // this warp has read q' and k' of the chunk for the last time
        }
        if (c + 1 < nch) {
          if (!role_wait(&bars.qk_full[(c + 1) & 1], (uint32_t)(((c + 1) >> 1) & 1), abort_flag, dead)) break;
          if (!role_wait(&bars.s1_empty, ph, abort_flag, dead)) break;
          tc_fence_after_sync();
          scores(c + 1);
        }
        if (!role_wait(&bars.p_full, ph, abort_flag, dead)) break;
        if (!role_wait(&bars.v_full[c & 1], (uint32_t)((c >> 1) & 1), abort_flag, dead)) break;
        tc_fence_after_sync();
        const uint32_t bv = lo_mn(base(c, VO));
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < 8; ++ks)
            umma_bf16_ta_h(acc1, tbase + LT_P + ks * 8, bv + inc_mn(ks), id_o, (ks > 0 || !steep) ? 1u : 0u);
          umma_commit(&bars.p_empty);
          umma_commit(&bars.acc_full[c & 1]);
        }
      }
    }
    __syncwarp();
  } else if (warp == LT_W_LOAD + 2) {
    // ---- MMA issuer of the state update ----
    const uint32_t id_z = idesc_bf16(128, 192, 1, 1), vd = lo_mn(smem_u32(sVd));
#pragma unroll 1
    for (int c = 0; c < nch && !dead; ++c) {
      if (!role_wait(&bars.qk_full[c & 1], (uint32_t)((c >> 1) & 1), abort_flag, dead)) break;
      const int set = set_of(c);
      if (c >= SETS && !role_wait(&bars.dz_empty[set], turn_of(c - SETS), abort_flag, dead)) break;
      if (!role_wait(&bars.vd_full[set], turn_of(c), abort_flag, dead)) break;
      tc_fence_after_sync();
      const uint32_t ak = lo_mn(smem_u32(sm + ((c & 1) * STAGE + KO) * BLK));
      if (elect_one()) {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) umma_bf16_h(tbase + DZ + set * 192, ak + inc_mn(ks), vd + set * ((3 * BLK) >> 4) + inc_mn(ks), id_z, ks > 0 ? 1u : 0u);
        umma_commit(&bars.dz_full[set]);
        umma_commit(&bars.vd_empty[set]);
        umma_commit(&bars.qk_empty[c & 1]);
      }
    }
    __syncwarp();
  } else if (!local && warp < 4) {
    {
      // ---- decay mask: thread = row t; slab j holds columns 32 j .. 32 j + 31 ----
      {
        uint32_t z[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = 0u;
#pragma unroll 1
        for (int j = 0; j < 4; ++j)
          if (rev ? j < q : j > q) tmem_st16(tmem_addr(tbase, q * 32, LT_P + j * 16), z);
        tmem_st_wait();
      }
      const int j0 = rev ? q : 0, j1 = rev ? 3 : q;
      // Column factors a^{c-s} (reverse a^{s-c}) run along the row by repeated multiplication, two chains of pairs: at most 32
      // products of rounded factors, off by 2^-18, against the 2^-8 of the rounding that follows.  Shared memory is busy with the
      // MMAs' operands: a table there costs its latency for every few elements.
      const int n0 = rev ? 32 * q - LT_REV_C : LT_FWD_C, d0 = rev ? 1 : -1;
      const float a4 = steep ? 0.f : power(pw, 4 * d0);
      const float2 step = make_float2(a4, a4);
      const float2 g0 = steep ? step : make_float2(power(pw, n0), power(pw, n0 + d0));
      const float2 g1 = steep ? step : make_float2(power(pw, n0 + 2 * d0), power(pw, n0 + 3 * d0));
#pragma unroll 1
      for (int c = 0; c < nch; ++c) {
        bool ok = role_wait(&bars.s1_full, (uint32_t)(c & 1), abort_flag, dead);
        if (c > 0) ok = role_wait(&bars.p_empty, (uint32_t)((c - 1) & 1), abort_flag, dead) && ok;
        if (ok) {
          tc_fence_after_sync();
          float2 f0 = g0, f1 = g1;
#pragma unroll 1
          for (int j = j0; j <= j1; ++j) {
            uint32_t r[32], o[16];
            tmem_ld32(tmem_addr(tbase, q * 32, LT_S1 + j * 32), r);
            tmem_ld_wait();
            if (!steep) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float2 u = mul2(f2(r[4 * i], r[4 * i + 1]), f0), w = mul2(f2(r[4 * i + 2], r[4 * i + 3]), f1);
                f0 = mul2(f0, step);
                f1 = mul2(f1, step);
                r[4 * i] = __float_as_uint(u.x);
                r[4 * i + 1] = __float_as_uint(u.y);
                r[4 * i + 2] = __float_as_uint(w.x);
                r[4 * i + 3] = __float_as_uint(w.y);
              }
            } else {
              // a^{t-s} from the powers themselves: at most 1 wherever the score is kept
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const int n = rev ? 32 * (j - q) + i - lane : 32 * (q - j) + lane - i;
                r[i] = __float_as_uint(__uint_as_float(r[i]) * pw[max(n, 0)]);
              }
            }
            if (j == q) {                                    // zero beyond the diagonal, whatever the score
#pragma unroll
              for (int i = 0; i < 32; ++i) r[i] = (rev ? i >= lane : i <= lane) ? r[i] : 0u;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = pack_bf16(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
            tmem_st16(tmem_addr(tbase, q * 32, LT_P + j * 16), o);
          }
          tmem_st_wait();
        }
        warp_arrive(&bars.s1_empty, false);
        if (lane == 0) mbar_arrive(&bars.p_full);
      }
    }
  } else if (warp >= 4 && warp < LT_W_V) {
    // ---- state: thread = state row x, ZE of its channels in registers ----
    constexpr int ZE = LT_E / LT_ZG;
    const int hf = (warp - 4) >> 2, ez = hf * ZE;            // first of this thread's channels in the tile
    const int x = q * 32 + lane;
    const int64_t head = (int64_t)b * p.H + h;
    float z[ZE];
#pragma unroll
    for (int e = 0; e < ZE; ++e) z[e] = 0.f;
    const bool live = x < X;
    if (!local && live) {
      // the carried state and the shares of the segments before this one, each with its decay since
      const int64_t off = x * J.xs + (e0 + ez) * J.es;
      if (J.z0) {
        const float* src = J.z0 + head * p.S + off;
#pragma unroll
        for (int e = 0; e < ZE; ++e) if (e0 + ez + e < E) z[e] = src[e * J.es];
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
          for (int e = 0; e < ZE; ++e) if (e0 + ez + e < E) z[e] = fmaf(f, z[e], src[e * J.es]);
        }
      }
    }
    if (!local) {
#pragma unroll
      for (int e = 0; e < ZE; ++e) z[e] *= zscale;
    }
    const float a_full = pw[LT_T];
#pragma unroll 1
    for (int c = 0; c < nch; ++c) {
      const int Tv = min(LT_T, s1 - chunk_start(c));
      if (!local) {
        bool ok = !dead;
        if (c > 0) ok = role_wait(&bars.zb_empty, (uint32_t)((c - 1) & 1), abort_flag, dead);
        if (ok) {
          const bool odd = rev && !steep && Tv != LT_T;      // a ragged chunk is counted from its own end backwards in time
          const float zs = odd ? __fdividef(1.f, pw[LT_T - Tv]) : 1.f;
#pragma unroll
          for (int j = 0; j < ZE / 8; ++j) {
            float2 y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              y[i] = make_float2(z[8 * j + 2 * i], z[8 * j + 2 * i + 1]);
              if (odd) y[i] = mul2(y[i], make_float2(zs, zs));
            }
            *reinterpret_cast<uint4*>(sZb + sw128_offset(x, ez / 8 + j)) =
                make_uint4(pack_bf16(y[0].x, y[0].y), pack_bf16(y[1].x, y[1].y), pack_bf16(y[2].x, y[2].y), pack_bf16(y[3].x, y[3].y));
          }
        }
        warp_arrive(&bars.zb_full, true);
      }
      const float aT = Tv == LT_T ? a_full : pw[Tv];
      const int set = set_of(c);
      if (role_wait(&bars.dz_full[set], turn_of(c), abort_flag, dead)) {
        tc_fence_after_sync();
        const uint32_t dz = tmem_addr(tbase, q * 32, DZ + set * 192 + ez);
#pragma unroll
        for (int j = 0; j < ZE / 8; ++j) {
          uint32_t hi[8], mi[8], lo[8];
          tmem_ld8(dz + j * 8, hi);
          tmem_ld8(dz + 64 + j * 8, mi);
          tmem_ld8(dz + 128 + j * 8, lo);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const float2 d = add2(f2(hi[i], hi[i + 1]), add2(f2(mi[i], mi[i + 1]), f2(lo[i], lo[i + 1])));
            const float2 y = fma2(make_float2(aT, aT), make_float2(z[8 * j + i], z[8 * j + i + 1]), d);
            z[8 * j + i] = y.x;
            z[8 * j + i + 1] = y.y;
          }
        }
      }
      warp_arrive(&bars.dz_empty[set], false);
    }
    float* out = local ? J.part + (head * p.nseg + seg) * p.S : (J.z1 && seg == (rev ? 0 : p.nseg - 1) ? J.z1 + head * p.S : nullptr);
    if (out && live && !dead) {
      out += x * J.xs + (e0 + ez) * J.es;
      const float unscale = 1.f / zscale;
#pragma unroll
      for (int e = 0; e < ZE; ++e) if (e0 + ez + e < E) out[e * J.es] = z[e] * unscale;
    }
  } else if (local || (warp >= LT_W_V && warp < LT_W_OUT)) {
    // ---- scaled v': thread = token s; f v is cut into its upper, middle and lower eight bits: three bfloat16 values whose sum is
    // the float32 product exactly ----
    constexpr int VJ = 8 / VG;                               // 16-byte pieces of a row
    const int g = warp >= LT_W_OUT ? 3 : warp >= LT_W_V ? (warp - LT_W_V) >> 2 : 2;
    const int s = q * 32 + lane, j0 = g * VJ;
    const float fz = local ? J.s_state : J.s_state * zscale;
    const float f_full = fz * pw[rev ? s + 1 : LT_T - 1 - s];
    const uint32_t row = s * 128u, sw = s & 7u;
#pragma unroll 1
    for (int c = 0; c < nch; ++c) {
      const int Tv = min(LT_T, s1 - chunk_start(c));
      const float f = Tv == LT_T ? f_full : s < Tv ? fz * pw[rev ? s + 1 : Tv - 1 - s] : 0.f;
      const uint8_t* v = sm + ((c & 1) * STAGE + VO) * BLK;
      uint4 w[VJ];
      bool ok = role_wait(&bars.v_full[c & 1], (uint32_t)((c >> 1) & 1), abort_flag, dead);
      if (ok) {
#pragma unroll
        for (int j = 0; j < VJ; ++j) w[j] = *reinterpret_cast<const uint4*>(v + row + (((j0 + j) ^ sw) << 4));   // all of them before the first store
      }
      if (local) {                                           // nothing else reads the v' tile there
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.v_empty[c & 1]);
      }
      const int set = set_of(c);
      if (c >= SETS) ok = role_wait(&bars.vd_empty[set], turn_of(c - SETS), abort_flag, dead) && ok;
      if (ok) {
#pragma unroll
        for (int j = 0; j < VJ; ++j) {
          uint4 oh, om, ol;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float2 y, t;
            const uint32_t w0 = reinterpret_cast<const uint32_t*>(&w[j])[i];
            unpack_bf16(w0, y.x, y.y);
            y = mul2(y, make_float2(f, f));
            const uint32_t hi = __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x7632);
            t = make_float2(__uint_as_float(__float_as_uint(y.x) & 0xffff0000u), __uint_as_float(__float_as_uint(y.y) & 0xffff0000u));
            y = fma2(t, make_float2(-1.f, -1.f), y);
            const uint32_t mid = __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x7632);
            t = make_float2(__uint_as_float(__float_as_uint(y.x) & 0xffff0000u), __uint_as_float(__float_as_uint(y.y) & 0xffff0000u));
            y = fma2(t, make_float2(-1.f, -1.f), y);
            reinterpret_cast<uint32_t*>(&oh)[i] = hi;
            reinterpret_cast<uint32_t*>(&om)[i] = mid;
            reinterpret_cast<uint32_t*>(&ol)[i] = pack_bf16(y.x, y.y);
          }
          uint8_t* dst = sVd + set * 3 * BLK + row + (((j0 + j) ^ sw) << 4);
          *reinterpret_cast<uint4*>(dst) = oh;
          *reinterpret_cast<uint4*>(dst + BLK) = om;
          *reinterpret_cast<uint4*>(dst + 2 * BLK) = ol;
        }
      }
      warp_arrive(&bars.vd_full[set], true);                     // ends in a warp barrier: every lane has read its part of v'
      if (!local && lane == 0) mbar_arrive(&bars.v_read[c & 1]);
    }
  } else if (warp < LT_W_LOAD) {
    // ---- read-out: thread = row t; the tile leaves from the place of the v' tile ----
    const int t = q * 32 + lane;
    const float fo = J.s_out * (steep ? 1.f : power(pw, rev ? LT_REV_C - t : t - LT_FWD_C));   // row factor
#pragma unroll 1
    for (int c = 0; c < nch; ++c) {
      const int t0 = chunk_start(c), Tv = min(LT_T, s1 - t0);
      uint8_t* out = sm + ((c & 1) * STAGE + VO) * BLK;
      bool ok = role_wait(&bars.acc_full[c & 1], (uint32_t)((c >> 1) & 1), abort_flag, dead);   // the product has read the v' tile ...
      ok = role_wait(&bars.v_read[c & 1], (uint32_t)((c >> 1) & 1), abort_flag, dead) && ok;    // ... and so has the scaling
      if (ok) {
        tc_fence_after_sync();
        const uint32_t acc = tmem_addr(tbase, q * 32, LT_O + (steep ? 64 : (c & 1) * 64));
        const float fi = steep && t < Tv ? J.s_in * pw[rev ? Tv - 1 - t : t + 1] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t r[16], o[8];
          tmem_ld16(acc + j * 16, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 v = mul2(make_float2(fo, fo), f2(r[2 * i], r[2 * i + 1]));
            r[2 * i] = __float_as_uint(v.x);
            r[2 * i + 1] = __float_as_uint(v.y);
          }
          if (steep) {                                       // the carried part with a row factor of its own
            uint32_t w[16];
            tmem_ld16(tmem_addr(tbase, q * 32, LT_O + j * 16), w);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(fmaf(fi, __uint_as_float(w[i]), __uint_as_float(r[i])));
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = pack_bf16(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
          *reinterpret_cast<uint4*>(out + sw128_offset(t, 2 * j)) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(out + sw128_offset(t, 2 * j + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
      }
      warp_arrive(&bars.acc_empty[c & 1], true);
      named_bar_sync(2, 128);
      if (tid == LT_W_OUT * 32) {
        if (ok) {
          tma_store_4d(my, out, e0, h, t0, b);
          bulk_commit_group();
          bulk_wait_group_read<0>();
        }
        mbar_arrive(&bars.v_empty[c & 1]);
      }
    }
    if (tid == LT_W_OUT * 32) bulk_wait_group<0>();
  }
  tc_fence_before_sync();
  __syncthreads();
  if (tid == 0 && *abort_flag && p.status) atomicExch(p.status, 1);
  if (warp == 0) tmem_dealloc(tbase, 512);
}

__global__ void __launch_bounds__(LT_THREADS, 1) la_tc_kernel(const __grid_constant__ LaTcArgs a, const int local) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ LtShared sh;
  const LaPlan& p = a.p;
  // tile index: e tile fastest, then head (neighbours in memory), segment, batch, and the job last: CTAs that run side by side then share their code
  // (jobs side by side would share q, k, v and dy in L2, but were 17 % slower in the backward pass)
  int64_t id = blockIdx.x;
  const int ne = p.ne;
  const int et = (int)(id % ne);
  id /= ne;
  const int h = (int)(id % p.H);
  id /= p.H;
  const int seg = (int)(id % p.nseg);
  id /= p.nseg;
  const int b = (int)(id % p.B), jb = (int)(id / p.B);
  const LaJob& J = p.job[jb];
  const int rev = J.reverse;
  if (et * LT_E >= J.E) return;
  if (local && seg == (rev ? 0 : p.nseg - 1)) return;        // nobody reads the last segment's share
  uint8_t* sm = align1024(smem_raw);
  const double ld = (double)p.log_decay[h];
  const bool steep = !(fabs(ld) <= 0.693147);
  if (local) {
    if (rev) la_tc_walk<true, false, true>(a, sh, sm, jb, b, h, seg, et, ld);
    else la_tc_walk<false, false, true>(a, sh, sm, jb, b, h, seg, et, ld);
  } else if (!steep) {
    if (rev) la_tc_walk<true, false, false>(a, sh, sm, jb, b, h, seg, et, ld);
    else la_tc_walk<false, false, false>(a, sh, sm, jb, b, h, seg, et, ld);
  } else {
    if (rev) la_tc_walk<true, true, false>(a, sh, sm, jb, b, h, seg, et, ld);
    else la_tc_walk<false, true, false>(a, sh, sm, jb, b, h, seg, et, ld);
  }
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
