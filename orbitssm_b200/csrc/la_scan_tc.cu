// Linear attention with a constant decay for each head on tcgen05 tensor cores (bfloat16, head widths that are multiples of 8
// up to 128).  The recurrence, its four roles (y, dq, dk, dv) and the split into segments are those of la_scan.cu; here a chunk
// is 128 tokens and its products are tensor-core tiles with float32 accumulators in TMEM.
//
// One CTA owns (batch, head, segment) and walks the chunks of its segment:
//   S1[t,s] = q'_t . k'_s                      128 x 128 x X   both operands as TMA wrote them
//   P[t,s]  = S1[t,s] a^{c-s} (s <= t, else 0) -> bfloat16     the only rounding of the part inside the chunk (the rows that
//                                                              a pass begins with, 32 at least: in two parts)
//   O[t,e]  = P v' + q' Zb^T                   128 x E x (128 + X)   P read from TMEM; Zb = a^{c+1} s_in / s_out Z rounded to
//                                                              bfloat16, the only rounding of that part
//   dZ[e,x] = sum_s (f_s v'_s[e]) k'_s[x]      128 x X x 384   f_s v' in three bfloat16 parts (their sum is it to 2^-25),
//                                                              read from TMEM, so that the float32 state and the state's gradient
//                                                              lose nothing to the operands' type
//   out = s_out a^{t-c} O;   Z = a^T Z + dZ                    Z [e, x] in registers, float32
// The decay a^{t-s} is split into a column factor on the scores and a row factor on the float32 accumulator, counted from the
// middle of the chunk (c = 64; backwards in time a^{s-c} and a^{c-t}, c = 63), so that both parts of the output meet in one
// accumulator and no operand is rounded twice.  It also takes a^{64} of the range of float32 at either end, so heads with
// a < 2^{-1/2} (`steep`) keep a^{t-s} on the scores, where it is at most 1, and their carried part is scaled row by row in TMEM before
// P v' joins it ([8, 4096, 16, 128, 128] forward 164 us instead of 118, backward 499 instead of 340; with the limit at 1/2 values of
// 2^80 gave NaN there, and gradients of 2^-60 lost the state's).
//
// What bounds it is no one unit: the chain of hand-overs between the roles within a chunk, and the power limit.  Counted over a
// forward launch at [8, 2048, 16, 128, 128] (of the cycles that an SM is active): tensor pipe 46 %, shared memory 54 % (30 for
// the operands of MMAs, 24 for ordinary accesses), issue 48 %.  Operands are kept in TMEM where it can hold them: per chunk and
// head of 128 x 128 the tiles move 96 KB in, 288 KB to the MMAs and 160 KB for the element passes.  (With the parts of f v' in shared
// memory and 64 channels a CTA it was 800 KB, and 158 us where it now takes 117.)  72 registers a thread at launch leave the six walks of
// this kernel 1396 bytes of spill stores and 2732 of loads: a walk compiled alone has 76 / 76, of steep heads 640 / 644, state-only
// none.
// Measured: forward [8, 4096, 16, 128, 128] 117 us (4.6 TB/s of operands and output), backward 340 us; prompt
// [1, 65536, 16, 128, 128] 340 us.  Random operands draw 1000 W and the SM clock falls to 1.4 to 1.6 GHz; zeros run 20% faster.
// bfloat16 calls that these tiles do not serve take the float32 kernels, which need 80 us for [1, 131, 16, 128, 128] where these
// need 18, and 3827 us for [8, 4096, 16, 128, 128].
//
// Warp-specialised, 28 warps that meet only through mbarriers (every wait bounded):
//   warps 0..3   decay mask: S1 -> P, in the place of S1 (thread = row t)
//   warps 4..11  state: Z in registers (thread = channel e, 64 state columns), writes Zb, adds dZ
//   warps 12..19 parts of f v' into TMEM (thread = channel e, 64 tokens)
//   warps 20..23 read-out: O -> output tile in the place of the v' tile -> TMA store (thread = row t)
//   warp 24      one lane issues the TMA loads (two stages); warp 25 the MMAs S1 and O, warp 26 those of dZ; warp 27 idles
// Two issuing warps: the tensor pipe then has work of one queue while the other waits for its operands.  Registers move from the
// other warpgroups to the state's (setmaxnreg: 112 of 72 at launch).
#include "common.cuh"
#include "la_args.h"
#include "tc_common.cuh"
#include "tc_scan_common.cuh"

namespace orbit {
using namespace tc;

constexpr int LT_T = 128;
constexpr int LT_W_STATE = 4, LT_W_V = 12, LT_W_OUT = 20, LT_W_LOAD = 24, LT_THREADS = 28 * 32;   // first warps of the roles
constexpr uint32_t LT_S1 = 0, LT_P = 0, LT_O = 128, LT_DZ = 256, LT_V = 384;   // TMEM columns: 128, 128, 128 and two sets of 3 x 16 (in 512)
constexpr uint32_t LT_REST = LT_V + 48, LT_REST_STRIDE = 64;   // 16 columns behind either set: the second parts of P
constexpr int LT_STAGE = 6;                                  // blocks of 16 KB in a stage: q' 2, k' 2, v' 2
constexpr int LT_SMEM = (2 * LT_STAGE + 2) * (int)BLK + 1024;
constexpr int LT_FWD_C = 64, LT_REV_C = 63;                  // the token that decays are counted from
// registers of a thread at launch, and of the warpgroups after they have been dealt out: mask, state (2), parts (2), read-out, issuers
constexpr int LT_R0 = 72, LT_R_MASK = 64, LT_R_STATE = 112, LT_R_V = 64, LT_R_OUT = 56, LT_R_ISSUE = 32;
static_assert(LT_R_MASK + 2 * LT_R_STATE + 2 * LT_R_V + LT_R_OUT + LT_R_ISSUE <= 7 * LT_R0, "the shares exceed what the block is launched with");

struct LaTcArgs {
  CUtensorMap map[3][4];                                     // q', k', v', output of each job
  LaPlan p;
};

struct LtBars {
  uint64_t qk_full[2], qk_empty[2], v_full[2], v_empty[2], v_read[2], s1_full, p_full, p_empty, o2_full, vd_full[2], vd_empty[2],
      zb_full, zb_empty, dz_full[2], dz_empty[2], acc_full, acc_empty;
};

template <int R> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }

// 16 lanes x 8 consecutive 32-bit columns <- 4 registers per thread, as 8 x 8 tiles of 16-bit pairs come out of ldmatrix: thread t
// writes lane t / 4, column t % 4 (r0), lane 8 + t / 4 (r1), and the same four columns further (r2, r3)
__device__ __forceinline__ void tmem_st_16x128b_x2(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
// four 8 x 8 tiles of 16-bit elements, transposed: thread t gets elements (row 2 (t % 4), column t / 4) and the row after it
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t saddr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(saddr) : "memory");
}
__device__ __forceinline__ uint32_t bf2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t bf2_mul(uint32_t a, uint32_t b) { return bf2_fma(a, b, 0x80008000u); }   // -0: the product's own sign of zero
__device__ __forceinline__ uint32_t bf2_add(uint32_t a, uint32_t b) { return bf2_fma(a, 0x3f803f80u, b); }
__device__ __forceinline__ uint32_t bf2_neg(uint32_t a) { return a ^ 0x80008000u; }

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
// a^n for |n| <= 128 from the table of a^0 .. a^128 (n < 0 only where a is at least 2^{-1/2})
__device__ __forceinline__ float power(const float* pw, int n) { return n >= 0 ? pw[n] : __fdividef(1.f, pw[-n]); }

// One lane of a converged warp, the same one every time.  Issued under a plain `lane == 0` test the compiler takes the MMA's
// operands for values that differ between lanes: 94 cycles an instruction at N = 64 against 75, and 94 against 42 with the
// operand in TMEM (measured alone).
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
  uint32_t fw[3][LT_T / 2];                                  // bfloat16 parts of the write factors f_s of the chunk, two tokens to a word
  uint32_t tmem_slot;
  int abort_flag;
};

// The walk of one CTA; the compiler's copies for each direction, kind of head and launch keep the loops of the roles short.
template <bool rev, bool steep, bool local>
__device__ __forceinline__ void la_tc_walk(const LaTcArgs& a, LtShared& sh, uint8_t* sm, const int jb, const int b, const int h,
                                           const int seg, const int et, const double ld) {
  const LaPlan& p = a.p;
  const LaJob& J = p.job[jb];
  const int X = J.X, e0 = et * 64, E = p.ne > 1 ? min(64, J.E - e0) : J.E;   // channels e0 .. e0 + E - 1 of v' and the output
  const CUtensorMap *mq = &a.map[jb][0], *mk = &a.map[jb][1], *mv = &a.map[jb][2], *my = &a.map[jb][3];
  LtBars& bars = sh.bars;
  const float* pw = sh.pw;
  uint8_t* sZb = sm + 2 * LT_STAGE * BLK;                    // entering state, bfloat16 [128 e][128 x] in two 64-column blocks
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, q = warp & 3;
  const int s0 = seg * p.seg_len, s1 = min(p.L, s0 + p.seg_len), nch = (s1 - s0 + LT_T - 1) / LT_T;
  const int xblocks = X > 64 ? 2 : 1, eblocks = E > 64 ? 2 : 1;   // a narrow head's second blocks are never loaded nor read
  // Where the pass over the sequence begins, P keeps the rest of its rounding as a second part: the scores among the first 32 tokens
  // (backwards in time: among the last two slabs, which hold the last 32 tokens of a ragged chunk).  Without a state these rows are
  // then rounded once, as the step's are, however many tokens follow.  It is two to four MMAs a sequence; of the whole of P it would
  // be 8 in every chunk: [8, 4096, 16, 128, 128] 138 us instead of 117 and backward 388 instead of 336, for an error of 1.33 times
  // the output rounding's own instead of 1.41 (Zb's rounding remains).
  const bool opens = !local && seg == (rev ? p.nseg - 1 : 0);
  const int rest_to = rev ? (min(LT_T, s1 - s0 - (nch - 1) * LT_T) - 1) >> 5 : 0, rest_from = rev ? max(rest_to - 1, 0) : 0;   // slabs
  // The state-only launch has room for two accumulators of dZ in the places of S1 and O: the next product need not wait for the state.
  constexpr int SETS = local ? 2 : 1;
  auto dz_column = [](int c) { return local ? (uint32_t)(c & 1) * 128u : LT_DZ; };
  auto dz_set = [](int c) { return c % SETS; };
  auto dz_turn = [](int c) { return (uint32_t)((c / SETS) & 1); };
  auto chunk_start = [&](int c) { return s0 + (rev ? nch - 1 - c : c) * LT_T; };

  if (tid == LT_THREADS - 1) {                               // the descriptors' first fetch, under the rest of the set-up
    if (!local) tma_prefetch_desc(mq);
    tma_prefetch_desc(mk);
    tma_prefetch_desc(mv);
    if (!local) tma_prefetch_desc(my);
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.qk_full[i], 1);
      mbar_init(&bars.qk_empty[i], local ? 1 : 2);           // by both issuing warps
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.v_empty[i], local ? 8 : 1);            // by the read-out, which puts its tile there (local: by those who read it)
      mbar_init(&bars.v_read[i], 8);
      mbar_init(&bars.vd_full[i], 8);
      mbar_init(&bars.vd_empty[i], 1);
      mbar_init(&bars.dz_full[i], 1);
      mbar_init(&bars.dz_empty[i], 8);
    }
    mbar_init(&bars.s1_full, 1);
    mbar_init(&bars.p_full, 4);
    mbar_init(&bars.p_empty, 1);
    mbar_init(&bars.o2_full, 1);
    mbar_init(&bars.zb_full, 8);
    mbar_init(&bars.zb_empty, 1);
    mbar_init(&bars.acc_full, 1);
    mbar_init(&bars.acc_empty, 4);
    mbar_fence_init();
    sh.abort_flag = 0;
  }
  if (tid <= LT_T) sh.pw[tid] = tid == 0 ? 1.f : (float)exp(ld * tid);
  if (warp == 0) tmem_alloc(&sh.tmem_slot, 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  // The state is kept times the factor that makes the carried part share the row factor of the other (steep heads and the
  // state-only launch: as it is), so that Zb is one rounding of what the registers hold.
  const float zscale = steep || local ? 1.f : J.s_in / J.s_out * power(pw, rev ? LT_T - 1 - LT_REV_C : LT_FWD_C + 1);
  const uint32_t tbase = sh.tmem_slot;
  volatile int* abort_flag = &sh.abort_flag;
  bool dead = false;

  if (warp >= LT_W_LOAD) {
    regs_dec<LT_R_ISSUE>();
    if (warp == LT_W_LOAD) {
      if (lane == 0) {
        // ---- producer ----
        int done_qk = 0, done_v = 0;                         // loads issued
#pragma unroll 1
        for (int c = 0; c < nch; ++c) {
          const int s = c & 1, t0 = chunk_start(c);
          const uint32_t turn = (uint32_t)(((c >> 1) - 1) & 1);
          uint8_t* st = sm + s * LT_STAGE * BLK;
          if (c >= 2 && !lane_wait(&bars.qk_empty[s], turn, abort_flag, dead)) break;
          mbar_expect_tx(&bars.qk_full[s], (uint32_t)(local ? xblocks : 2 * xblocks) * BLK);
          for (int i = 0; i < xblocks; ++i) {
            if (!local) tma_load_4d(st + i * BLK, mq, &bars.qk_full[s], i * 64, h, t0, b);
            tma_load_4d(st + (2 + i) * BLK, mk, &bars.qk_full[s], i * 64, h, t0, b);
          }
          ++done_qk;
          if (c >= 2 && !lane_wait(&bars.v_empty[s], turn, abort_flag, dead)) break;
          mbar_expect_tx(&bars.v_full[s], (uint32_t)eblocks * BLK);
          for (int i = 0; i < eblocks; ++i) tma_load_4d(st + (4 + i) * BLK, mv, &bars.v_full[s], e0 + i * 64, h, t0, b);
          ++done_v;
        }
        if (dead) {                                          // wind-down: what was issued has to land before the CTA goes
          for (int k = max(0, done_qk - 2); k < done_qk; ++k) mbar_wait(&bars.qk_full[k & 1], (uint32_t)((k >> 1) & 1));
          for (int k = max(0, done_v - 2); k < done_v; ++k) mbar_wait(&bars.v_full[k & 1], (uint32_t)((k >> 1) & 1));
        }
      }
      __syncwarp();
    } else if (warp == LT_W_LOAD + 1) {
      // ---- MMA issuer of the scores and the output: the warp waits, one lane issues ----
      if (!local) {
        const uint32_t id_s = idesc_bf16(128, 128, 0, 0), id_o2 = idesc_bf16(128, 64 * eblocks, 0, 0), id_o = idesc_bf16(128, 64 * eblocks, 0, 1);
        const int kx = (X + 15) / 16;
        const uint32_t zb = lo_k(smem_u32(sZb));
        auto base = [&](int c, int blk) { return smem_u32(sm + ((c & 1) * LT_STAGE + blk) * BLK); };
#pragma unroll 1
        for (int c = 0; c < nch && !dead; ++c) {
          const uint32_t ph = (uint32_t)(c & 1), prev = ph ^ 1u, turn = (uint32_t)((c >> 1) & 1);
          if (!role_wait(&bars.qk_full[c & 1], turn, abort_flag, dead)) break;
          if (c > 0 && !role_wait(&bars.p_empty, prev, abort_flag, dead)) break;      // P of the last chunk, which lies in S1's place
          tc_fence_after_sync();
          const uint32_t aq = lo_k(base(c, 0)), bk = lo_k(base(c, 2));
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
              if (ks < kx) umma_bf16_h(tbase + LT_S1, aq + inc_k(ks), bk + inc_k(ks), id_s, ks > 0 ? 1u : 0u);
            umma_commit(&bars.s1_full);
          }
          if (!role_wait(&bars.zb_full, ph, abort_flag, dead)) break;
          if (c > 0 && !role_wait(&bars.acc_empty, prev, abort_flag, dead)) break;
          tc_fence_after_sync();
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
              if (ks < kx) umma_bf16_h(tbase + LT_O, aq + inc_k(ks), zb + inc_k(ks), id_o2, ks > 0 ? 1u : 0u);
            umma_commit(&bars.zb_empty);
            umma_commit(&bars.qk_empty[c & 1]);              // this warp has read q' and k' of the chunk for the last time
            if (steep) umma_commit(&bars.o2_full);
          }
          if (!role_wait(&bars.p_full, ph, abort_flag, dead)) break;
          if (!role_wait(&bars.v_full[c & 1], turn, abort_flag, dead)) break;
          tc_fence_after_sync();
          const uint32_t bv = lo_mn(base(c, 4));
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
              umma_bf16_ta_h(tbase + LT_O, tbase + LT_P + ks * 8, bv + inc_mn(ks), id_o, 1u);
            if (c == 0 && opens) {
              for (int j = rest_from; j <= rest_to; ++j)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
                  umma_bf16_ta_h(tbase + LT_O, tbase + LT_REST + (j - rest_from) * LT_REST_STRIDE + ks * 8, bv + inc_mn(2 * j + ks), id_o, 1u);
            }
            umma_commit(&bars.p_empty);
            umma_commit(&bars.acc_full);
          }
        }
      }
      __syncwarp();
    } else if (warp == LT_W_LOAD + 2) {
      // ---- MMA issuer of the state update ----
      const uint32_t id_z = idesc_bf16(128, 64 * xblocks, 0, 1);
#pragma unroll 1
      for (int c = 0; c < nch && !dead; ++c) {
        if (!role_wait(&bars.qk_full[c & 1], (uint32_t)((c >> 1) & 1), abort_flag, dead)) break;
        if (c >= SETS && !role_wait(&bars.dz_empty[dz_set(c)], dz_turn(c - SETS), abort_flag, dead)) break;
        const uint32_t bk = lo_mn(smem_u32(sm + ((c & 1) * LT_STAGE + 2) * BLK));
        // quarters of 32 tokens, two sets of parts in turn: the next quarter is split while this one is multiplied
#pragma unroll 1
        for (int k = 0; k < 4; ++k) {
          const int set = k & 1;
          if (!role_wait(&bars.vd_full[set], (uint32_t)((k >> 1) & 1), abort_flag, dead)) break;
          tc_fence_after_sync();
          const uint32_t av = tbase + LT_V + set * 64, bq = bk + (uint32_t)k * (2 * 2048 >> 4);
          if (elect_one()) {
#pragma unroll
            for (int part = 0; part < 3; ++part)
#pragma unroll
              for (int ks = 0; ks < 2; ++ks)
                umma_bf16_ta_h(tbase + dz_column(c), av + part * 16 + ks * 8, bq + inc_mn(ks), id_z, (k > 0 || part > 0 || ks > 0) ? 1u : 0u);
            umma_commit(&bars.vd_empty[set]);
            if (k == 3) {
              umma_commit(&bars.dz_full[dz_set(c)]);
              umma_commit(&bars.qk_empty[c & 1]);
            }
          }
        }
      }
      __syncwarp();
    }
  } else if (warp < LT_W_STATE) {
    regs_dec<LT_R_MASK>();
    if (!local) {
      // ---- decay mask: thread = row t; slab j holds columns 32 j .. 32 j + 31 of S1 and goes to columns 16 j .. of the same place,
      // which slabs up to j / 2 filled: read by then, the slabs being taken in rising order ----
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
        const bool ok = role_wait(&bars.s1_full, (uint32_t)(c & 1), abort_flag, dead);
        if (ok) {
          tc_fence_after_sync();
          float2 f0 = g0, f1 = g1;
#pragma unroll 1
          for (int j = 0; j < 4; ++j) {
            uint32_t o[16];
            if (rev ? j < q : j > q) {                       // wholly beyond the diagonal
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = 0u;
              if (c == 0 && opens && j >= rest_from && j <= rest_to) tmem_st16(tmem_addr(tbase, q * 32, LT_REST + (j - rest_from) * LT_REST_STRIDE), o);
            } else {
              uint32_t r[32];
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
              if (j == q) {                                  // zero beyond the diagonal, whatever the score
#pragma unroll
                for (int i = 0; i < 32; ++i) r[i] = (rev ? i >= lane : i <= lane) ? r[i] : 0u;
              }
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = pack_bf16(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
              if (c == 0 && opens && j >= rest_from && j <= rest_to) {
                const bool keeps = q >= rest_from && q <= rest_to;   // the other rows' scores with these tokens stay as they are
                uint32_t rest[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  float lo, hi;
                  unpack_bf16(o[i], lo, hi);
                  rest[i] = keeps ? pack_bf16(__uint_as_float(r[2 * i]) - lo, __uint_as_float(r[2 * i + 1]) - hi) : 0u;
                }
                tmem_st16(tmem_addr(tbase, q * 32, LT_REST + (j - rest_from) * LT_REST_STRIDE), rest);
              }
            }
            tmem_st16(tmem_addr(tbase, q * 32, LT_P + j * 16), o);
          }
          tmem_st_wait();
        }
        if (steep) {
          // the carried part with a row factor of its own, before P v' is added to it
          if (role_wait(&bars.o2_full, (uint32_t)(c & 1), abort_flag, dead)) {
            tc_fence_after_sync();
            const int Tv = min(LT_T, s1 - chunk_start(c)), t = q * 32 + lane;
            const float fi = t < Tv ? J.s_in / J.s_out * pw[rev ? Tv - 1 - t : t + 1] : 0.f;
#pragma unroll 1
            for (int j = 0; j < 4 * eblocks; ++j) {
              uint32_t r[16];
              tmem_ld16(tmem_addr(tbase, q * 32, LT_O + j * 16), r);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * fi);
              tmem_st16(tmem_addr(tbase, q * 32, LT_O + j * 16), r);
            }
            tmem_st_wait();
          }
        }
        warp_arrive(&bars.p_full, false);
      }
    }
  } else if (warp < LT_W_V) {
    regs_inc<LT_R_STATE>();
    // ---- state: thread = channel e, 64 state columns x in registers ----
    constexpr int ZX = 64;
    const int e = q * 32 + lane, x0 = ((warp - LT_W_STATE) >> 2) * ZX;
    const int64_t head = (int64_t)b * p.H + h;
    float z[ZX];
#pragma unroll
    for (int x = 0; x < ZX; ++x) z[x] = 0.f;
    const bool live = e < E && x0 < X;
    if (!local && live) {
      // the state that enters the segment (joined from the segments' shares, or the carried one)
      const float* src = J.part ? J.part + (head * p.nseg + seg) * p.S : J.z0 ? J.z0 + head * p.S : nullptr;
      if (src) {
        src += x0 * J.xs + (e0 + e) * J.es;
        if (J.xs == 1 && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {       // 64 values side by side; X is a multiple of 8
#pragma unroll
          for (int x = 0; x < ZX; x += 4)
            if (x0 + x < X) {
              const float4 w = *reinterpret_cast<const float4*>(src + x);
              z[x] = w.x; z[x + 1] = w.y; z[x + 2] = w.z; z[x + 3] = w.w;
            }
        } else {
#pragma unroll
          for (int x = 0; x < ZX; ++x) if (x0 + x < X) z[x] = src[x * J.xs];
        }
      }
    }
    if (!local) {
#pragma unroll
      for (int x = 0; x < ZX; ++x) z[x] *= zscale;
    }
    const float a_full = pw[LT_T];
    uint8_t* zrow = sZb + (x0 / 64) * BLK;
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
          for (int j = 0; j < ZX / 8; ++j) {
            float2 y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              y[i] = make_float2(z[8 * j + 2 * i], z[8 * j + 2 * i + 1]);
              if (odd) y[i] = mul2(y[i], make_float2(zs, zs));
            }
            *reinterpret_cast<uint4*>(zrow + sw128_offset(e, j)) =
                make_uint4(pack_bf16(y[0].x, y[0].y), pack_bf16(y[1].x, y[1].y), pack_bf16(y[2].x, y[2].y), pack_bf16(y[3].x, y[3].y));
          }
        }
        warp_arrive(&bars.zb_full, true);
      }
      const float aT = Tv == LT_T ? a_full : pw[Tv];
      if (role_wait(&bars.dz_full[dz_set(c)], dz_turn(c), abort_flag, dead)) {
        tc_fence_after_sync();
#pragma unroll
        for (int j = 0; j < ZX / 32; ++j) {
          uint32_t r[32];
          tmem_ld32(tmem_addr(tbase, q * 32, dz_column(c) + x0 + j * 32), r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 y = fma2(make_float2(aT, aT), make_float2(z[32 * j + i], z[32 * j + i + 1]), f2(r[i], r[i + 1]));
            z[32 * j + i] = y.x;
            z[32 * j + i + 1] = y.y;
          }
        }
      }
      warp_arrive(&bars.dz_empty[dz_set(c)], false);
    }
    float* out = local ? J.part + (head * p.nseg + seg) * p.S : (J.z1 && seg == (rev ? 0 : p.nseg - 1) ? J.z1 + head * p.S : nullptr);
    if (out && live && !dead) {
      out += x0 * J.xs + (e0 + e) * J.es;
      const float unscale = 1.f / zscale;
      if (J.xs == 1 && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
#pragma unroll
        for (int x = 0; x < ZX; x += 4)
          if (x0 + x < X) *reinterpret_cast<float4*>(out + x) = make_float4(z[x] * unscale, z[x + 1] * unscale, z[x + 2] * unscale, z[x + 3] * unscale);
      } else {
#pragma unroll
        for (int x = 0; x < ZX; ++x) if (x0 + x < X) out[x * J.xs] = z[x] * unscale;
      }
    }
  } else if (warp < LT_W_OUT) {
    regs_dec<LT_R_V>();
    // ---- parts of f v' into TMEM (lane = channel, two tokens to a column): a warp takes 32 channels and 16 tokens of each quarter
    // of the chunk, transposed on the way by ldmatrix.  All in packed bfloat16 arithmetic (fma with one rounding): with the factor
    // f = f1 + f2 + f3 in bfloat16 parts (24 bits),
    //   hi = rn(v f1),  m = v f1 - hi and n = rn(v f2) (both exact to eight bits of theirs),  mid = rn(m + n),
    //   lo = rn(v f3 + (m + n - mid) + (v f2 - n)), the rounding error of the sum by five more additions
    // and hi + mid + lo is f v to 2^-25 of it. ----
    const int half = (warp - LT_W_V) >> 2;
    const int mrow = half * 16 + ((lane >> 4) << 3) + (lane & 7);          // this lane's row (token) of the tiles it addresses
    const int mch = q * 32 + ((lane >> 3) & 1) * 8;                        // and first channel; 16 channels further in the second load
    // the factors of a chunk of Tv tokens, by the 256 threads of the role: once for the whole chunks, once for the ragged one
    const float fz = J.s_state * zscale;
    auto factors = [&](int Tv) {
      named_bar_sync(3, 256);                                // the last chunk's factors have been read
      const int i = tid - LT_W_V * 32;
      if (i < LT_T / 2) {
        float y[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const int t = 2 * i + m;
          y[m] = t < Tv ? fz * pw[rev ? t + 1 : Tv - 1 - t] : 0.f;
        }
#pragma unroll
        for (int m = 0; m < 3; ++m) {
          const uint32_t w = pack_bf16(y[0], y[1]);
          sh.fw[m][i] = w;
          float lo, hi;
          unpack_bf16(w, lo, hi);
          y[0] -= lo;
          y[1] -= hi;
        }
      }
      named_bar_sync(3, 256);
    };
    int filled = 0;
#pragma unroll 1
    for (int c = 0; c < nch; ++c) {
      const int Tv = min(LT_T, s1 - chunk_start(c));
      if (Tv != filled) {
        factors(Tv);
        filled = Tv;
      }
      const uint32_t v = smem_u32(sm + ((c & 1) * LT_STAGE + 4) * BLK);
      role_wait(&bars.v_full[c & 1], (uint32_t)((c >> 1) & 1), abort_flag, dead);
#pragma unroll 1
      for (int k = 0; k < 4; ++k) {
        uint32_t w[2][4];
        if (!dead) {
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const int ch = mch + hh * 16;
            ldmatrix_x4_trans(v + (uint32_t)(ch >> 6) * BLK + (uint32_t)(k * 32 + mrow) * 128u + ((((uint32_t)(ch & 63) >> 3) ^ (uint32_t)(lane & 7)) << 4), w[hh]);
          }
        }
        const int set = k & 1;
        if (c > 0 || k > 1) role_wait(&bars.vd_empty[set], (uint32_t)(((k >> 1) + 1) & 1), abort_flag, dead);
        if (!dead) {
          tc_fence_after_sync();
          uint32_t f[2][3];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int m = 0; m < 3; ++m) f[i][m] = sh.fw[m][k * 16 + half * 8 + i * 4 + (lane & 3)];
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            uint32_t t[3][4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {                    // r: channels 0-7 | 8-15, tokens 0-7; the same, tokens 8-15
              const uint32_t x = w[hh][r], *ff = f[r >> 1];
              const uint32_t h1 = bf2_mul(x, ff[0]), m = bf2_fma(x, ff[0], bf2_neg(h1)), nn = bf2_mul(x, ff[1]);
              const uint32_t s2 = bf2_add(m, nn), bb = bf2_add(s2, bf2_neg(m));
              const uint32_t err = bf2_add(bf2_add(m, bf2_neg(bf2_add(s2, bf2_neg(bb)))), bf2_add(nn, bf2_neg(bb)));
              t[0][r] = h1;
              t[1][r] = s2;
              t[2][r] = bf2_fma(x, ff[2], bf2_add(err, bf2_fma(x, ff[1], bf2_neg(nn))));
            }
#pragma unroll
            for (int m = 0; m < 3; ++m) tmem_st_16x128b_x2(tmem_addr(tbase, q * 32 + hh * 16, LT_V + set * 64 + m * 16 + half * 8), t[m]);
          }
          tmem_st_wait();
        }
        if (k == 3) {
          __syncwarp();                                      // every lane has its part of v'
          if (lane == 0) mbar_arrive(local ? &bars.v_empty[c & 1] : &bars.v_read[c & 1]);
        }
        warp_arrive(&bars.vd_full[set], false);
      }
    }
  } else {
    regs_dec<LT_R_OUT>();
    if (!local) {
      // ---- read-out: thread = row t; the tile leaves from the place of the v' tile ----
      const int t = q * 32 + lane;
      const float fo = J.s_out * (steep ? 1.f : power(pw, rev ? LT_REV_C - t : t - LT_FWD_C));   // row factor
#pragma unroll 1
      for (int c = 0; c < nch; ++c) {
        const uint32_t turn = (uint32_t)((c >> 1) & 1);
        uint8_t* out = sm + ((c & 1) * LT_STAGE + 4) * BLK;
        bool ok = role_wait(&bars.acc_full, (uint32_t)(c & 1), abort_flag, dead);             // the product has read the v' tile ...
        ok = role_wait(&bars.v_read[c & 1], turn, abort_flag, dead) && ok;                    // ... and so has the splitting
        if (ok) {
          tc_fence_after_sync();
#pragma unroll 1
          for (int j = 0; j < 2 * eblocks; ++j) {
            uint32_t r[32];
            tmem_ld32(tmem_addr(tbase, q * 32, LT_O + j * 32), r);
            tmem_ld_wait();
            uint8_t* dst = out + (j >> 1) * BLK;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t o[4];
#pragma unroll
              for (int m = 0; m < 4; ++m) {
                const float2 y = mul2(make_float2(fo, fo), f2(r[8 * i + 2 * m], r[8 * i + 2 * m + 1]));
                o[m] = pack_bf16(y.x, y.y);
              }
              *reinterpret_cast<uint4*>(dst + sw128_offset(t, 4 * (j & 1) + i)) = make_uint4(o[0], o[1], o[2], o[3]);
            }
          }
        }
        warp_arrive(&bars.acc_empty, true);
        named_bar_sync(2, 128);
        if (tid == LT_W_OUT * 32) {
          if (ok) {
            for (int i = 0; i < eblocks; ++i) tma_store_4d(my, out + i * BLK, e0 + i * 64, h, chunk_start(c), b);
            bulk_commit_group();
            bulk_wait_group_read<0>();
          }
          mbar_arrive(&bars.v_empty[c & 1]);
        }
      }
      if (tid == LT_W_OUT * 32) bulk_wait_group<0>();
    }
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
  // tile index: channel half, then head (neighbours in memory), then segment, batch, and the job last: CTAs that run side by side then share
  // their code (jobs side by side would share q, k, v and dy in L2, but were 17 % slower in the backward pass)
  int64_t id = blockIdx.x;
  const int et = (int)(id % p.ne);
  id /= p.ne;
  const int h = (int)(id % p.H);
  id /= p.H;
  const int seg = (int)(id % p.nseg);
  id /= p.nseg;
  const int b = (int)(id % p.B), jb = (int)(id / p.B);
  const int rev = p.job[jb].reverse;
  if (et * 64 >= p.job[jb].E) return;
  if (local && seg == (rev ? 0 : p.nseg - 1)) return;        // nobody reads the last segment's share
  uint8_t* sm = align1024(smem_raw);
  const double ld = (double)p.log_decay[h];
  const bool steep = !(fabs(ld) <= 0.346573);                // a at least 2^{-1/2}
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

// Row factors and the kept state hold scale (or its reciprocal) times a^64 and more, 2^-33 at the least: a scale beyond 2^+-40 could leave
// the range of float32 with them, and goes to the float32 kernels, whose factors are at most 1.
bool la_tc_serves(const LaArgs& a, bool bwd, int dtype) {
  if (dtype != BF16 || a.Dk % 8 || a.Dv % 8 || a.Dk > 128 || a.Dv > 128) return false;
  if (!(fabsf(a.scale) >= 0x1p-40f && fabsf(a.scale) <= 0x1p40f)) return false;
  bool ok = tc_operand(a.q, a.q_bs, a.q_ls, a.q_hs) && tc_operand(a.k, a.k_bs, a.k_ls, a.k_hs) && tc_operand(a.v, a.v_bs, a.v_ls, a.v_hs);
  if (!bwd) return ok && tc_operand(a.y, a.y_bs, a.y_ls, a.y_hs);
  return ok && tc_operand(a.dy, a.dy_bs, a.dy_ls, a.dy_hs) && tc_operand(a.dq, a.dq_bs, a.dq_ls, a.dq_hs) &&
         tc_operand(a.dk, a.dk_bs, a.dk_ls, a.dk_hs) && tc_operand(a.dv, a.dv_bs, a.dv_ls, a.dv_hs);
}

// How a call is spread over the SMs: segments of the sequence, and for heads wider than 64 channels one CTA a head or one for each
// half of its channels (`ne`).  A half costs three quarters of a whole chunk step (scores and the products of the state are made for
// either half), but needs no first launch; so it is taken where it fills SMs that segments would fill at a higher price.  Heads of
// 128 x 128, whole heads against halves: [1, 131, 16] 20 us and 16, [1, 2048, 16] 53 and 47; [8, 4096, 16] 113 and 183, [1, 65536, 16]
// 341 and 594.  Prologue and state cost about three steps a CTA, the joining launch five (with two: [2, 1000, 8] 38 us instead of 31).
static int tc_split(const LaArgs& a, bool bwd, int* seg_len, int* ne) {
  const int64_t heads = (int64_t)a.B * a.H;
  const int wide = (a.Dv > 64) + (bwd ? 2 * (a.Dk > 64) : 0), jobs = bwd ? 3 : 1;
  double whole = 0., halves = 0.;
  const int n1 = la_segments(heads * jobs, a.L, LT_T, 3., 5., seg_len, &whole);
  *ne = 1;
  if (wide == 0) return n1;
  int len2 = 0;
  const int n2 = la_segments(heads * (jobs + wide), a.L, LT_T, 3., 5., &len2, &halves);
  if (0.75 * halves >= 0.95 * whole) return n1;
  *ne = 2;
  *seg_len = len2;
  return n2;
}

int la_tc_segments(const LaArgs& a, bool bwd, int* seg_len) {
  int ne;
  return tc_split(a, bwd, seg_len, &ne);
}

// [B, L, H, D] with any strides as 128-token boxes of 64 channels of one head; what lies outside reads as zero and is not written
static int tc_map(CUtensorMap* m, const void* base, int D, int64_t bs, int64_t ls, int64_t hs, const LaPlan& p) {
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)p.H, (uint64_t)p.L, (uint64_t)p.B};
  const uint64_t str[3] = {(uint64_t)hs * 2, (uint64_t)ls * 2, (uint64_t)bs * 2};
  const uint32_t box[4] = {64, 1, LT_T, 1};
  return make_tensor_map_bf16(m, base, 4, dims, str, box);
}

int la_tc_launch(const LaArgs& a, bool bwd, cudaStream_t st) {
  int seg_len = 0, ne = 1, rc;
  const int nseg = tc_split(a, bwd, &seg_len, &ne);
  ORBIT_CHECK_CUDA(cudaFuncSetAttribute(la_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LT_SMEM));
  for (int local = nseg > 1 ? 1 : 0; local >= 0; --local) {
    LaTcArgs t;
    if ((rc = la_plan(a, bwd, nseg, seg_len, local != 0, &t.p)) != OK) return rc;
    for (int i = 0; i < t.p.njobs; ++i) {
      const LaJob& j = t.p.job[i];
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
    if (local && (rc = la_join(t.p, st)) != OK) return rc;
  }
  return OK;
}

}  // namespace orbit
