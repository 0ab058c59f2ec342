// Argument block of the linear-attention entry points inside the library (the public one, under this namespace).
#pragma once
#include "../../include/orbit_b200.h"

namespace orbit {
using LaArgs = orbit_la_args;

// One pass over the sequence as the kernels see it.  Every direction of linear attention is the same recurrence with its
// operands in other roles:
//   Z_i = a Z_{i-1} + sz k'_i (x) v'_i,    out_i[e] = so sum_{j<=i} a^{i-j} (q'_i . k'_j) v'_j[e] + si f_i sum_x q'_i[x] Zin[x, e]
//   forward  y  : q, k, v    forwards in time     state Z = S^T
//   backward dq : dy, v, k   forwards             state Z = S
//   backward dk : v, dy, q   backwards            state Z = gradient of S
//   backward dv : k, q, dy   backwards            state Z = its transpose
// X is the contracted width (of q' and k'), E the width of v' and of the output.  The state lives in memory as [B, H, Dv, Dk]
// in every role; (xs, es) are the strides of its x and e axes.
struct LaJob {
  const void *q, *k, *v;
  int64_t q_bs, q_ls, q_hs, k_bs, k_ls, k_hs, v_bs, v_ls, v_hs;
  void* y;
  int64_t y_bs, y_ls, y_hs;
  int X, E, reverse;
  float s_out, s_in, s_state;
  const float* z0;    // state before the sequence (reverse: gradient of the state after it) or null
  float* z1;          // state after it (reverse: gradient of the state before it) or null
  float* part;        // [B*H][nseg][Dv*Dk]: what each segment alone adds to the state, then (joined) the state that enters each
                      // segment; null when nseg == 1
  int64_t xs, es;
};
struct LaPlan {
  int B, L, H, S;     // S = Dk * Dv, elements of a head's state
  int njobs, nseg, seg_len, ne;   // ne: CTAs that share a head's channels (tensor-core launch)
  const float* log_decay;
  int* status;
  LaJob job[3];
};

// the jobs of one direction (local: the two state-only passes that feed `part`)
int la_plan(const LaArgs& a, bool bwd, int nseg, int seg_len, bool local, LaPlan* p);
// the launch between the two: shares of the segments -> states that enter them, in place, for the jobs of the state-only plan
int la_join(const LaPlan& p, cudaStream_t st);
// segments the sequence is split into so that `units` CTAs per segment fill the GPU (chunk = tokens of one tile)
int la_segments(int64_t units, int L, int chunk, double setup, double join, int* seg_len, double* cost = nullptr);

bool la_tc_serves(const LaArgs& a, bool bwd, int dtype);
int la_tc_launch(const LaArgs& a, bool bwd, cudaStream_t st);
int la_tc_segments(const LaArgs& a, bool bwd, int* seg_len);
}  // namespace orbit
