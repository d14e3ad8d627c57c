// Shared by the token-by-token and the chunked state space scans (ssm.hip, ssm_chunk.hip).
//
// The state space recurrence of head h (S is [head_dim, d_state], f32) is
//   S = exp(d_t A) S + d_t x_t B_t^T,   y_t = S C_t + D x_t
// so a piece of rows t0 .. t1 maps its start state S to decay S + E, with
//   decay = exp(A sum d_t)   and   E = sum_t exp(A sum_{u > t} d_u) d_t x_t B_t^T
// both independent of S. A long sequence is cut into pieces that run at once: one launch forms every
// piece's E and decay (all pieces but a sequence's last), one joins them in order into the pieces'
// start states, one runs the pieces from those. A sequence of one piece has no place in the workspace.
#pragma once

#include "packed.hpp"
#include "ssm_plan.hpp"

namespace ema {

enum SsmPhase {
  kSsmWhole = 0,   // a piece is a sequence: start from the pool, write y and the pool
  kSsmEnds = 1,    // E and decay of each piece that is not its sequence's last
  kSsmPieces = 2,  // from the joined start states: y, and the pool from the last piece
};

#if defined(__HIPCC__)
// softplus(r) = max(r, 0) + log(1 + u) with u = e^-|r| at most 1, and log(1 + u) = 2 atanh(u / (2 + u))
// by the series of atanh: the argument is at most 1/3, so eight terms leave 2^-29 of it.
__device__ __forceinline__ float softplus_(float r) {
  const float u = expf(-fabsf(r));
  const float s = u * __builtin_amdgcn_rcpf(2.0f + u), q = s * s;
  float p = 1.0f / 15;
  p = fmaf(p, q, 1.0f / 13);
  p = fmaf(p, q, 1.0f / 11);
  p = fmaf(p, q, 1.0f / 9);
  p = fmaf(p, q, 1.0f / 7);
  p = fmaf(p, q, 1.0f / 5);
  p = fmaf(p, q, 1.0f / 3);
  p = fmaf(p, q, 1.0f);
  return fmaf(2.0f * s, p, r > 0.0f ? r : 0.0f);
}
// The step of raw value r (dt + bias): softplus, then the limits.
__device__ __forceinline__ float ssm_step(float r, const SsmArgs& a) {
  const float sp = softplus_(r);
  r = a.softplus ? sp : r;  // (no branch)
  r = r < a.dt_min ? a.dt_min : r;  // (NaN stays)
  return r > a.dt_max ? a.dt_max : r;
}
#endif

// The workspace's order of a head's state: token by token [head_dim][d_state]; chunks: accumulator tiles
// of 16 columns (of head_dim) by 16 of d_state, the four values that a lane holds after each other.
// Values 4 v .. of it are the pool's from this place on.
EMA_HD int ssm_carry_element(int v, int d_state) {
  const int lane = v & 63, T = (v >> 6) % (d_state / 16), col = (v >> 6) / (d_state / 16);
  const int p = 32 * (col >> 1) + 8 * ((lane & 15) >> 2) + 4 * (col & 1) + (lane & 3);
  return p * d_state + 32 * (T >> 1) + 8 * (lane >> 4) + 4 * (T & 1);
}
hipError_t launch_ssm_chunk(hipStream_t s, const SsmArgs& a, int64_t pieces, SsmPhase phase);

}  // namespace ema
