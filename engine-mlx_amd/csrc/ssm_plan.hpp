// How a state space scan runs: on which kernels, and whether and where its sequences are cut in time. Host
// rules on sizes, free of HIP, so that the CPU test (tests/cpp/test_ssm_plan.cpp) checks the definitions
// that the calls use.
#pragma once

#include <stdint.h>

#include "packed.hpp"

namespace ema {

// Pieces of how many rows, on which kernels.
struct SsmPlan {
  int piece;        // rows of a piece, 0: no cut
  int64_t pieces;   // piece numbers
  int64_t places;   // states in the workspace
  bool chunks;      // on the matrix cores
  uint64_t bytes;   // of the workspace
};

// Chunked scan on the matrix cores (bf16): the shapes it takes, and the workgroups of a piece.
constexpr int kSsmChunk = 32;  // rows of a chunk
constexpr int kSsmCols = 32;   // columns of x of a wave
inline bool ssm_chunk_shape(int head_dim, int d_state) {
  return head_dim % kSsmCols == 0 && (d_state == 64 || d_state == 128 || d_state == 256);
}
inline int ssm_chunk_workgroups(int heads, int head_dim, int groups) {
  return groups * ((heads / groups * (head_dim / kSsmCols) + 3) / 4);
}

// Rules of a form: chunks, or token by token.
struct SsmCut {
  int64_t wgs;      // workgroups of a piece (token by token: of R = 4)
  int64_t fill;     // workgroups that occupy the chip: two a CU, or four
  int step, least;  // pieces are a multiple of step rows, at least `least`
  int by_even, by;  // cut where the longest sequence has 0.1 (by_even E + by) rows and more, E = rows * wgs / fill
};
// Cut where the sequences' heads leave much of the chip idle: into pieces that fill it, of E rows if there are no
// shorter ones. Chunks, 64 heads of 64, d_state 128: a whole sequence takes 6 us and 0.082 us a row of the longest,
// cut ones 25 us and 0.0123 us a row of all (ends, joining, pieces; 0.197 E), so that the longest has to be 240 rows
// and 2.5 E: 4 x 2048 rows 121 us cut, 173 whole, 4 x 1024 77 and 90, 6 x 1024 119 and 92, 5 x 1638 146 and 143, 512
// rows 34 and 47, 320 29 and 32, 256 29 and 26. The state's size moves both sides: d_state 64, 32 heads 210 rows and
// 3.7 E (384 rows 23 cut, 27 whole, 4096 45 and 234), d_state 256, 16 heads of 128 240 and 3.3 E (384 46 and 63,
// 4 x 2048 146 and 300). Token by token (f32, d_state 128): whole 0.2 us a row of the longest and 0.72 E, cut 20 us
// and 1.66 E: 24 heads of 64, 2048 rows 112 us cut, 414 whole, 128 rows 24 and 25, 8 x 300 120 and 109; 64
// heads, 8192 rows 785 and 1994, 4 x 2048 800 and 765.
inline SsmCut ssm_cut(bool chunks, int heads, int head_dim, int groups, int cus) {
  if (chunks) return SsmCut{ssm_chunk_workgroups(heads, head_dim, groups), 2 * cus, kSsmChunk, 4 * kSsmChunk, 25, 2400};
  return SsmCut{heads * (int64_t)((head_dim + 63) / 64), 4 * cus, 16, 32, 47, 1000};
}
inline uint64_t ssm_places_bytes(int64_t places, int heads, int head_dim, int d_state) {
  return (uint64_t)places * heads * ((uint64_t)head_dim * d_state + 4) * 4;
}

// ws_bytes: the workspace that there is; vectors: bf16 rows that allow 16-byte accesses.
inline SsmPlan plan_ssm(int batch, int n_rows, int max_rows, int heads, int head_dim, int d_state, int groups,
                        bool vectors, int cus, uint64_t ws_bytes) {
  SsmPlan p{};
  p.chunks = vectors && max_rows >= 32 && ssm_chunk_shape(head_dim, d_state);
  p.pieces = batch;
  const SsmCut c = ssm_cut(p.chunks, heads, head_dim, groups, cus);
  const int64_t even = (n_rows * c.wgs + c.fill - 1) / c.fill;
  if ((int64_t)max_rows * 10 < even * c.by_even + c.by) return p;
  int64_t piece = even < c.least ? c.least : (even + c.step - 1) / c.step * c.step;
  for (; piece < max_rows; piece *= 2) {
    const int64_t pieces = packed_pieces(n_rows, batch, (int)piece), places = packed_places(n_rows, batch, (int)piece);
    const uint64_t bytes = ssm_places_bytes(places, heads, head_dim, d_state);
    if (bytes > ws_bytes) continue;
    p.piece = (int)piece;
    p.pieces = pieces;
    p.places = places;
    p.bytes = bytes;
    break;
  }
  return p;
}

// The workspace that every call of at most these sequences, rows and rows of a sequence can use, in either form.
// With n rows a call's pieces are of max(E, least) rows and more: at most fill / wgs of them fit its rows, or
// n_rows / least. Calls are cut at all where one that is a single sequence of max_rows is (E not rounded up:
// the condition is linear in the rows, and does not hold for none).
inline uint64_t ssm_workspace_bytes(int batch, int n_rows, int max_rows, int heads, int head_dim, int d_state, int groups,
                                    bool bf16, int cus) {
  uint64_t most = 0;
  if (max_rows > n_rows) max_rows = n_rows;
  for (int chunks = 0; chunks < 2; ++chunks) {
    if (chunks && !(bf16 && ssm_chunk_shape(head_dim, d_state))) continue;
    const SsmCut c = ssm_cut(chunks, heads, head_dim, groups, cus);
    if ((int64_t)max_rows * 10 * c.fill < max_rows * c.wgs * c.by_even + c.by * c.fill) continue;
    const int64_t q = n_rows / c.least < c.fill / c.wgs ? n_rows / c.least : c.fill / c.wgs;
    const uint64_t bytes = ssm_places_bytes(q + (batch < q ? batch : q), heads, head_dim, d_state);
    if (bytes > most) most = bytes;
  }
  return most;
}

}  // namespace ema
