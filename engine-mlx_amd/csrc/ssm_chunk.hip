// Selective state space scan in chunks of 32 rows on the matrix cores, bf16 activations.
//
// With a_t = d_t A and sums over rows of the chunk, a chunk that starts from the state H gives
//   y_t = e^(a_0 + .. + a_t) H C_t + sum_{s <= t} M[t][s] x_s + D x_t,
//   M[t][s] = (C_t . B_s) e^(a_(s+1) + .. + a_t) d_s,
//   H'  = e^(a_0 + .. + a_31) H + sum_s (d_s e^(a_(s+1) + .. + a_31) x_s) B_s^T,
// so C B^T is the same for all heads of a group, and the rest is products with 32-row operands.
//
// A workgroup of four waves takes 128 columns of x (two heads of 64, one of 128, ...) of one group,
// a wave 32 of them: its H^T [d_state, 32] stays in 32-bit accumulators over the rows of the piece.
// All products are 16x16x32 in forms that chain without moving data between lanes:
//   C B^T as [s, t]          A = B rows,       B = C rows (columns t)
//   y^T [p, t]              A = H (the accumulators, in two bf16 parts) and x^T, B = C and M
//   H^T [n, p]              A = B^T,           B = x^T scaled
// A pair of 16x16 accumulator tiles holds, in lane group c, rows 4 c + (0..3) of both tiles. The rows of
// the state's tiles are numbered so that these are d_state 8 c + (0..7) of a 32-wide step (B^T's columns
// are read in that order): rows of C are then read whole. Columns of x are numbered in the same way
// over the wave's two tiles, so that a lane holds 8 neighbours of a row of y. M's are rows 4 c + (0..3) and 16 + 4 c +
// (0..3); x^T and B^T are read from LDS in the same order of rows, by the transposing read. The
// decays of M are products of factors at most 1 (A <= 0): from s to the end of its 16-row tile (g), and
// from t's tile's start to t (f); inside the tiles on the diagonal each is of a sum over its own rows,
// s + 1 to t (a difference of two long sums keeps no more than their last bit: behind rows that decay
// by 2^-100 each it was up to 2^-13 off).
//
// Operands of the products: x, B and C are exact in bf16. H and M enter y in two bf16 parts, 16 bits
// together: off by at most 2^-16 of the term, 2^-8 of what y's own rounding may take (in one part y was 0.0022
// off in place of 0.0017, and 0.0027 from the same sums in 32 bits; now 0.00006). D x is added in 32 bits. The state
// itself takes the scaled x as three bf16 parts, 24 bits together (two left it 1.5e-6 off, three 5e-8),
// products and sums in 32 bits; the ends of pieces as well, since a head that hardly decays hands on all of them.
//
// A value of x that is not finite would reach rows before it through M's zeros (0 times infinity):
// chunks with such values (a dot product with zeros finds them while they are staged) take those
// columns' sums without them and put NaN into the rows from the value on.
//
// Chunks of 32 rows and not of 64: per row they cost a third more vector instructions for the state
// (its decay and its rounding come twice as often), but 64 rows need more registers than two
// workgroups a CU leave, and spilled the loads under way (131 us against 74 at the time).
//
// Bound by issue and waits: a chunk of a wave is 100 products (16 cycles each) and about 680 vector
// instructions (by the counters; 48 and 190 in the ends), 4300 cycles a wave and 8600 for the two of a SIMD
// if none overlap, of the 5.2 us that a chunk takes. 8192 rows of 64 heads of 64, d_state 128, 8 groups: ends
// 33, joining 13, pieces 84 us, together 119 us, 1.5 TB/s of what has to move, 0.18 PFLOP/s of the recurrence's
// operations. With H and M in one bf16 part, D among M and the ends in two parts it was 30, 13 and 64, at
// y 0.0022 off and the state 16 bits. No gain at that time: products interleaved with vector instructions by
// scheduling groups, the state's decay kept as a factor (66), y stored a chunk later (67), one column tile a
// wave in workgroups of eight waves (104, spilled).
#include <type_traits>

#include "ssm.hpp"

namespace ema {
namespace {

constexpr int kQ = kSsmChunk, kCols = kSsmCols;
constexpr int kXW = 4 * kCols;
constexpr int kThreads = 256;

typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Per-head values of a chunk (floats): index by row unless said otherwise.
struct Dec {
  static constexpr int kW = 0;       // d times the decay from behind the row to the chunk's end
  static constexpr int kAll = 32;    // decay over the chunk; its log2 at 33
  static constexpr int kEnds = 36;   // (that is all that the pieces' ends need)
  static constexpr int kL = 36;      // log2 decay of the row
  static constexpr int kStep = 68;   // d
  static constexpr int kF = 100;     // decay from the tile's start: 2^kCum
  static constexpr int kE = 132;     // decay from the chunk's start
  static constexpr int kG = 164;     // d times the decay from behind the row to its tile's end
  static constexpr int kQ = 196;     // [tile][4][16]: sum of log2 decays from row 4 i + 4 of the tile to the row, included
  static constexpr int kFloats = 324;
};

// Row pitch and swizzle of the LDS tiles of W-wide rows: 16-byte piece q of row r lies at piece
// q ^ x(r), so that 16 rows at one piece, and 8 rows at two neighbouring ones, are in distinct banks.
template <int W>
__device__ __forceinline__ int swizzle(int r) {
  return W == 64 ? ((r >> 1) & 3) * 2 | ((r >> 3) & 1) : (r & 7) * 2 | ((r >> 3) & 1);
}
template <int W>
__device__ __forceinline__ int tile_at(int r, int q) {  // bytes
  return r * (W * 2) + ((q ^ swizzle<W>(r)) << 4);
}

// Two values in two bf16 parts: their own bits, and those of what is left.
__device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(a, b);
  lo = pack_bf16x2(a - bf16_lo(hi), b - bf16_hi(hi));
}
__device__ __forceinline__ bf16x8 join(u32x2 lo, u32x2 hi) { return as_bf16x8(u32x4{lo[0], lo[1], hi[0], hi[1]}); }
__device__ __forceinline__ u32x2 read_tr(const uint8_t* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
}
template <int CTRL>
__device__ __forceinline__ float dpp_shift(float v) {  // 0 where there is no such lane in the row of 16
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_value(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }

// Decays of two heads' 32 rows, a row a lane (lanes 32..63: the second head; dec is the lane's
// head's). `raw` is dt + bias; rows from n on take no step.
template <bool kOutputs>
__device__ __forceinline__ void chunk_decays(float raw, int n, float A2, const SsmArgs& a, float* dec) {
  const int lane = threadIdx.x & 63, row = lane & 31;
  const float d = row < n ? ssm_step(raw, a) : 0.f;
  // log2 of the row's decay; below 2^-150 it is 0 either way, and sums stay finite (NaN stays NaN)
  float l = d * A2;
  l = row >= n ? 0.f : (l < -150.f ? -150.f : l);
  float down = l;  // sum over the 16-row tile from the row on
  down += dpp_shift<0x101>(down);
  down += dpp_shift<0x102>(down);
  down += dpp_shift<0x104>(down);
  down += dpp_shift<0x108>(down);
  const float behind = dpp_shift<0x101>(down);  // from behind the row to its tile's end
  const bool second = lane >= 32, tile1 = row >= 16;
  const float t0 = second ? lane_value(down, 32) : lane_value(down, 0), t1 = second ? lane_value(down, 48) : lane_value(down, 16);
  dec[Dec::kW + row] = d * exp2_(behind + (tile1 ? 0.f : t1));
  dec[Dec::kAll] = exp2_(t0 + t1);  // (every lane the same)
  dec[Dec::kAll + 1] = t0 + t1;
  if constexpr (kOutputs) {
    float up = l;  // up to the row
    up += dpp_shift<0x111>(up);
    up += dpp_shift<0x112>(up);
    up += dpp_shift<0x114>(up);
    up += dpp_shift<0x118>(up);
    // from the second, third and fourth four rows of the tile on
    const int r16 = row & 15;
    float q[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      q[i] = r16 >= 4 * i + 4 ? l : 0.f;
      q[i] += dpp_shift<0x111>(q[i]);
      q[i] += dpp_shift<0x112>(q[i]);
      if (i < 2) q[i] += dpp_shift<0x114>(q[i]);
      if (i < 1) q[i] += dpp_shift<0x118>(q[i]);
      dec[Dec::kQ + 64 * (row >> 4) + 16 * i + r16] = q[i];
    }
    dec[Dec::kQ + 64 * (row >> 4) + 48 + r16] = 0.f;
    dec[Dec::kL + row] = l;
    dec[Dec::kStep + row] = d;
    dec[Dec::kF + row] = exp2_(up);
    dec[Dec::kE + row] = exp2_(up + (tile1 ? t0 : 0.f));
    dec[Dec::kG + row] = d * exp2_(behind);
  }
}

// LDS (bytes): B, x and (for outputs) C, twice; the heads' decays of two groups of chunks; the flags of
// three chunks, whether they have values that are not finite.
template <int N, int HEADS, bool kOutputs>
struct Lds {
  // chunks whose decays are formed at once, by a wave each (two heads a wave)
  static constexpr int kGroup = HEADS == 4 ? 2 : 4;
  static constexpr int kX = kQ * N * 2;
  static constexpr int kC = kX + kQ * kXW * 2;
  static constexpr int kBuf = kC + (kOutputs ? kQ * N * 2 : 0);
  static constexpr int kDec = 2 * kBuf;
  static constexpr int kDecHead = kOutputs ? Dec::kFloats : Dec::kEnds;
  static constexpr int kFlag = kDec + 2 * kGroup * HEADS * kDecHead * 4;
  static constexpr int kBytes = kFlag + 16;
};

struct ChunkGrid {
  int units;       // 32-column pieces of a group: heads per group * head_dim / 32
  int per_head;    // head_dim / 32
  int wgs;         // workgroups of a (piece, group)
  int64_t pairs;   // (piece, group)
};

template <int N, int HEADS, int PHASE>
__global__ __launch_bounds__(kThreads, N == 256 ? 1 : 2) void ssm_chunk_kernel(SsmArgs a, ChunkGrid gr) {
  constexpr bool kOutputs = PHASE != kSsmEnds;
  typedef Lds<N, HEADS, kOutputs> L;
  constexpr int KS = N / 32;   // 32-wide steps over d_state
  constexpr int NT = N / 16;   // 16-row tiles of it
  constexpr int kParts = 3;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];

  // the workgroups of a (piece, group) read the same B and C: on one XCD (blocks go to the XCDs in turn)
  const uint32_t xcd = blockIdx.x & 7, k8 = blockIdx.x >> 3;
  const int wg = (int)(k8 % (uint32_t)gr.wgs);
  const int64_t pair = xcd + 8 * (int64_t)(k8 / (uint32_t)gr.wgs);
  if (pair >= gr.pairs) return;
  const int grp = (int)((uint32_t)pair % (uint32_t)a.groups), index = (int)((uint32_t)pair / (uint32_t)a.groups);
  const Piece pc = packed_piece(a.starts, a.batch, a.n_rows, a.T, a.piece, index);
  if (pc.n == 0) return;
  const bool last = pc.row + pc.n == pc.begin + pc.all;
  if (PHASE == kSsmEnds && last) return;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, c4 = lane >> 4;
  const int P = a.head_dim;
  const int head0 = grp * (a.heads / a.groups);       // of the group
  const int unit0 = wg * 4;
  const int first_head = unit0 / gr.per_head;         // of the workgroup, in the group
  const int last_unit = unit0 + 3 < gr.units ? unit0 + 3 : gr.units - 1;
  const int n_heads = last_unit / gr.per_head - first_head + 1;
  const bool idle = unit0 + wave > last_unit;
  const int unit = idle ? last_unit : unit0 + wave;
  const int hh = unit / gr.per_head - first_head;     // this wave's head among the workgroup's
  const int head = head0 + first_head + hh;
  const int p0 = (unit % gr.per_head) * kCols;        // its first column of the head
  const int slot = packed_slot(a.slots, pc.b, a.n_slots);
  float* const pool = a.state + ((int64_t)slot * a.heads + head) * P * N;
  // (the workspace holds a wave's state in the order of its accumulators: ssm_carry_element)
  const int64_t place = packed_first_place(pc.begin, pc.b, a.piece) + pc.index - pc.first;  // (of a longer sequence)
  float* const carry = a.carry + (place * a.heads + head) * P * N + p0 * N + 4 * lane;
  const int st_at = (p0 + 8 * (l16 >> 2) + (l16 & 3)) * N + 8 * c4;

  float* const decs = (float*)(lds + L::kDec);
  int* const flags = (int*)(lds + L::kFlag);

  // ---- state: h[ct][T] holds n = 32 (T / 2) + 8 c4 + 4 (T % 2) + i of column l16 of tile ct, which is
  // p0 + 8 (l16 / 4) + 4 ct + l16 % 4
  f32x4 h[2][NT];
  {
    // a sequence of one piece starts from the pool; pieces of a longer one never read what its last
    // piece writes there
    const float* from = nullptr;
    int step_ct = 4 * N, step_T = 32, step_u = 4;
    if (PHASE == kSsmPieces && pc.all > a.piece) {
      from = carry;
      step_ct = NT * 256;
      step_T = 512;
      step_u = 256;
    } else if (kOutputs && slot >= 0 && packed_continues(a.offsets, pc.b)) {
      from = pool + st_at;
    }
#pragma unroll
    for (int ct = 0; ct < 2; ++ct)
#pragma unroll
      for (int T = 0; T < NT; ++T) h[ct][T] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (from)
#pragma unroll
      for (int ct = 0; ct < 2; ++ct)
#pragma unroll
        for (int T = 0; T < NT; ++T) h[ct][T] = *(const f32x4*)(from + (ct * step_ct + (T >> 1) * step_T + (T & 1) * step_u));
  }

  // ---- staging: 16-byte pieces of rows, in registers from one chunk to the next
  constexpr int kRowB = N / 8;                     // pieces of a B or C row
  constexpr int kIn = kQ * kRowB / kThreads;       // pieces of B (or C) a thread
  constexpr int kInX = kQ * 16 / kThreads;
  u32x4 rb[kIn], rc[kIn], rx[kInX];
  // rows within a chunk are 32-bit offsets from a uniform base (ld* < 2^23)
  const uint8_t* const bp = (const uint8_t*)((const uint16_t*)a.b + (int64_t)pc.row * a.ldb + grp * N);
  const uint8_t* const cp = (const uint8_t*)((const uint16_t*)a.c + (int64_t)pc.row * a.ldc + grp * N);
  const uint8_t* const xp = (const uint8_t*)((const uint16_t*)a.x + (int64_t)pc.row * a.ldx + (int64_t)head0 * P + unit0 * kCols);
  const uint32_t ldb2 = (uint32_t)a.ldb * 2, ldc2 = (uint32_t)a.ldc * 2, ldx2 = (uint32_t)a.ldx * 2;
  const int x_pieces = (last_unit - unit0 + 1) * (kCols / 8);
  // rows behind the piece are its last row again: what they would add has step 0 (and columns of no
  // unit the last one's again: their wave is idle)
  auto load = [&](int t0) __attribute__((always_inline)) {
    const uint32_t end = (uint32_t)(pc.n - t0 - 1);
    const uint8_t* const b0 = bp + (int64_t)t0 * ldb2;
    const uint8_t* const c0 = cp + (int64_t)t0 * ldc2;
    const uint8_t* const x0 = xp + (int64_t)t0 * ldx2;
#pragma unroll
    for (int i = 0; i < kIn; ++i) {
      const uint32_t id = i * kThreads + tid, r = id / kRowB, q = id % kRowB;
      const uint32_t row = r < end ? r : end;
      rb[i] = *(const u32x4*)(b0 + (row * ldb2 + 16 * q));
      if constexpr (kOutputs) rc[i] = *(const u32x4*)(c0 + (row * ldc2 + 16 * q));
    }
#pragma unroll
    for (int i = 0; i < kInX; ++i) {
      const uint32_t id = i * kThreads + tid, r = id >> 4, q = id & 15;
      rx[i] = *(const u32x4*)(x0 + ((r < end ? r : end) * ldx2 + 16 * ((int)q < x_pieces ? q : x_pieces - 1)));
    }
  };
  auto store = [&](int step) __attribute__((always_inline)) {
    uint8_t* const buf = lds + (step & 1) * L::kBuf;
#pragma unroll
    for (int i = 0; i < kIn; ++i) {
      const int id = i * kThreads + tid, at = tile_at<N>(id / kRowB, id % kRowB);
      *(u32x4*)(buf + at) = rb[i];
      if constexpr (kOutputs) *(u32x4*)(buf + L::kC + at) = rc[i];
    }
    float zero = 0.f;
#pragma unroll
    for (int i = 0; i < kInX; ++i) {
      const int id = i * kThreads + tid;
      *(u32x4*)(buf + L::kX + tile_at<kXW>(id >> 4, id & 15)) = rx[i];
      if constexpr (kOutputs)
#pragma unroll
        for (int e = 0; e < 4; ++e) zero = dot2_bf16(rx[i][e], 0u, zero);
    }
    if constexpr (kOutputs)
      if (zero != zero) flags[step % 3] = 1;
  };
  // the decays of a group of chunks: each wave one chunk's of two heads
  constexpr int kGroup = L::kGroup;
  const int d_chunk = wave % kGroup, d_pair = 2 * (wave / kGroup);
  const int d_head = d_pair + (lane >> 5) < n_heads ? d_pair + (lane >> 5) : (d_pair < n_heads ? d_pair : 0);
  const uint16_t* const dp = (const uint16_t*)a.dt + (int64_t)pc.row * a.lddt + head0 + first_head + d_head;
  const float A2 = a.a[head0 + first_head + d_head] * kLog2e;
  const float bias = a.dt_bias ? a.dt_bias[head0 + first_head + d_head] : 0.f;
  // The chunks in the order in which they are taken: their number `step` begins at row row_of(step). The
  // ends of a piece (whole chunks) are taken from its last rows on: the decay from behind a chunk to the
  // piece's end then goes into the chunk's factors, and the sums are never scaled.
  const int n_steps = (pc.n + kQ - 1) / kQ;
  auto row_of = [&](int step) __attribute__((always_inline)) { return kOutputs ? step * kQ : (n_steps - 1 - step) * kQ; };
  uint16_t rdt = 0;
  auto load_dt = [&](int step) __attribute__((always_inline)) {  // of the wave's chunk in the group of `step`
    const int s = step + d_chunk < n_steps ? step + d_chunk : n_steps - 1;
    const int r = row_of(s) + (lane & 31);
    rdt = dp[(int64_t)(r < pc.n ? r : pc.n - 1) * a.lddt];
  };
  auto dec_of = [&](int step, int head) __attribute__((always_inline)) {
    return decs + (step % (2 * kGroup) * HEADS + head) * L::kDecHead;
  };
  auto decays = [&](int step) __attribute__((always_inline)) {
    const int s = step + d_chunk < n_steps ? step + d_chunk : n_steps - 1;  // (a chunk that is not there: not read)
    chunk_decays<kOutputs>(bf16_to_f32(rdt) + bias, pc.n - row_of(s), A2, a, dec_of(step + d_chunk, d_head));
  };

  if constexpr (kOutputs) {
    if (tid < 3) flags[tid] = 0;
    __syncthreads();  // the flags are set after they are cleared
  }

  // lane parts of the operand addresses
  const int x_of_row = swizzle<N>(l16);
  const int tr_row = 4 * c4 + (l16 >> 2);  // transposed reads: row, and 16 more (of the same swizzle)
  // the 8 values of step ks of row 16 tile + l16 of B or C
  auto row_operand = [&](const uint8_t* base, int tile, int ks) __attribute__((always_inline)) {
    return as_bf16x8(*(const u32x4*)(base + tile * 16 * (N * 2) + (l16 * (N * 2) + (((4 * ks + c4) ^ x_of_row) << 4))));
  };
  // the chunk's rows of column l16 of the wave's column tile ct
  auto x_operand = [&](const uint8_t* xs, int ct) __attribute__((always_inline)) {
    const uint8_t* const at =
        xs + (tr_row * (2 * kXW) + 8 * ct + (((4 * wave + (l16 & 3)) ^ swizzle<kXW>(tr_row)) << 4));
    return join(read_tr(at), read_tr(at + 16 * (2 * kXW)));
  };
  // the chunk's rows of the columns of state tile T of B
  auto b_operand = [&](const uint8_t* bs, int T) __attribute__((always_inline)) {
    const uint8_t* const at =
        bs + (tr_row * (N * 2) + 8 * (T & 1) + (((4 * (T >> 1) + (l16 & 3)) ^ swizzle<N>(tr_row)) << 4));
    return join(read_tr(at), read_tr(at + 16 * (N * 2)));
  };

  const float D_h = kOutputs && a.d ? a.d[head] : 0.f;
  float total = 0.f;  // log2 of the decay over the piece
  uint8_t* const yp = (uint8_t*)((uint16_t*)a.y + (int64_t)pc.row * a.ldy + (int64_t)head * P + p0);
  const uint32_t ldy2 = (uint32_t)a.ldy * 2, y_at = l16 * ldy2 + 16 * c4;
  load_dt(0);
  load(row_of(0));
  decays(0);
  store(0);
  if (n_steps > kGroup) load_dt(kGroup);
  if (n_steps > 1) load(row_of(1));
  for (int step = 0; step < n_steps; ++step) {
    __syncthreads();  // the chunk is staged, the buffers of the one before are free
    const int t0 = row_of(step);
    const bool more = step + 1 < n_steps;
    const uint8_t* const buf = lds + (step & 1) * L::kBuf;
    const float* const dec = dec_of(step, hh);
    const float all = dec[Dec::kAll], behind = kOutputs ? 1.f : exp2_(total);
    total += dec[Dec::kAll + 1];
    bf16x8 xt[2];  // x^T of the column tiles
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) xt[ct] = x_operand(buf + L::kX, ct);
    // x scaled, in three bf16 parts: two neighbouring rows of one column a call
    u32x4 part[kParts][2];
    f32x4 wt[2] = {*(const f32x4*)&dec[Dec::kW + 4 * c4], *(const f32x4*)&dec[Dec::kW + 16 + 4 * c4]};
    if constexpr (!kOutputs) {
      wt[0] *= behind;
      wt[1] *= behind;
    }
    auto scaled = [&](int ct, int e) __attribute__((always_inline)) {
      const uint32_t xw = __builtin_bit_cast(u32x4, xt[ct])[e];
      const f32x4 w = wt[e >> 1];
      float v0 = bf16_lo(xw) * w[2 * (e & 1)], v1 = bf16_hi(xw) * w[2 * (e & 1) + 1];
#pragma unroll
      for (int k = 0; k < kParts; ++k) {
        const uint32_t u = pack_bf16x2(v0, v1);
        part[k][ct][e] = u;
        if (k < kParts - 1) {
          v0 -= bf16_lo(u);
          v1 -= bf16_hi(u);
        }
      }
    };
    // ---- the next chunk to LDS, the one behind it on its way
    if (more) {
      store(step + 1);
      if (step + 2 < n_steps) load(row_of(step + 2));
    }
    if constexpr (kOutputs) {
      // (the chunk before this one has been read, the one after the next is not stored yet)
      if (tid == 0) flags[(step + 2) % 3] = 0;
      const bool bad = __builtin_amdgcn_readfirstlane(flags[step % 3]) != 0;
      // ---- C B^T, its tiles (0, 0), (0, 1) and (1, 1) of [s, t]; H C_t for the wave's columns; the state's
      // decay. Each wave forms C B^T for itself: sharing the tiles through LDS took a barrier more
      // (69.6 against 64.6 us of pieces) than it saved
      const uint8_t* const Bs = buf;
      const uint8_t* const Cs = buf + L::kC;
      f32x4 s00 = {0.f, 0.f, 0.f, 0.f}, s01 = s00, s11 = s00;
      f32x4 acc[2][2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) acc[t][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const bf16x8 c0 = row_operand(Cs, 0, ks), c1 = row_operand(Cs, 1, ks);
        const bf16x8 b0 = row_operand(Bs, 0, ks), b1 = row_operand(Bs, 1, ks);
        s00 = mfma16(b0, c0, s00);
        s01 = mfma16(b0, c1, s01);
        s11 = mfma16(b1, c1, s11);
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
          const f32x4 u = h[ct][2 * ks], v = h[ct][2 * ks + 1];
          uint32_t hi[4], lo[4];
          split(u[0], u[1], hi[0], lo[0]);
          split(u[2], u[3], hi[1], lo[1]);
          split(v[0], v[1], hi[2], lo[2]);
          split(v[2], v[3], hi[3], lo[3]);
          h[ct][2 * ks] = u * all;
          h[ct][2 * ks + 1] = v * all;
          const bf16x8 hl = as_bf16x8(u32x4{lo[0], lo[1], lo[2], lo[3]}), hb = as_bf16x8(u32x4{hi[0], hi[1], hi[2], hi[3]});
          acc[0][ct] = mfma16(hl, c0, acc[0][ct]);
          acc[1][ct] = mfma16(hl, c1, acc[1][ct]);
          acc[0][ct] = mfma16(hb, c0, acc[0][ct]);
          acc[1][ct] = mfma16(hb, c1, acc[1][ct]);
        }
      }
      // ---- M: lane (l16, c4) holds rows s = 4 c4 + i of its tiles in column t = l16
      auto parts = [&](const f32x4 v, u32x2* m) __attribute__((always_inline)) {
        uint32_t hi[2], lo[2];
        split(v[0], v[1], hi[0], lo[0]);
        split(v[2], v[3], hi[1], lo[1]);
        m[0] = u32x2{hi[0], hi[1]};
        m[1] = u32x2{lo[0], lo[1]};
      };
      auto diagonal = [&](const f32x4 s, int tile) __attribute__((always_inline)) {
        const f32x4 l = *(const f32x4*)&dec[Dec::kL + 16 * tile + 4 * c4];
        const f32x4 step_s = *(const f32x4*)&dec[Dec::kStep + 16 * tile + 4 * c4];
        float sum = dec[Dec::kQ + 64 * tile + lane];  // of rows from 4 c4 + 4 to t, then from s + 1
        f32x4 v;
#pragma unroll
        for (int i = 3; i >= 0; --i) {
          v[i] = 4 * c4 + i <= l16 ? s[i] * (exp2_(sum) * step_s[i]) : 0.f;
          sum += 4 * c4 + i <= l16 ? l[i] : 0.f;
        }
        return v;
      };
      const f32x4 below = s01 * *(const f32x4*)&dec[Dec::kG + 4 * c4] * dec[Dec::kF + 16 + l16];
      u32x2 m00[2], m01[2], m11[2];
      parts(diagonal(s00, 0), m00);
      parts(below, m01);
      parts(diagonal(s11, 1), m11);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float e = dec[Dec::kE + 16 * t + l16];
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) acc[t][ct] *= e;
      }
      auto add = [&](f32x4& acc, const bf16x8 xv, int t) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 1; k >= 0; --k) acc = mfma16(xv, t ? join(m01[k], m11[k]) : join(m00[k], u32x2{0u, 0u}), acc);
      };
      if (!bad) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int ct = 0; ct < 2; ++ct) add(acc[t][ct], xt[ct], t);
      } else {
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
          int first = kQ;  // first row that is not finite in column l16 of tile ct
          u32x4 v = __builtin_bit_cast(u32x4, xt[ct]);
#pragma unroll
          for (int j = 7; j >= 0; --j) {
            const uint32_t mask = j & 1 ? 0x7f800000u : 0x7f80u;
            if ((v[j >> 1] & mask) == mask) {
              const int r = 4 * c4 + (j < 4 ? j : 12 + j);
              first = r < first ? r : first;
              v[j >> 1] &= j & 1 ? 0xffffu : 0xffff0000u;
            }
          }
          int other = __shfl_xor(first, 16, 64);
          first = other < first ? other : first;
          other = __shfl_xor(first, 32, 64);
          first = other < first ? other : first;
#pragma unroll
          for (int t = 0; t < 2; ++t) add(acc[t][ct], as_bf16x8(v), t);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int from = __shfl(first, 4 * c4 + i, 64);
#pragma unroll
            for (int t = 0; t < 2; ++t)
              if (16 * t + l16 >= from) acc[t][ct][i] = __builtin_nanf("");
          }
        }
      }
      if (!idle)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          uint8_t* const row = yp + (int64_t)(t0 + 16 * t) * ldy2;
          // the lane's 8 values of the row of x
          const u32x4 xw = *(const u32x4*)(buf + L::kX + tile_at<kXW>(16 * t + l16, 4 * wave + c4));
          f32x4 u = acc[t][0], v = acc[t][1];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            u[2 * e] = fmaf(D_h, bf16_lo(xw[e]), u[2 * e]);
            u[2 * e + 1] = fmaf(D_h, bf16_hi(xw[e]), u[2 * e + 1]);
            v[2 * e] = fmaf(D_h, bf16_lo(xw[2 + e]), v[2 * e]);
            v[2 * e + 1] = fmaf(D_h, bf16_hi(xw[2 + e]), v[2 * e + 1]);
          }
          if (16 * t + l16 < pc.n - t0)
            *(u32x4*)(row + y_at) = u32x4{pack_bf16x2(u[0], u[1]), pack_bf16x2(u[2], u[3]), pack_bf16x2(v[0], v[1]),
                                          pack_bf16x2(v[2], v[3])};
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) scaled(e >> 2, e & 3);
    // ---- the state, and the next group's decays (they have a place of their own)
#pragma unroll
    for (int T = 0; T < NT; ++T) {
      const bf16x8 bt = b_operand(buf, T);
#pragma unroll
      for (int k = kParts - 1; k >= 0; --k)
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) h[ct][T] = mfma16(bt, as_bf16x8(part[k][ct]), h[ct][T]);
    }
    if (more && (step + 1) % kGroup == 0) {
      decays(step + 1);
      if (step + 1 + kGroup < n_steps) load_dt(step + 1 + kGroup);
    }
  }

  if (PHASE == kSsmEnds) {
    if (!idle)
#pragma unroll
      for (int ct = 0; ct < 2; ++ct)
#pragma unroll
        for (int T = 0; T < NT; ++T) *(f32x4*)(carry + (ct * NT + T) * 256) = h[ct][T];
  } else if (last && slot >= 0 && !idle) {
#pragma unroll
    for (int ct = 0; ct < 2; ++ct)
#pragma unroll
      for (int T = 0; T < NT; ++T) *(f32x4*)(pool + (st_at + 4 * ct * N + 32 * (T >> 1) + 4 * (T & 1))) = h[ct][T];
  }
  if (PHASE == kSsmEnds && !idle && p0 == 0 && lane == 0) a.carry_decay[place * a.heads + head] = exp2_(total);
}

template <int N, int HEADS, int PHASE>
hipError_t launch_phase(hipStream_t s, const SsmArgs& a, const ChunkGrid& g) {
  constexpr int bytes = Lds<N, HEADS, PHASE != kSsmEnds>::kBytes;
  static std::atomic<uint64_t> done{0};
  const void* fn = (const void*)ssm_chunk_kernel<N, HEADS, PHASE>;
  if (allow_lds_once(fn, bytes, &done, "ema_ssm_scan LDS") != EMA_OK) return hipErrorInvalidValue;
  const int64_t blocks = (g.pairs + 7) / 8 * 8 * g.wgs;
  hipLaunchKernelGGL((ssm_chunk_kernel<N, HEADS, PHASE>), dim3((unsigned)blocks), dim3(kThreads), bytes, s, a, g);
  return hipGetLastError();
}
template <int N, int HEADS>
hipError_t launch_heads(hipStream_t s, const SsmArgs& a, const ChunkGrid& g, SsmPhase phase) {
  return phase == kSsmWhole ? launch_phase<N, HEADS, kSsmWhole>(s, a, g)
         : phase == kSsmEnds ? launch_phase<N, HEADS, kSsmEnds>(s, a, g)
                             : launch_phase<N, HEADS, kSsmPieces>(s, a, g);
}
// The heads that a workgroup's four 32-column pieces touch at most: four of 32, one of 128, else two.
template <int N>
hipError_t launch_state(hipStream_t s, const SsmArgs& a, const ChunkGrid& g, SsmPhase phase) {
  return g.per_head == 1   ? launch_heads<N, 4>(s, a, g, phase)
         : g.per_head == 4 ? launch_heads<N, 1>(s, a, g, phase)
                           : launch_heads<N, 2>(s, a, g, phase);
}

}  // namespace

hipError_t launch_ssm_chunk(hipStream_t s, const SsmArgs& a, int64_t pieces, SsmPhase phase) {
  ChunkGrid g;
  g.per_head = a.head_dim / kCols;
  g.units = a.heads / a.groups * g.per_head;
  g.wgs = (g.units + 3) / 4;
  g.pairs = pieces * a.groups;
  return a.d_state == 64    ? launch_state<64>(s, a, g, phase)
         : a.d_state == 128 ? launch_state<128>(s, a, g, phase)
                            : launch_state<256>(s, a, g, phase);
}

}  // namespace ema
