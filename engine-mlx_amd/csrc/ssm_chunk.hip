// Selective state space scan in chunks of 64 rows on the matrix cores, bf16 activations.
//
// With a_t = d_t A and sums over rows of the chunk, a chunk that starts from the state H gives
//   y_t = e^(a_0 + .. + a_t) H C_t + sum_{s <= t} M[t][s] x_s,
//   M[t][s] = (C_t . B_s) e^(a_(s+1) + .. + a_t) d_s  (+ D for s = t),
//   H'  = e^(a_0 + .. + a_63) H + sum_s (d_s e^(a_(s+1) + .. + a_63) x_s) B_s^T,
// so C B^T is formed once for all heads of a group, and the rest is products with 64-row operands.
//
// A workgroup of four waves takes 128 columns of x (two heads of 64, one of 128, ...) of one group,
// a wave 32 of them: its H^T [d_state, 32] stays in 32-bit accumulators over the rows of the piece.
// All products are 16x16x32 in forms that chain without moving data between lanes:
//   C B^T as [s, t]          A = B rows,       B = C rows (columns t)
//   y^T [p, t]              A = H (the accumulators, rounded to bf16) and x^T, B = C and M
//   H^T [n, p]              A = B^T,           B = x^T scaled
// An accumulator pair holds k slots in the order 4 c + (0..3), 16 + 4 c + (0..3) of lane group c;
// operands from LDS are read in the same order (C and B rows in two 8-byte reads; x^T and B^T by
// the transposing read). The decays of M are products of factors at most 1 (A <= 0): from s to the
// end of its 16-row tile and the tiles between (g), and from t's tile's start to t (f); differences
// of sums only inside the tiles on the diagonal.
//
// Rounded to bf16: H and M where they are operands of y (as an attention's weights are; x, B and C
// are exact), each by at most 2^-8 of the term. The state itself takes the scaled x as three bf16
// parts, 24 bits together (two left it 1.5e-6 off, three 5e-8), products and sums in 32 bits.
//
// A value of x that is not finite would reach rows before it through M's zeros (0 times infinity):
// chunks with such values (a dot product with zeros finds them while they are staged) take those
// columns' sums without them and put NaN into the rows from the value on.
#include <type_traits>

#include "ssm.hpp"

namespace ema {
namespace {

constexpr int kQ = 64;        // rows of a chunk
constexpr int kCols = 32;     // columns of x of a wave
constexpr int kThreads = 256;

typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Per-head values of a chunk (floats), written by one wave: index by row unless said otherwise.
struct Dec {
  static constexpr int kCum = 0;     // sum of log2 decays from the row's 16-row tile's start, the row included
  static constexpr int kStep = 64;   // d
  static constexpr int kF = 128;     // decay from the tile's start: 2^kCum
  static constexpr int kE = 192;     // decay from the chunk's start
  static constexpr int kW = 256;     // d times the decay from behind the row to the chunk's end
  static constexpr int kG = 320;     // [3][64]: d times the decay from behind row s to the start of tile 1, 2, 3
  static constexpr int kAll = 512;   // decay over the chunk; its log2 at 513
  static constexpr int kD = 514;     // D
  static constexpr int kFloats = 516;
};

// Row pitch and swizzle of the LDS tiles of N-wide rows: 16-byte piece q of row r lies at piece
// q ^ x(r), so that 16 rows at one piece, and 8 rows at two neighbouring ones, are in distinct banks.
template <int W>
__device__ __forceinline__ int swizzle(int r) {
  return W == 64 ? ((r >> 1) & 3) * 2 | ((r >> 3) & 1) : (r & 7) * 2 | ((r >> 3) & 1);
}
template <int W>
__device__ __forceinline__ int tile_at(int r, int q) {  // bytes
  return r * (W * 2) + ((q ^ swizzle<W>(r)) << 4);
}

__device__ __forceinline__ bf16x8 join(u32x2 lo, u32x2 hi) { return as_bf16x8(u32x4{lo[0], lo[1], hi[0], hi[1]}); }
__device__ __forceinline__ u32x2 read8(const uint8_t* p) { return *(const u32x2*)p; }
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

// Decays of one head's 64 rows, a row a lane; `raw` is dt + bias, rows from n on take no step.
template <bool kOutputs>
__device__ __forceinline__ void chunk_decays(float raw, int n, float A2, float D, const SsmArgs& a, float* dec) {
  const int lane = threadIdx.x & 63;
  const float d = lane < n ? ssm_step(raw, a) : 0.f;
  // log2 of the row's decay; below 2^-150 it is 0 either way, and sums stay finite
  const float l = fmaxf(d * A2, -150.f);
  float up = l, down = l;  // sums over the 16-row tile: up to the row, from the row on
  up += dpp_shift<0x111>(up);
  down += dpp_shift<0x101>(down);
  up += dpp_shift<0x112>(up);
  down += dpp_shift<0x102>(down);
  up += dpp_shift<0x114>(up);
  down += dpp_shift<0x104>(down);
  up += dpp_shift<0x118>(up);
  down += dpp_shift<0x108>(down);
  const float behind = dpp_shift<0x101>(down);  // from behind the row to its tile's end
  const float t0 = lane_value(up, 15), t1 = lane_value(up, 31), t2 = lane_value(up, 47), t3 = lane_value(up, 63);
  const int tile = lane >> 4;
  const float later = tile == 0 ? t1 + t2 + t3 : tile == 1 ? t2 + t3 : tile == 2 ? t3 : 0.f;
  dec[Dec::kW + lane] = d * exp2_(behind + later);
  if (lane == 0) {
    const float all = (t0 + t1) + (t2 + t3);
    dec[Dec::kAll] = exp2_(all);
    dec[Dec::kAll + 1] = all;
    dec[Dec::kD] = D;
  }
  if constexpr (kOutputs) {
    const float before = tile == 0 ? 0.f : tile == 1 ? t0 : tile == 2 ? t0 + t1 : t0 + t1 + t2;
    dec[Dec::kCum + lane] = up;
    dec[Dec::kStep + lane] = d;
    dec[Dec::kF + lane] = exp2_(up);
    dec[Dec::kE + lane] = exp2_(up + before);
    dec[Dec::kG + lane] = d * exp2_(behind);  // tile 0 to the start of tile 1
    dec[Dec::kG + 64 + lane] = d * exp2_(behind + (tile == 0 ? t1 : 0.f));
    dec[Dec::kG + 128 + lane] = d * exp2_(behind + (tile == 0 ? t1 + t2 : tile == 1 ? t2 : 0.f));
  }
}

// LDS (bytes): B, x, then for outputs C, M of every head of the workgroup; the heads' decays, twice;
// the flags of chunks with values that are not finite, twice.
template <int N, bool kOutputs>
struct Lds {
  static constexpr int kB = 0;
  static constexpr int kX = kB + kQ * N * 2;
  static constexpr int kC = kX + kQ * 4 * kCols * 2;
  static constexpr int kM = kC + (kOutputs ? kQ * N * 2 : 0);
  static constexpr int kMHead = 6 * 1024;  // (row tile, 32-row step): (0,0) (1,0) (2,0) (2,1) (3,0) (3,1)
  static constexpr __host__ __device__ int dec(int heads) { return kM + (kOutputs ? heads * kMHead : 0); }
  static constexpr __host__ __device__ int flag(int heads) { return dec(heads) + 2 * heads * Dec::kFloats * 4; }
  static constexpr __host__ __device__ int bytes(int heads) { return flag(heads) + 16; }
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
  typedef Lds<N, kOutputs> L;
  constexpr int KS = N / 32;   // 32-wide steps over d_state
  constexpr int NT = N / 16;   // 16-row tiles of it
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];

  // the workgroups of a (piece, group) read the same B and C: on one XCD (blocks go to the XCDs in turn)
  const uint32_t xcd = blockIdx.x & 7, k8 = blockIdx.x >> 3;
  const int wg = (int)(k8 % (uint32_t)gr.wgs);
  const int64_t pair = xcd + 8 * (int64_t)(k8 / (uint32_t)gr.wgs);
  if (pair >= gr.pairs) return;
  const int grp = (int)(pair % a.groups), index = (int)(pair / a.groups);
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
  float* const carry = a.carry + ((int64_t)index * a.heads + head) * P * N;
  const int64_t st_at = (int64_t)(p0 + l16) * N + 4 * c4;

  uint8_t* const Bs = lds + L::kB;
  uint8_t* const Xs = lds + L::kX;
  uint8_t* const Cs = lds + L::kC;
  uint8_t* const Ms = lds + L::kM;
  float* const decs = (float*)(lds + L::dec(HEADS));
  int* const flags = (int*)(lds + L::flag(HEADS));

  // ---- state: h[ct][T] holds n = 16 T + 4 c4 + i of column p0 + 16 ct + l16
  f32x4 h[2][NT];
  {
    const float* from = nullptr;
    if (PHASE == kSsmPieces && pc.all > a.piece)
      from = carry;
    else if (kOutputs && slot >= 0 && packed_continues(a.offsets, pc.b))
      from = pool;
#pragma unroll
    for (int ct = 0; ct < 2; ++ct)
#pragma unroll
      for (int T = 0; T < NT; ++T) {
        h[ct][T] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (from) h[ct][T] = *(const f32x4*)(from + st_at + (int64_t)16 * ct * N + 16 * T);
      }
  }

  // ---- staging: 16-byte pieces of rows, a chunk ahead in registers
  constexpr int kRowB = N / 8;                     // pieces of a B or C row
  constexpr int kIn = kQ * kRowB / kThreads;       // pieces of B (or C) a thread
  constexpr int kInX = kQ * 16 / kThreads;
  u32x4 rb[kIn], rc[kOutputs ? kIn : 1], rx[kInX];
  float rdt = 0.f;
  // rows within a chunk are 32-bit offsets from a uniform base (64 rows of ld* < 2^23: plan_ssm)
  const uint8_t* const bp = (const uint8_t*)((const uint16_t*)a.b + (int64_t)pc.row * a.ldb + grp * N);
  const uint8_t* const cp = (const uint8_t*)((const uint16_t*)a.c + (int64_t)pc.row * a.ldc + grp * N);
  const uint8_t* const xp = (const uint8_t*)((const uint16_t*)a.x + (int64_t)pc.row * a.ldx + (int64_t)head0 * P + unit0 * kCols);
  const uint32_t ldb2 = (uint32_t)a.ldb * 2, ldc2 = (uint32_t)a.ldc * 2, ldx2 = (uint32_t)a.ldx * 2;
  const int x_pieces = (last_unit - unit0 + 1) * (kCols / 8);
  const bool scalars = wave < n_heads;             // this wave forms a head's decays
  const int s_head = head0 + first_head + (scalars ? wave : 0);
  const uint16_t* const dp = (const uint16_t*)a.dt + (int64_t)pc.row * a.lddt + s_head;
  const float A2 = a.a[s_head] * kLog2e, bias = a.dt_bias ? a.dt_bias[s_head] : 0.f;
  const float D = a.d ? a.d[s_head] : 0.f;

  // rows behind the piece are its last row again: what they would add has step 0
  auto fetch = [&](int t0) __attribute__((always_inline)) {
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
      const uint32_t row = r < end ? r : end;
      rx[i] = (int)q < x_pieces ? *(const u32x4*)(x0 + (row * ldx2 + 16 * q)) : u32x4{0u, 0u, 0u, 0u};
    }
    if (scalars) rdt = bf16_to_f32(dp[(int64_t)(t0 + (int)((uint32_t)lane < end ? (uint32_t)lane : end)) * a.lddt]);
  };
  auto stage = [&](int t0, int par) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kIn; ++i) {
      const int id = i * kThreads + tid, r = id / kRowB, q = id % kRowB;
      *(u32x4*)(Bs + tile_at<N>(r, q)) = rb[i];
      if constexpr (kOutputs) *(u32x4*)(Cs + tile_at<N>(r, q)) = rc[i];
    }
    float zero = 0.f;
#pragma unroll
    for (int i = 0; i < kInX; ++i) {
      const int id = i * kThreads + tid, r = id >> 4, q = id & 15;
      *(u32x4*)(Xs + tile_at<4 * kCols>(r, q)) = rx[i];
      if constexpr (kOutputs)
#pragma unroll
        for (int e = 0; e < 4; ++e) zero = dot2_bf16(rx[i][e], 0u, zero);
    }
    if constexpr (kOutputs)
      if (zero != zero) flags[par] = 1;
    if (scalars) chunk_decays<kOutputs>(rdt + bias, pc.n - t0, A2, D, a, decs + (par * HEADS + wave) * Dec::kFloats);
  };

  if constexpr (kOutputs) {
    // the upper halves of the steps (0, 0) and (2, 1) are tiles above the diagonal: zero for good
    for (int i = tid; i < n_heads * 64; i += kThreads) {
      uint8_t* const m = Ms + (i >> 6) * L::kMHead + (i & 63) * 16 + 8;
      *(u32x2*)m = u32x2{0u, 0u};
      *(u32x2*)(m + 3 * 1024) = u32x2{0u, 0u};
    }
    if (tid < 2) flags[tid] = 0;
  }
  __syncthreads();  // the flags are set after they are cleared

  // lane parts of the operand addresses
  const int x_of_row = swizzle<N>(l16);
  const int row_b = l16 * (N * 2) + 8 * (c4 & 1);                  // rows of B and C at a tile's start
  const int tr_row = 4 * c4 + (l16 >> 2);                          // transposed reads: row, and 16 more
  const int tr_half = 8 * (l16 & 1), tr_q = (l16 & 3) >> 1;
  // 8 values (slots of step ks) of row 16 tile + l16 of B or C
  auto row_operand = [&](const uint8_t* base, int tile, int ks) __attribute__((always_inline)) {
    const uint8_t* const r = base + tile * 16 * (N * 2) + row_b;
    return join(read8(r + (((4 * ks + (c4 >> 1)) ^ x_of_row) << 4)), read8(r + (((4 * ks + 2 + (c4 >> 1)) ^ x_of_row) << 4)));
  };
  // 8 rows (slots of step kt) of column 16 tile + l16
  auto col_operand = [&](auto width, const uint8_t* base, int tile, int kt) __attribute__((always_inline)) {
    constexpr int W = decltype(width)::value;
    const uint8_t* const r = base + (32 * kt) * (W * 2) + tr_half;
    const int q = 2 * tile + tr_q;
    const int sw = swizzle<W>(tr_row);  // (rows 16 apart have the same)
    const uint8_t* const at = r + tr_row * (W * 2) + ((q ^ sw) << 4);
    return join(read_tr(at), read_tr(at + 16 * (W * 2)));
  };
  typedef std::integral_constant<int, 4 * kCols> XW;
  typedef std::integral_constant<int, N> BW;

  float total = 0.f;  // log2 of the decay over the piece
  uint16_t* const yp = (uint16_t*)a.y + (int64_t)pc.row * a.ldy + (int64_t)head * P + p0 + 4 * c4;
  fetch(0);
  stage(0, 0);
  for (int t0 = 0, par = 0; t0 < pc.n; t0 += kQ, par ^= 1) {
    __syncthreads();  // the chunk is staged
    const bool more = t0 + kQ < pc.n;
    if (more) fetch(t0 + kQ);
    const float* const dec = decs + (par * HEADS + hh) * Dec::kFloats;
    bf16x8 xt[2][2];  // x^T: [column tile][32-row step]
    if constexpr (kOutputs) {
      // ---- C B^T tiles, and M of every head from them: a wave takes the diagonal tile (w, w) and two
      // below it, (3, 0) (3, 1) | (2, 0) (3, 2) | (2, 1) twice | (1, 0) twice
      f32x4 s[3];
      int tt[3], st[3];
      tt[0] = st[0] = wave;
      tt[1] = wave == 0 ? 3 : wave == 3 ? 1 : 2;
      st[1] = wave == 2 ? 1 : 0;
      tt[2] = wave < 2 ? 3 : tt[1];
      st[2] = wave == 0 ? 1 : wave == 1 ? 2 : st[1];
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        s[k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s[k] = mfma16(row_operand(Bs, st[k], ks), row_operand(Cs, tt[k], ks), s[k]);
      }
#pragma unroll
      for (int j = 0; j < HEADS; ++j) {
        if (j > 0 && j >= n_heads) break;
        const float* const dj = decs + (par * HEADS + j) * Dec::kFloats;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const int t = 16 * tt[k] + l16, s0 = 16 * st[k] + 4 * c4;
          f32x4 v;
          if (k == 0) {
            const f32x4 cum = *(const f32x4*)&dj[Dec::kCum + s0], step = *(const f32x4*)&dj[Dec::kStep + s0];
            const float ct = dj[Dec::kCum + t];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[i] = s0 + i <= t ? s[k][i] * (exp2_(ct - cum[i]) * step[i]) : 0.f;
              if (s0 + i == t) v[i] += dj[Dec::kD];
            }
          } else {
            const f32x4 g = *(const f32x4*)&dj[Dec::kG + 64 * (tt[k] - 1) + s0];
            const float f = dj[Dec::kF + t];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = s[k][i] * g[i] * f;
          }
          const int slot_m = tt[k] < 2 ? tt[k] : 2 * tt[k] - 2 + (st[k] >> 1);
          *(u32x2*)(Ms + j * L::kMHead + slot_m * 1024 + lane * 16 + 8 * (st[k] & 1)) =
              u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        }
      }
      // ---- H C_t for the wave's columns
      f32x4 acc[4][2];
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) acc[tt][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        bf16x8 hb[2];
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
          const f32x4 u = h[ct][2 * ks], v = h[ct][2 * ks + 1];
          hb[ct] = as_bf16x8(u32x4{pack_bf16x2(u[0], u[1]), pack_bf16x2(u[2], u[3]), pack_bf16x2(v[0], v[1]),
                                   pack_bf16x2(v[2], v[3])});
        }
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const bf16x8 co = row_operand(Cs, tt, ks);
#pragma unroll
          for (int ct = 0; ct < 2; ++ct) acc[tt][ct] = mfma16(hb[ct], co, acc[tt][ct]);
        }
      }
#pragma unroll
      for (int ct = 0; ct < 2; ++ct)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) xt[ct][kt] = col_operand(XW(), Xs, 2 * wave + ct, kt);
      __syncthreads();  // M is whole
      const bool bad = __builtin_amdgcn_readfirstlane(flags[par]) != 0;
      int first[2] = {kQ, kQ};  // first row whose x is not finite, in column 16 ct + l16
      if (bad) {
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) {
            u32x4 v = __builtin_bit_cast(u32x4, xt[ct][kt]);
#pragma unroll
            for (int j = 7; j >= 0; --j) {
              const uint32_t mask = j & 1 ? 0x7f800000u : 0x7f80u;
              if ((v[j >> 1] & mask) == mask) {
                const int r = 32 * kt + 4 * c4 + (j < 4 ? j : 12 + j);
                first[ct] = r < first[ct] ? r : first[ct];
                v[j >> 1] &= j & 1 ? 0xffffu : 0xffff0000u;
              }
            }
            xt[ct][kt] = as_bf16x8(v);
          }
          int other = __shfl_xor(first[ct], 16, 64);
          first[ct] = other < first[ct] ? other : first[ct];
          other = __shfl_xor(first[ct], 32, 64);
          first[ct] = other < first[ct] ? other : first[ct];
        }
      }
      const uint8_t* const mh = Ms + hh * L::kMHead + lane * 16;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const float e = dec[Dec::kE + 16 * tt + l16];
        const int base = tt < 2 ? tt : 2 * tt - 2;
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) acc[tt][ct] *= e;
#pragma unroll
        for (int kt = 0; kt <= tt >> 1; ++kt) {
          const bf16x8 mo = as_bf16x8(*(const u32x4*)(mh + (base + kt) * 1024));
#pragma unroll
          for (int ct = 0; ct < 2; ++ct) acc[tt][ct] = mfma16(xt[ct][kt], mo, acc[tt][ct]);
        }
      }
      if (bad) {
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int from = __shfl(first[ct], 4 * c4 + i, 64);
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
              if (16 * tt + l16 >= from) acc[tt][ct][i] = __builtin_nanf("");
          }
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) xt[ct][kt] = col_operand(XW(), Xs, 2 * wave + ct, kt);
        }
      }
      if (!idle)
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const int t = t0 + 16 * tt + l16;
          if (t < pc.n)
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) {
              const f32x4 v = acc[tt][ct];
              *(u32x2*)(yp + (int64_t)t * a.ldy + 16 * ct) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
            }
        }
    } else {
#pragma unroll
      for (int ct = 0; ct < 2; ++ct)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) xt[ct][kt] = col_operand(XW(), Xs, 2 * wave + ct, kt);
    }
    // ---- the state
    const float all = dec[Dec::kAll];
    total += dec[Dec::kAll + 1];
#pragma unroll
    for (int ct = 0; ct < 2; ++ct)
#pragma unroll
      for (int T = 0; T < NT; ++T) h[ct][T] *= all;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const f32x4 wl = *(const f32x4*)&dec[Dec::kW + 32 * kt + 4 * c4], wh = *(const f32x4*)&dec[Dec::kW + 32 * kt + 16 + 4 * c4];
      bf16x8 part[3][2];
#pragma unroll
      for (int ct = 0; ct < 2; ++ct) {
        const u32x4 xw = __builtin_bit_cast(u32x4, xt[ct][kt]);
        u32x4 u[3];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v0 = bf16_lo(xw[e]) * (e < 2 ? wl[2 * e] : wh[2 * e - 4]);
          float v1 = bf16_hi(xw[e]) * (e < 2 ? wl[2 * e + 1] : wh[2 * e - 3]);
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            u[k][e] = pack_bf16x2(v0, v1);
            if (k < 2) {
              v0 -= bf16_lo(u[k][e]);
              v1 -= bf16_hi(u[k][e]);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) part[k][ct] = as_bf16x8(u[k]);
      }
#pragma unroll
      for (int T = 0; T < NT; ++T) {
        const bf16x8 bt = col_operand(BW(), Bs, T, kt);
#pragma unroll
        for (int k = 2; k >= 0; --k)
#pragma unroll
          for (int ct = 0; ct < 2; ++ct) h[ct][T] = mfma16(bt, part[k][ct], h[ct][T]);
      }
    }
    __syncthreads();  // the chunk's tiles are free
    if (kOutputs && tid == 0) flags[par] = 0;
    if (more) stage(t0 + kQ, par ^ 1);
  }

  float* const to = PHASE == kSsmEnds ? carry : (last && slot >= 0 ? pool : nullptr);
  if (to && !idle)
#pragma unroll
    for (int ct = 0; ct < 2; ++ct)
#pragma unroll
      for (int T = 0; T < NT; ++T) *(f32x4*)(to + st_at + (int64_t)16 * ct * N + 16 * T) = h[ct][T];
  if (PHASE == kSsmEnds && !idle && p0 == 0 && lane == 0) a.carry_decay[(int64_t)index * a.heads + head] = exp2_(total);
}

template <int N, int HEADS, int PHASE>
hipError_t launch_phase(hipStream_t s, const SsmArgs& a, const ChunkGrid& g) {
  constexpr int bytes = Lds<N, PHASE != kSsmEnds>::bytes(HEADS);
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

bool ssm_chunk_shape(int head_dim, int d_state) {
  return head_dim % kCols == 0 && (d_state == 64 || d_state == 128 || d_state == 256);
}

int ssm_chunk_workgroups(int heads, int head_dim, int groups) {
  return groups * ((heads / groups * (head_dim / kCols) + 3) / 4);
}

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
