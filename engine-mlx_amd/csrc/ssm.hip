// Selective state space scan, one decay per head, token by token; the launches of all its kernels.
//
// Lane layout: 16 lanes share a state row (one value of head_dim); lane p holds its elements
// n = 4 p + 64 i + j (i < NI, j < 4), so a 16-byte state access of a wave covers 256 contiguous
// bytes of each of 4 rows, and y is a sum of 4 NI products and four DPP steps. A wave holds R
// times 4 rows, which share the lane's B and C values. The state stays in registers over the rows of
// the piece.
// One row (a decode step): HBM-bound, 8 bytes of state traffic per element against 6 flops: 32 users of
// 64 heads of 64, d_state 128, 135 MB in 21.4 us (6.3 TB/s). Many rows: bound by the vector instructions of
// a row (R = 4: 128, of which 96 are the recurrence's) and, for smaller R, by the loads of B and C, which
// each of a wave's four groups of 16 lanes makes: 8192 rows of 64 heads in f32 0.79 ms. Rows are loaded
// kAhead at a time from bases that are uniform: behind a row's sums the row kAhead later, but the first row of
// each kAhead waits for all of their loads (the first ones are conditional, so that the compiler cannot count on
// any behind the row's own). One ahead, with addresses formed in each lane, 2048 rows of 24 heads took 913 us
// whole and 137 cut in time, now 414 and 112.
#include "ssm.hpp"

namespace ema {
namespace {

constexpr int kWaves = 4;

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
// Sum over 16 lanes, in all of them: quad_perm [1,0,3,2] and [2,3,0,1], row_half_mirror, row_mirror.
__device__ __forceinline__ float row_sum16(float v) {
  v = dpp_add<0xB1>(v);
  v = dpp_add<0x4E>(v);
  v = dpp_add<0x141>(v);
  return dpp_add<0x140>(v);
}

__device__ __forceinline__ float lane_value(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// kEnds: E and the decay of the pieces that are not their sequence's last; else y, and the state.
// kAhead: rows in registers, loaded ahead of their sums.
template <typename A, int NI, int R, bool kWhole, bool kEnds, int kAhead>
__global__ __launch_bounds__(64 * kWaves) void ssm_token_kernel(SsmArgs a, int row_blocks) {
  typedef typename A::T T;
  uint32_t id = blockIdx.x;
  const int rb = (int)(id % (uint32_t)row_blocks);
  id /= (uint32_t)row_blocks;
  const int h = (int)(id % (uint32_t)a.heads);
  const int index = (int)(id / (uint32_t)a.heads);
  const Piece pc = packed_piece(a.starts, a.batch, a.n_rows, a.T, a.piece, index);
  if (pc.n == 0) return;
  const bool last = pc.row + pc.n == pc.begin + pc.all;
  if (kEnds && last) return;
  if ((rb * kWaves + (int)(threadIdx.x >> 6)) * 4 * R >= a.head_dim) return;  // (a whole wave; there are no barriers)

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int p = lane & 15;
  const int row0 = (rb * kWaves + wave) * 4 * R + (lane >> 4);  // rows row0 + 4 i
  const int N = a.d_state, P = a.head_dim;
  const int g = h / (a.heads / a.groups);
  const int slot = packed_slot(a.slots, pc.b, a.n_slots);
  float* const pool = a.state + ((int64_t)slot * a.heads + h) * P * N;
  const int64_t place = packed_first_place(pc.begin, pc.b, a.piece) + pc.index - pc.first;  // (of a longer sequence)
  float* const carry = a.carry + (place * a.heads + h) * P * N;

  // Whole: every lane has its state rows and elements. Else the lanes behind the last take the last
  // one's inputs; elements from d_state on are zeros, rows from head_dim on are not stored.
  bool on[NI];
  uint32_t n_at[NI], x_at[R];
#pragma unroll
  for (int k = 0; k < NI; ++k) {
    on[k] = kWhole || 4 * p + 64 * k < N;
    n_at[k] = on[k] ? 4 * p + 64 * k : N - 4;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) x_at[i] = kWhole || row0 + 4 * i < P ? row0 + 4 * i : P - 1;
  f32x4 s[R][NI];
  {
    // a sequence of one piece starts from the pool; pieces of a longer one never read what its
    // last piece writes there
    const float* from = nullptr;
    if (!kEnds && pc.all > a.piece)
      from = carry;
    else if (!kEnds && slot >= 0 && packed_continues(a.offsets, pc.b))
      from = pool;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int k = 0; k < NI; ++k) {
        s[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (from && (kWhole || (row0 + 4 * i < P && on[k]))) s[i][k] = *(const f32x4*)(from + (int64_t)(row0 + 4 * i) * N + 4 * p + 64 * k);
      }
  }
  const float A_h = a.a[h], D_h = a.d ? a.d[h] : 0.f, bias = a.dt_bias ? a.dt_bias[h] : 0.f;
  const T* const dp = (const T*)a.dt + (int64_t)pc.row * a.lddt + h;
  // the next row to load and to write: uniform, a lane's place in it a 32-bit offset
  const T* xp = (const T*)a.x + (int64_t)pc.row * a.ldx + h * P;
  const T* bp = (const T*)a.b + (int64_t)pc.row * a.ldb + g * N;
  const T* cp = (const T*)a.c + (int64_t)pc.row * a.ldc + g * N;
  T* yp = (T*)a.y + (int64_t)pc.row * a.ldy + h * P;

  struct Row {
    Vec<A, 4> b[NI], c[NI];
    T x[R];
  };
  int left = pc.n;  // rows not loaded (from the last on it is loaded again)
  auto fetch = [&](Row& r) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < R; ++i) r.x[i] = xp[x_at[i]];
#pragma unroll
    for (int k = 0; k < NI; ++k) {
      r.b[k].load(bp + n_at[k]);
      if (!kEnds) r.c[k].load(cp + n_at[k]);
    }
    const bool more = --left > 0;
    xp += more ? a.ldx : 0;
    bp += more ? a.ldb : 0;
    if (!kEnds) cp += more ? a.ldc : 0;
  };
  // the steps of 64 rows, a row a lane
  T raw = dp[(int64_t)(lane < pc.n ? lane : pc.n - 1) * a.lddt];
  float steps = 0.f, decays = 0.f, sum = 0.f;
  auto step64 = [&](int t) __attribute__((always_inline)) {
    steps = ssm_step(A::to(raw) + bias, a);
    decays = steps * A_h;
    if (kEnds) sum += t + lane < pc.n ? decays : 0.f;
    decays = expf(decays);
    const int at = t + 64 + lane;
    if (t + 64 < pc.n) raw = dp[(int64_t)(at < pc.n ? at : pc.n - 1) * a.lddt];
  };
  auto row = [&](int t, const Row& r) __attribute__((always_inline)) {
    const float d = lane_value(steps, t & 63), decay = lane_value(decays, t & 63);
    T out[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float xv = A::to(r.x[i]);
      const float dx = d * xv;
      float y = 0.f;
#pragma unroll
      for (int k = 0; k < NI; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][k][j] = fmaf(dx, on[k] ? r.b[k][j] : 0.f, decay * s[i][k][j]);
          if (!kEnds) y = fmaf(s[i][k][j], r.c[k][j], y);
        }
      if (!kEnds) out[i] = A::from(fmaf(D_h, xv, row_sum16(y)));
    }
    if (!kEnds) {
      if (p == 0)
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (kWhole || row0 + 4 * i < P) yp[x_at[i]] = out[i];
      yp += a.ldy;
    }
  };
  Row rows[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (i < pc.n) fetch(rows[i]);
  int t = 0;
  for (; t + kAhead <= pc.n; t += kAhead) {
    if ((t & 63) == 0) step64(t);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      row(t + i, rows[i]);
      fetch(rows[i]);
    }
  }
  if (t < pc.n && (t & 63) == 0) step64(t);
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (t + i < pc.n) row(t + i, rows[i]);
  float* const to = kEnds ? carry : (last && slot >= 0 ? pool : nullptr);
  if (to)
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int k = 0; k < NI; ++k)
        if (kWhole || (row0 + 4 * i < P && on[k])) *(f32x4*)(to + (int64_t)(row0 + 4 * i) * N + 4 * p + 64 * k) = s[i][k];
  if (kEnds && rb == 0 && wave == 0) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m, 64);
    if (lane == 0) a.carry_decay[place * a.heads + h] = expf(sum);
  }
}

// Joins a sequence's pieces in order: each piece's E in the workspace becomes its start state.
// A lane per 4 elements of (head, state), one piece after the other: a piece's loads wait for the store before
// them (they may be of the same place, for all that the compiler knows), a round trip to memory a piece. 17 pieces
// of 64 heads of 64, d_state 128: 13.1 us for 67 MB, 5.1 TB/s; 10 pieces of 12 heads 5.7 us, the round trips.
__global__ __launch_bounds__(256) void ssm_join_kernel(SsmArgs a, bool chunks) {
  const int b = blockIdx.y;
  const PackedRows r = packed_sequence(a.starts, b, a.n_rows, a.T);
  if (r.n <= a.piece) return;
  const int per_head = a.head_dim * a.d_state / 4;
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= a.heads * per_head) return;
  const int h = v / per_head;
  const int first = packed_first_place(r.begin, b, a.piece), n = (r.n + a.piece - 1) / a.piece;
  const int64_t stride = (int64_t)a.heads * per_head;
  f32x4* const c = (f32x4*)a.carry + first * stride + v;
  const float* const decay = a.carry_decay + (int64_t)first * a.heads + h;
  const int slot = packed_slot(a.slots, b, a.n_slots);
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (slot >= 0 && packed_continues(a.offsets, b)) {
    const int e = v - h * per_head;
    s = *(const f32x4*)(a.state + ((int64_t)slot * a.heads + h) * per_head * 4 + (chunks ? ssm_carry_element(e, a.d_state) : 4 * e));
  }
  for (int i = 0; i < n - 1; ++i) {
    const f32x4 e = c[i * stride];
    c[i * stride] = s;
    s = s * decay[(int64_t)i * a.heads] + e;
  }
  c[(n - 1) * stride] = s;
}

template <typename A, int NI, int R, bool kWhole>
hipError_t launch_phase(hipStream_t s, const SsmArgs& a, int64_t pieces, SsmPhase phase) {
  // A call's pieces are long and their waves few: rows ahead; whole sequences of R = 4 may be tokens and come
  // with many waves, which gain more from registers: one token of 32 users of 64 heads, d_state 128 21.2 us
  // against 23.8 with four rows ahead, 31 tokens of 128 users of 24 heads of 48 x 80 111 and 137, 31 of 32
  // users of 64 heads 83.0 and 82.3; pieces of 8192 rows of 64 heads (f32) 849 and 785.
  constexpr int kAhead = NI == 4 ? 2 : 4, kWholeAhead = R == 4 && NI < 4 ? 1 : kAhead;
  const int rb = (a.head_dim + 4 * R * kWaves - 1) / (4 * R * kWaves);
  const dim3 grid((unsigned)(pieces * a.heads * rb)), block(64 * kWaves);
  if (phase == kSsmEnds)
    hipLaunchKernelGGL((ssm_token_kernel<A, NI, R, kWhole, true, kAhead>), grid, block, 0, s, a, rb);
  else if (phase == kSsmWhole)
    hipLaunchKernelGGL((ssm_token_kernel<A, NI, R, kWhole, false, kWholeAhead>), grid, block, 0, s, a, rb);
  else
    hipLaunchKernelGGL((ssm_token_kernel<A, NI, R, kWhole, false, kAhead>), grid, block, 0, s, a, rb);
  return hipGetLastError();
}
template <typename A, int NI, int R>
hipError_t launch_lanes(hipStream_t s, const SsmArgs& a, int64_t pieces, SsmPhase phase) {
  return a.d_state == 64 * NI && a.head_dim % (16 * R) == 0 ? launch_phase<A, NI, R, true>(s, a, pieces, phase)
                                                            : launch_phase<A, NI, R, false>(s, a, pieces, phase);
}
// A wave's 4 R state rows share its loads of B and C, which bound the kernel once its waves fill the chip;
// fewer rows a wave give more waves. 16 heads of 64, d_state 128, f32, 64 rows of 4 / 12 / 32 / 64
// sequences: R = 1 14.8 / 33 / 75 / 144 us, R = 2 17.9 / 28.5 / 48 / 88, R = 4 26.7 / 30.0 / 44 / 75. So
// R = 1 while its waves have a SIMD each, R = 4 from two waves of it a SIMD on.
template <typename A, int NI>
hipError_t launch_rows(hipStream_t s, const SsmArgs& a, int64_t pieces, SsmPhase phase) {
  const int64_t waves = pieces * a.heads * ((a.head_dim + 15) / 16);  // of R = 4
  const int simds = 4 * device_cus();
  return waves >= 2 * simds  ? launch_lanes<A, NI, 4>(s, a, pieces, phase)
         : 4 * waves > simds ? launch_lanes<A, NI, 2>(s, a, pieces, phase)
                             : launch_lanes<A, NI, 1>(s, a, pieces, phase);
}
template <typename A>
hipError_t launch_state(hipStream_t s, const SsmArgs& a, int64_t pieces, SsmPhase phase) {
  switch ((a.d_state + 63) / 64) {
    case 1: return launch_rows<A, 1>(s, a, pieces, phase);
    case 2: return launch_rows<A, 2>(s, a, pieces, phase);
    default: return launch_rows<A, 4>(s, a, pieces, phase);
  }
}

}  // namespace

int32_t launch_ssm(hipStream_t s, SsmArgs& a, const SsmPlan& plan, void* ws, int dtype) {
  auto phase = [&](SsmPhase ph) {
    return plan.chunks              ? launch_ssm_chunk(s, a, plan.pieces, ph)
           : dtype == EMA_DTYPE_BF16  ? launch_state<ActBf16>(s, a, plan.pieces, ph)
           : dtype == EMA_DTYPE_F16 ? launch_state<ActF16>(s, a, plan.pieces, ph)
                                    : launch_state<ActF32>(s, a, plan.pieces, ph);
  };
  const char* what = "ema_ssm_scan launch";
  a.piece = plan.piece ? plan.piece : 1 << 30;
  if (!plan.piece) return check_hip(phase(kSsmWhole), what);
  a.carry = (float*)ws;
  a.carry_decay = a.carry + (uint64_t)plan.places * a.heads * a.head_dim * a.d_state;
  hipError_t e = phase(kSsmEnds);
  if (e != hipSuccess) return check_hip(e, what);
  const int vecs = a.heads * (a.head_dim * a.d_state / 4);
  hipLaunchKernelGGL(ssm_join_kernel, dim3((unsigned)((vecs + 255) / 256), (unsigned)a.batch), dim3(256), 0, s, a,
                     plan.chunks);
  if ((e = hipGetLastError()) != hipSuccess) return check_hip(e, what);
  return check_hip(phase(kSsmPieces), what);
}

}  // namespace ema
