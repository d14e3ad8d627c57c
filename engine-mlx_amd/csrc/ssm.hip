// Selective state space scan, one decay per head, token by token; the plan of all its kernels.
//
// Lane layout: 16 lanes share a state row (one value of head_dim); lane p holds its elements
// n = 4 p + 64 i + j (i < NI, j < 4), so a 16-byte state access of a wave covers 256 contiguous
// bytes of each of 4 rows, and y is a sum of 4 NI products and four DPP steps. A wave holds R
// times 4 rows, which share the lane's B and C values. The state stays in registers over the rows of
// the piece; the next row's inputs are loaded under this one's sums.
// One row (a decode step): HBM-bound, 8 bytes of state traffic per element against 6 flops: 32 users of
// 64 heads of 64, d_state 128, 135 MB in 22 us (6.1 TB/s). Many rows: bound by the vector instructions
// of a row, 0.44 us a row for one sequence of 24 heads in f32, and cut in time as long as that
// fills the chip (2048 rows 137 us; whole 913).
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

template <typename A, int NI, int R, int PHASE>
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
  if (PHASE == kSsmEnds && last) return;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int p = lane & 15;
  const int row0 = (rb * kWaves + wave) * 4 * R + (lane >> 4);  // rows row0 + 4 i
  const int N = a.d_state, P = a.head_dim;
  const int g = h / (a.heads / a.groups);
  const int slot = packed_slot(a.slots, pc.b, a.n_slots);
  float* const pool = a.state + ((int64_t)slot * a.heads + h) * P * N;
  float* const carry = a.carry + ((int64_t)index * a.heads + h) * P * N;

  bool on[NI];
#pragma unroll
  for (int k = 0; k < NI; ++k) on[k] = 4 * p + 64 * k < N;
  f32x4 s[R][NI];
  {
    // a sequence of one piece starts from the pool; pieces of a longer one never read what its
    // last piece writes there
    const float* from = nullptr;
    if (PHASE == kSsmPieces && pc.all > a.piece)
      from = carry;
    else if (PHASE != kSsmEnds && slot >= 0 && packed_continues(a.offsets, pc.b))
      from = pool;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int k = 0; k < NI; ++k) {
        s[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (from && row0 + 4 * i < P && on[k]) s[i][k] = *(const f32x4*)(from + (int64_t)(row0 + 4 * i) * N + 4 * p + 64 * k);
      }
  }
  const float A_h = a.a[h], D_h = a.d ? a.d[h] : 0.f, bias = a.dt_bias ? a.dt_bias[h] : 0.f;
  const T* const xp = (const T*)a.x + (int64_t)pc.row * a.ldx + h * P + row0;
  const T* const bp = (const T*)a.b + (int64_t)pc.row * a.ldb + g * N + 4 * p;
  const T* const cp = (const T*)a.c + (int64_t)pc.row * a.ldc + g * N + 4 * p;
  const T* const dp = (const T*)a.dt + (int64_t)pc.row * a.lddt + h;
  T* const yp = (T*)a.y + (int64_t)pc.row * a.ldy + h * P + row0;

  struct Row {
    Vec<A, 4> b[NI], c[NI];
    T x[R];
  };
  auto fetch = [&](int t, Row& r) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < R; ++i) r.x[i] = row0 + 4 * i < P ? xp[(int64_t)t * a.ldx + 4 * i] : T(0);
#pragma unroll
    for (int k = 0; k < NI; ++k) {
      r.b[k].zero();
      r.c[k].zero();
      if (on[k]) {
        r.b[k].load(bp + (int64_t)t * a.ldb + 64 * k);
        if (PHASE != kSsmEnds) r.c[k].load(cp + (int64_t)t * a.ldc + 64 * k);
      }
    }
  };
  // the steps of 64 rows, a row a lane
  T raw = dp[(int64_t)(lane < pc.n ? lane : pc.n - 1) * a.lddt];
  float steps = 0.f, decays = 0.f, sum = 0.f;
  Row now, next;
  fetch(0, now);
  for (int t = 0; t < pc.n; ++t) {
    if (t + 1 < pc.n) fetch(t + 1, next);
    if ((t & 63) == 0) {
      steps = ssm_step(A::to(raw) + bias, a);
      decays = steps * A_h;
      if (PHASE == kSsmEnds) sum += t + lane < pc.n ? decays : 0.f;
      decays = expf(decays);
      const int at = t + 64 + lane;
      if (t + 64 < pc.n) raw = dp[(int64_t)(at < pc.n ? at : pc.n - 1) * a.lddt];
    }
    const float d = lane_value(steps, t & 63), decay = lane_value(decays, t & 63);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float xv = A::to(now.x[i]);
      const float dx = d * xv;
      float y = 0.f;
#pragma unroll
      for (int k = 0; k < NI; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][k][j] = fmaf(dx, now.b[k][j], decay * s[i][k][j]);
          if (PHASE != kSsmEnds) y = fmaf(s[i][k][j], now.c[k][j], y);
        }
      if (PHASE != kSsmEnds) {
        y = fmaf(D_h, xv, row_sum16(y));
        if (p == 0 && row0 + 4 * i < P) yp[(int64_t)t * a.ldy + 4 * i] = A::from(y);
      }
    }
    now = next;
  }
  float* const to = PHASE == kSsmEnds ? carry : (last && slot >= 0 ? pool : nullptr);
  if (to)
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int k = 0; k < NI; ++k)
        if (row0 + 4 * i < P && on[k]) *(f32x4*)(to + (int64_t)(row0 + 4 * i) * N + 4 * p + 64 * k) = s[i][k];
  if (PHASE == kSsmEnds && rb == 0 && wave == 0) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m, 64);
    if (lane == 0) a.carry_decay[(int64_t)index * a.heads + h] = expf(sum);
  }
}

// Joins a sequence's pieces in order: each piece's E in the workspace becomes its start state.
// A lane per 4 elements of (head, state); the pieces' loads do not depend on the sums.
__global__ __launch_bounds__(256) void ssm_join_kernel(SsmArgs a, bool chunks) {
  const int b = blockIdx.y;
  const PackedRows r = packed_sequence(a.starts, b, a.n_rows, a.T);
  if (r.n <= a.piece) return;
  const int per_head = a.head_dim * a.d_state / 4;
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= a.heads * per_head) return;
  const int h = v / per_head;
  const int first = packed_first_piece(r.begin, b, a.piece), n = (r.n + a.piece - 1) / a.piece;
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

template <typename A, int NI, int R>
hipError_t launch_phase(hipStream_t s, const SsmArgs& a, int64_t pieces, SsmPhase phase) {
  const int rb = (a.head_dim + 4 * R * kWaves - 1) / (4 * R * kWaves);
  const dim3 grid((unsigned)(pieces * a.heads * rb)), block(64 * kWaves);
  if (phase == kSsmWhole)
    hipLaunchKernelGGL((ssm_token_kernel<A, NI, R, kSsmWhole>), grid, block, 0, s, a, rb);
  else if (phase == kSsmEnds)
    hipLaunchKernelGGL((ssm_token_kernel<A, NI, R, kSsmEnds>), grid, block, 0, s, a, rb);
  else
    hipLaunchKernelGGL((ssm_token_kernel<A, NI, R, kSsmPieces>), grid, block, 0, s, a, rb);
  return hipGetLastError();
}
template <typename A, int NI>
hipError_t launch_rows(hipStream_t s, const SsmArgs& a, int64_t pieces, SsmPhase phase) {
  // 64 state rows a workgroup where that gives the chip two of them per CU, else 16
  const int64_t wgs = pieces * a.heads * ((a.head_dim + 63) / 64);
  return wgs >= 2 * device_cus() ? launch_phase<A, NI, 4>(s, a, pieces, phase) : launch_phase<A, NI, 1>(s, a, pieces, phase);
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

SsmPlan plan_ssm(int batch, int n_rows, int max_rows, int heads, int head_dim, int d_state, int groups, int dtype,
                 bool vectors, uint64_t ws_bytes) {
  SsmPlan p{};
  p.chunks = dtype == EMA_DTYPE_BF16 && vectors && max_rows >= 32 && ssm_chunk_shape(head_dim, d_state);
  p.pieces = batch;
  // Cut where the sequences' heads leave much of the chip idle: into pieces that give every CU two
  // (chunks) or four workgroups. Chunks, 64 heads of 64, d_state 128: a whole sequence takes 0.065 us
  // a row of the longest, cut ones 25 us and 0.0105 us a row of all (ends, joining, pieces), so that
  // the longest has to be 384 rows and 2.6 pieces: 4 x 2048 rows 106 us cut, 133 whole, 5 x 1638
  // 123 and 106, 512 rows 33 and 37, 256 the same. Token by token (f32): 8 x 300 rows of 24 heads
  // 164 cut, 173 whole, 2048 rows 150 and 948.
  const int per_cu = p.chunks ? 2 : 4, step = p.chunks ? kSsmChunk : 16, least = p.chunks ? 4 * kSsmChunk : 32;
  const int64_t wgs = p.chunks ? (int64_t)ssm_chunk_workgroups(heads, head_dim, groups)
                               : heads * (int64_t)((head_dim + 63) / 64);
  const int64_t even = (n_rows * wgs + per_cu * device_cus() - 1) / (per_cu * device_cus());
  if ((int64_t)max_rows * 5 < even * 13 + (p.chunks ? 1920 : 320)) return p;
  int64_t piece = even < least ? least : (even + step - 1) / step * step;
  for (; piece < max_rows; piece *= 2) {
    const int64_t pieces = packed_pieces(n_rows, batch, (int)piece);
    const uint64_t bytes = (uint64_t)pieces * heads * ((uint64_t)head_dim * d_state + 4) * 4;
    if (bytes > ws_bytes) continue;
    p.piece = (int)piece;
    p.pieces = pieces;
    p.bytes = bytes;
    break;
  }
  return p;
}

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
  a.carry_decay = a.carry + (uint64_t)plan.pieces * a.heads * a.head_dim * a.d_state;
  hipError_t e = phase(kSsmEnds);
  if (e != hipSuccess) return check_hip(e, what);
  const int vecs = a.heads * (a.head_dim * a.d_state / 4);
  hipLaunchKernelGGL(ssm_join_kernel, dim3((unsigned)((vecs + 255) / 256), (unsigned)a.batch), dim3(256), 0, s, a,
                     plan.chunks);
  if ((e = hipGetLastError()) != hipSuccess) return check_hip(e, what);
  return check_hip(phase(kSsmPieces), what);
}

}  // namespace ema
