// Short causal convolution over time, one filter of W taps per channel, gfx950.
//
//   v[t, c] = bias[c] + sum_j w[c, j] x[t - W + 1 + j, c],   y = v or v * sigmoid(v)
//
// over the packed rows of a ragged batch; rows before a sequence's first come from its kept state,
// its last W - 1 inputs. Every channel is alone, so a lane takes V neighbouring channels (16 bytes
// of bf16) down a piece of L rows of one sequence, the last W - 1 rows in registers: each input is
// loaded once, W - 1 rows of each piece once more. The piece that begins a sequence also writes its
// new state, whose old rows its lanes have read themselves, so no other lane reads what it writes.
//
// HBM-bound: 7617 rows of 6144 bf16 channels, 188 MB, in 42.6 us (4.4 TB/s; a copy of 512 MB runs at
// 5.3). Stores past the caches take 37 us, but the scan that reads y next takes longer by more:
// convolution, scan and norms of 8192 rows 276 us against 267. Pieces of 16 or 64 rows, 4 or 16 rows
// loaded ahead, workgroups of 256 lanes: within 5 %, none faster. A token's call is 3.5 us, the launch.
#include "packed.hpp"

namespace ema {
namespace {

constexpr int kRows = 32;    // rows of a piece
constexpr int kBatch = 8;    // rows loaded ahead of their sums
constexpr int kLanes = 64;   // lanes of a workgroup

template <typename A, int W, int V>
__global__ __launch_bounds__(kLanes) void causal_conv_kernel(CausalConvArgs a) {
  typedef typename A::T T;
  const Piece p = packed_piece(a.starts, a.batch, a.n_rows, a.T, kRows, (int)blockIdx.x);
  if (p.n == 0) return;
  const int c = (blockIdx.y * kLanes + threadIdx.x) * V;
  if (c >= a.channels) return;
  const T* const x = (const T*)a.x + c;
  T* const y = (T*)a.y + (int64_t)p.row * a.ldy + c;

  float w[W][V], bias[V];
  {
    T raw[V * W];
    const T* const wp = (const T*)a.w + (int64_t)c * W;
    if constexpr (V > 1) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        Vec<A, V> t;
        t.load(wp + i * V);
#pragma unroll
        for (int e = 0; e < V; ++e) raw[i * V + e] = t.v[e];
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) raw[i] = wp[i];
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
#pragma unroll
      for (int j = 0; j < W; ++j) w[j][e] = A::to(raw[e * W + j]);
    Vec<A, V> t;
    t.zero();
    if (a.bias) t.load((const T*)a.bias + c);
#pragma unroll
    for (int e = 0; e < V; ++e) bias[e] = t[e];
  }

  // the W - 1 rows before the piece
  Vec<A, V> win[W - 1];
  const int at = p.row - p.begin;
  const int slot = a.state ? packed_slot(a.slots, p.b, a.n_slots) : -1;
  const bool kept = slot >= 0 && packed_continues(a.offsets, p.b);
  T* const st = (T*)a.state + (int64_t)slot * (W - 1) * a.channels + c;
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    const int t = at - (W - 1) + j;  // (a piece after the first begins at least kRows >= W - 1 rows in)
    if (t >= 0)
      win[j].load(x + (int64_t)(p.begin + t) * a.ldx);
    else if (kept)
      win[j].load(st + (int64_t)j * a.channels);
    else
      win[j].zero();
  }
  if (at == 0 && slot >= 0) {
    // row i of the new state is row n + i of (old state, the sequence's rows)
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
      const int t = p.all - (W - 1) + i;
      Vec<A, V> r;
      if (t >= 0) {
        r.load(x + (int64_t)(p.begin + t) * a.ldx);
      } else {
        r = win[W - 2];
#pragma unroll
        for (int j = 0; j < W - 2; ++j)
          if (j == p.all + i) r = win[j];
      }
      r.store(st + (int64_t)i * a.channels);
    }
  }

  auto row = [&](const Vec<A, V>& now, T* out) __attribute__((always_inline)) {
    Vec<A, V> o;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float v = bias[e];
#pragma unroll
      for (int j = 0; j < W - 1; ++j) v = fmaf(w[j][e], win[j][e], v);
      v = fmaf(w[W - 1][e], now[e], v);
      o.set(e, a.silu ? v * sigmoid_(v) : v);
    }
    o.store(out);
#pragma unroll
    for (int j = 0; j < W - 2; ++j) win[j] = win[j + 1];
    win[W - 2] = now;
  };
  const T* in = x + (int64_t)p.row * a.ldx;
  int t = 0;
  for (; t + kBatch <= p.n; t += kBatch) {
    Vec<A, V> now[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) now[i].load(in + (int64_t)(t + i) * a.ldx);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) row(now[i], y + (int64_t)(t + i) * a.ldy);
  }
  for (; t < p.n; ++t) {
    Vec<A, V> now;
    now.load(in + (int64_t)t * a.ldx);
    row(now, y + (int64_t)t * a.ldy);
  }
}

template <typename A, int W, int V>
hipError_t launch_v(hipStream_t s, const CausalConvArgs& a) {
  const dim3 grid((unsigned)packed_pieces(a.n_rows, a.batch, kRows), (unsigned)((a.channels + kLanes * V - 1) / (kLanes * V)));
  hipLaunchKernelGGL((causal_conv_kernel<A, W, V>), grid, dim3(kLanes), 0, s, a);
  return hipGetLastError();
}
template <typename A, int V>
hipError_t launch_w(hipStream_t s, const CausalConvArgs& a) {
  return a.width == 4 ? launch_v<A, 4, V>(s, a) : a.width == 3 ? launch_v<A, 3, V>(s, a) : launch_v<A, 2, V>(s, a);
}
// 16-byte accesses where every row of x, y and the state begins at a multiple of them (and so do
// the taps and the bias); else one channel a lane.
template <typename A, int V>
hipError_t launch_a(hipStream_t s, const CausalConvArgs& a) {
  const uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.w | (uintptr_t)a.bias | (uintptr_t)a.state;
  const bool wide = !(at & 15u) && !(a.channels % V) && !(a.ldx % V) && !(a.ldy % V);
  return wide ? launch_w<A, V>(s, a) : launch_w<A, 1>(s, a);
}

}  // namespace

int32_t launch_causal_conv(hipStream_t s, const CausalConvArgs& a, int dtype) {
  const hipError_t e = dtype == EMA_DTYPE_BF16  ? launch_a<ActBf16, 8>(s, a)
                       : dtype == EMA_DTYPE_F16 ? launch_a<ActF16, 8>(s, a)
                                                : launch_a<ActF32, 4>(s, a);
  return check_hip(e, "ema_causal_conv launch");
}

}  // namespace ema
