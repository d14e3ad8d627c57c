// RMS norms with a gate or around the residual stream, gfx950.
//
//   gated:     y = norm(x) w act(gate), or norm(x act(gate)) w, over groups of a row's values
//   residual:  u = norm(branch) post_w;  h = residual + scale gate u;  out = norm(h) pre_w
//   norm(u) = u / sqrt(mean u^2 + eps)
//
// HBM-bound: each value is read once and written once. The values of a norm stay in registers
// between the sum of squares and the products, in vectors of 8 neighbours a lane (16 bytes of
// bf16), so that nothing is read twice. Up to 512 values a sub-wave of 8 to 64 lanes takes a norm
// (a head's 128 values: 16 lanes), more are a workgroup's. Sizes, strides or addresses that do not
// allow vectors go value by value in the same kernels (V = 1).
//
// Gated, 8192 rows of 4096 bf16 in groups of 512: 36.8 us, 5.5 TB/s; residual with two norms, a gate and
// a 32-bit stream, 8192 x 4096: 88 us, 5.3 TB/s (a copy of 512 MB: 5.3). Value by value, rows of 1111 bf16:
// 2.9 TB/s: a lane's access is 2 bytes there, and rows that begin at odd elements allow no more for all of
// them; a head and a tail around 16-byte pieces was not built, as widths of layers are multiples of 8.
// One row: 2.3 us, the launch.
#include <type_traits>

#include "packed.hpp"

namespace ema {
namespace {

template <int LPG>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int m = LPG / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}
// Sum over a workgroup; `part` holds a value per wave and is free again after the next barrier.
template <int THREADS>
__device__ __forceinline__ float group_sum(float v, float* part) {
  v = lanes_sum<64>(v);
  if constexpr (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) v += part[i];
  }
  return v;
}

__device__ __forceinline__ float act(float g, uint32_t flags) {
  const float s = sigmoid_(g);
  return flags & EMA_NORM_GATE_SIGMOID ? s : g * s;
}
template <typename A, int V>
__device__ __forceinline__ float weight(const Vec<A, V>& w, int e, uint32_t flags) {
  return flags & EMA_NORM_UNIT_OFFSET ? 1.0f + w[e] : w[e];
}

// ------------------------------------------------------------------ gated
// One vector of 8 of the norms numbered `id` (row-major over rows and their groups) per lane.
template <typename A, int LPG>
__global__ __launch_bounds__(256) void gated_small_kernel(GatedNormArgs a) {
  typedef typename A::T T;
  const uint32_t id = blockIdx.x * (256 / LPG) + threadIdx.x / LPG;
  if (id >= (uint32_t)a.n_rows * (uint32_t)a.groups) return;  // (a whole sub-wave)
  const uint32_t row = id / (uint32_t)a.groups, g = id - row * (uint32_t)a.groups;
  const int e0 = (threadIdx.x % LPG) * 8;
  const bool on = e0 < a.group;
  const int at = (int)g * a.group + e0;
  Vec<A, 8> x, z, w;
  x.zero();
  z.zero();
  w.zero();
  if (on) {
    x.load((const T*)a.x + (int64_t)row * a.ldx + at);
    if (a.gate) z.load((const T*)a.gate + (int64_t)row * a.ldg + at);
    if (a.w) w.load((const T*)a.w + (a.flags & EMA_NORM_SHARED_WEIGHT ? e0 : at));
  }
  float u[8], k[8], ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    k[e] = a.gate ? act(z[e], a.flags) : 1.0f;
    u[e] = a.flags & EMA_NORM_GATE_FIRST ? x[e] * k[e] : x[e];
    ss = fmaf(u[e], u[e], ss);
  }
  ss = lanes_sum<LPG>(ss);
  const float inv = 1.0f / sqrtf(ss / (float)a.group + a.eps);
  if (!on) return;
  Vec<A, 8> y;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float v = u[e] * inv;
    if (a.w) v *= weight(w, e, a.flags);
    y.set(e, a.flags & EMA_NORM_GATE_FIRST ? v : v * k[e]);
  }
  y.store((T*)a.y + (int64_t)row * a.ldy + at);
}

// A workgroup per norm.
template <typename A, int V, int THREADS, int N>
__global__ __launch_bounds__(THREADS) void gated_kernel(GatedNormArgs a) {
  typedef typename A::T T;
  __shared__ float part[THREADS / 64];
  const uint32_t row = blockIdx.x / (uint32_t)a.groups, g = blockIdx.x - row * (uint32_t)a.groups;
  const int at = (int)g * a.group;
  const T* const xp = (const T*)a.x + (int64_t)row * a.ldx + at;
  const T* const zp = (const T*)a.gate + (int64_t)row * a.ldg + at;
  Vec<A, V> x[N], z[N];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = (i * THREADS + threadIdx.x) * V;
    x[i].zero();
    z[i].zero();
    if (e < a.group) {
      x[i].load(xp + e);
      if (a.gate) z[i].load(zp + e);
    }
  }
  float u[N][V], k[N][V];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      k[i][e] = a.gate ? act(z[i][e], a.flags) : 1.0f;
      u[i][e] = a.flags & EMA_NORM_GATE_FIRST ? x[i][e] * k[i][e] : x[i][e];
      ss = fmaf(u[i][e], u[i][e], ss);
    }
  const float inv = 1.0f / sqrtf(group_sum<THREADS>(ss, part) / (float)a.group + a.eps);
  const T* const wp = (const T*)a.w + (a.flags & EMA_NORM_SHARED_WEIGHT ? 0 : at);
  T* const yp = (T*)a.y + (int64_t)row * a.ldy + at;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = (i * THREADS + threadIdx.x) * V;
    if (e >= a.group) continue;
    Vec<A, V> w, y;
    if (a.w) w.load(wp + e);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float v = u[i][j] * inv;
      if (a.w) v *= weight(w, j, a.flags);
      y.set(j, a.flags & EMA_NORM_GATE_FIRST ? v : v * k[i][j]);
    }
    y.store(yp + e);
  }
}

// ------------------------------------------------------------------ residual
// A workgroup per row. S: the type of the residual stream.
template <typename A, typename S, int V, int THREADS, int N>
__global__ __launch_bounds__(THREADS) void residual_kernel(ResidualNormArgs a) {
  typedef typename A::T T;
  typedef typename S::T R;
  __shared__ float part[2][THREADS / 64];
  const int64_t row = blockIdx.x;
  const T* const bp = (const T*)a.branch + row * a.ldx;
  const T* const gp = (const T*)a.gate + row * a.ldg;
  R* const rp = (R*)a.residual + row * a.ldr;
  Vec<A, V> b[N], g[N];
  Vec<S, V> r[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = (i * THREADS + threadIdx.x) * V;
    b[i].zero();
    g[i].zero();
    r[i].zero();
    if (e < a.dim) {
      b[i].load(bp + e);
      r[i].load(rp + e);
      if (a.gate) g[i].load(gp + e);
    }
  }
  float scale = a.scale;
  if (a.post_w) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) ss = fmaf(b[i][j], b[i][j], ss);
    scale *= 1.0f / sqrtf(group_sum<THREADS>(ss, part[0]) / (float)a.dim + a.eps);
  }
  float h[N][V], ss = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = (i * THREADS + threadIdx.x) * V;
    Vec<A, V> w;
    w.zero();
    if (a.post_w && e < a.dim) w.load((const T*)a.post_w + e);
    Vec<S, V> o;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float u = b[i][j] * scale;
      if (a.post_w) u *= weight(w, j, a.flags);
      if (a.gate) u *= g[i][j];
      h[i][j] = e < a.dim ? r[i][j] + u : 0.f;
      ss = fmaf(h[i][j], h[i][j], ss);
      o.set(j, h[i][j]);
    }
    if (e < a.dim) o.store(rp + e);
  }
  if (!a.out) return;
  const float inv = 1.0f / sqrtf(group_sum<THREADS>(ss, part[1]) / (float)a.dim + a.eps);
  T* const op = (T*)a.out + row * a.ldo;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = (i * THREADS + threadIdx.x) * V;
    if (e >= a.dim) continue;
    Vec<A, V> w, o;
    w.load((const T*)a.pre_w + e);
#pragma unroll
    for (int j = 0; j < V; ++j) o.set(j, h[i][j] * inv * weight(w, j, a.flags));
    o.store(op + e);
  }
}

// Calls f(threads, vectors a lane) with the smallest workgroup whose lanes hold n values.
template <int THREADS, int N>
struct Shape {
  static constexpr int kThreads = THREADS, kN = N;
};
template <typename F>
hipError_t with_shape(int n, bool wide, F f) {
  if (wide) {
    if (n <= 64 * 8) return f(std::integral_constant<int, 8>(), Shape<64, 1>());
    if (n <= 256 * 8) return f(std::integral_constant<int, 8>(), Shape<256, 1>());
    if (n <= 256 * 16) return f(std::integral_constant<int, 8>(), Shape<256, 2>());
    if (n <= 512 * 16) return f(std::integral_constant<int, 8>(), Shape<512, 2>());
    return f(std::integral_constant<int, 8>(), Shape<1024, 2>());
  }
  if (n <= 64 * 8) return f(std::integral_constant<int, 1>(), Shape<64, 8>());
  if (n <= 256 * 8) return f(std::integral_constant<int, 1>(), Shape<256, 8>());
  if (n <= 1024 * 8) return f(std::integral_constant<int, 1>(), Shape<1024, 8>());
  return f(std::integral_constant<int, 1>(), Shape<1024, 16>());
}

template <typename A>
hipError_t launch_gated(hipStream_t s, const GatedNormArgs& a) {
  const uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.gate | (uintptr_t)a.w | (uintptr_t)a.y;
  const bool wide = !(at & 15u) && !(a.group % 8) && !(a.ldx % 8) && !(a.ldg % 8) && !(a.ldy % 8);
  const int64_t norms = (int64_t)a.n_rows * a.groups;
  if (wide && a.group <= 512) {
    auto small = [&](auto lpg) {
      constexpr int L = decltype(lpg)::value;
      hipLaunchKernelGGL((gated_small_kernel<A, L>), dim3((unsigned)((norms + 256 / L - 1) / (256 / L))), dim3(256), 0,
                         s, a);
      return hipGetLastError();
    };
    if (a.group <= 64) return small(std::integral_constant<int, 8>());
    if (a.group <= 128) return small(std::integral_constant<int, 16>());
    if (a.group <= 256) return small(std::integral_constant<int, 32>());
    return small(std::integral_constant<int, 64>());
  }
  return with_shape(a.group, wide, [&](auto v, auto shape) {
    typedef decltype(shape) Sh;
    hipLaunchKernelGGL((gated_kernel<A, decltype(v)::value, Sh::kThreads, Sh::kN>), dim3((unsigned)norms),
                       dim3(Sh::kThreads), 0, s, a);
    return hipGetLastError();
  });
}

template <typename A, typename S>
hipError_t launch_residual(hipStream_t s, const ResidualNormArgs& a) {
  const uintptr_t at = (uintptr_t)a.branch | (uintptr_t)a.gate | (uintptr_t)a.post_w | (uintptr_t)a.pre_w |
                       (uintptr_t)a.residual | (uintptr_t)a.out;
  const bool wide = !(at & 15u) && !(a.dim % 8) && !(a.ldx % 8) && !(a.ldg % 8) && !(a.ldr % 8) && !(a.ldo % 8);
  return with_shape(a.dim, wide, [&](auto v, auto shape) {
    typedef decltype(shape) Sh;
    hipLaunchKernelGGL((residual_kernel<A, S, decltype(v)::value, Sh::kThreads, Sh::kN>), dim3((unsigned)a.n_rows),
                       dim3(Sh::kThreads), 0, s, a);
    return hipGetLastError();
  });
}

}  // namespace

int32_t launch_gated_norm(hipStream_t s, const GatedNormArgs& a, int dtype) {
  const hipError_t e = dtype == EMA_DTYPE_BF16  ? launch_gated<ActBf16>(s, a)
                       : dtype == EMA_DTYPE_F16 ? launch_gated<ActF16>(s, a)
                                                : launch_gated<ActF32>(s, a);
  return check_hip(e, "ema_gated_norm launch");
}

int32_t launch_residual_norm(hipStream_t s, const ResidualNormArgs& a, int dtype, int residual_dtype) {
  hipError_t e;
  if (dtype == EMA_DTYPE_F32)
    e = launch_residual<ActF32, ActF32>(s, a);
  else if (residual_dtype == EMA_DTYPE_F32)
    e = dtype == EMA_DTYPE_BF16 ? launch_residual<ActBf16, ActF32>(s, a) : launch_residual<ActF16, ActF32>(s, a);
  else
    e = dtype == EMA_DTYPE_BF16 ? launch_residual<ActBf16, ActBf16>(s, a) : launch_residual<ActF16, ActF16>(s, a);
  return check_hip(e, "ema_residual_norm launch");
}

}  // namespace ema
