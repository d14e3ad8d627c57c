// Ragged batches of the mixer calls: packed rows, the pieces of L rows that sequences are cut
// into, state slots, and typed 16-byte accesses. The integer parts are host/device functions,
// checked on the CPU (tests/cpp/test_packed.cpp).
#pragma once

#if defined(__HIPCC__)
#include "ema_common.hpp"
#endif
#include "ema_schedule.hpp"

namespace ema {

constexpr int kPackedMaxB = 4096;  // sequences of one call (two ballots find a piece's)

// Rows of sequence b: packed rows [begin, begin + n). Row starts from the device are taken as
// given only inside [0, n_rows].
struct PackedRows {
  int begin, n;
};
EMA_HD PackedRows packed_rows(int s0, int s1, int n_rows) {
  s0 = s0 < 0 ? 0 : (s0 > n_rows ? n_rows : s0);
  s1 = s1 < s0 ? s0 : (s1 > n_rows ? n_rows : s1);
  return PackedRows{s0, s1 - s0};
}

// Pieces of at most L rows. Sequence b's first piece has number starts[b] / L + b: numbers
// ascend with b and leave room for ceil(n / L) pieces of each (floor(s + n) - floor(s) + 1 is at
// least that many), so that a piece's sequence is found by a search over the row starts alone,
// and the numbers stay below n_rows / L + batch. Some numbers have no rows.
EMA_HD int packed_first_piece(int s0, int b, int L) { return (int)((uint32_t)s0 / (uint32_t)L) + b; }
// The sequence of piece number `index` where all have T rows: the last b with b T / L + b <= index,
// that is b (T + L) < (index + 1) L.
EMA_HD int packed_uniform_sequence(int index, int T, int L, int batch) {
  const int64_t b = ((int64_t)index * L + L - 1) / ((int64_t)T + L);
  return b < batch ? (int)b : batch - 1;
}
EMA_HD int64_t packed_pieces(int n_rows, int batch, int L) { return (int64_t)n_rows / L + batch; }
// Places of what the pieces of longer sequences (more than L rows: two pieces and more) hand on to each
// other: sequence b's are consecutive from q + min(b, q) on, with q = starts[b] / L, so that sequences
// of one piece take none. They do not meet: from start s to end e of a sequence of k L + r rows (0 < r <= L)
// q grows by k at least, and where by no more than k, the minimum by one (b does, and q), which
// makes the k + 1 places that its pieces need; all lie below the same of n_rows and batch.
EMA_HD int packed_first_place(int s0, int b, int L) {
  const int q = (int)((uint32_t)s0 / (uint32_t)L);
  return q + (b < q ? b : q);
}
EMA_HD int64_t packed_places(int n_rows, int batch, int L) {
  const int64_t q = n_rows / L;
  return q + (batch < q ? batch : q);
}

}  // namespace ema

#if defined(__HIPCC__)
namespace ema {

// One piece: sequence b's rows [row, row + n) of its [begin, begin + all); piece number `first` is
// the sequence's first. n = 0: nothing to do.
struct Piece {
  int b, begin, all, row, n, index, first;
};

typedef const __attribute__((address_space(4))) int32_t packed_cint;
__device__ __forceinline__ int packed_ld(const int32_t* p, int64_t i) { return ((packed_cint*)p)[i]; }

// Rows of sequence b (uniform over the wave). starts null: T rows each.
__device__ __forceinline__ PackedRows packed_sequence(const int32_t* starts, int b, int n_rows, int T) {
  if (!starts) return PackedRows{b * T, T};
  return packed_rows(packed_ld(starts, b), packed_ld(starts, b + 1), n_rows);
}

// Piece number `index` (uniform over the wave).
__device__ __forceinline__ Piece packed_piece(const int32_t* starts, int batch, int n_rows, int T, int L, int index) {
  Piece p;
  p.index = index;
  p.b = 0;
  if (!starts) {  // uniform rows: the same search, by a division
    p.b = packed_uniform_sequence(index, T, L, batch);
  } else if (batch > 1) {
    const int lane = threadIdx.x & 63;
    const int step = (batch + 63) >> 6;
    const int i = lane * step;
    const int ii = i < batch ? i : 0;
    int s = starts[ii];
    s = s < 0 ? 0 : (s > n_rows ? n_rows : s);
    uint64_t le = __ballot(i < batch && packed_first_piece(s, ii, L) <= index);
    int b = le ? (63 - __builtin_clzll(le)) * step : 0;
    if (step > 1) {
      const int j = b + lane;
      const bool in = lane < step && j < batch;
      s = starts[in ? j : 0];
      s = s < 0 ? 0 : (s > n_rows ? n_rows : s);
      le = __ballot(in && packed_first_piece(s, j, L) <= index);
      b += le ? 63 - __builtin_clzll(le) : 0;
    }
    p.b = __builtin_amdgcn_readfirstlane(b);
  }
  const PackedRows r = packed_sequence(starts, p.b, n_rows, T);
  p.begin = r.begin;
  p.all = r.n;
  p.first = packed_first_piece(r.begin, p.b, L);
  const int64_t at = (int64_t)(index - p.first) * L;
  if (index < p.first || at >= r.n) {
    p.row = r.begin;
    p.n = 0;
  } else {
    p.row = r.begin + (int)at;
    p.n = r.n - (int)at < L ? r.n - (int)at : L;
  }
  return p;
}

// Slot of sequence b, or -1; and whether what it holds is the start.
__device__ __forceinline__ int packed_slot(const int32_t* slots, int b, int n_slots) {
  const int s = slots ? packed_ld(slots, b) : b;
  return (uint32_t)s < (uint32_t)n_slots ? s : -1;
}
__device__ __forceinline__ bool packed_continues(const int32_t* offsets, int b) {
  return !offsets || packed_ld(offsets, b) > 0;
}

// Activation element types.
struct ActBf16 {
  typedef uint16_t T;
  static __device__ __forceinline__ float to(uint16_t v) { return bf16_to_f32(v); }
  static __device__ __forceinline__ uint16_t from(float v) { return (uint16_t)f32_to_bf16_bits(v); }
};
struct ActF16 {
  typedef uint16_t T;
  static __device__ __forceinline__ float to(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ uint16_t from(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};
struct ActF32 {
  typedef float T;
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};

// V consecutive elements, V = 8 or 4 (16- or 8-byte aligned) or 1.
template <typename A, int V>
struct Vec {
  typedef typename A::T T;
  T v[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V * sizeof(T) >= 16) {
#pragma unroll
      for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i) ((u32x4*)v)[i] = ((const u32x4*)p)[i];
    } else if constexpr (V * sizeof(T) == 8) {
      *(u32x2*)v = *(const u32x2*)p;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V * sizeof(T) >= 16) {
#pragma unroll
      for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i) ((u32x4*)p)[i] = ((const u32x4*)v)[i];
    } else if constexpr (V * sizeof(T) == 8) {
      *(u32x2*)p = *(const u32x2*)v;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = v[i];
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return A::to(v[i]); }
  __device__ __forceinline__ void set(int i, float x) { v[i] = A::from(x); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = T(0);
  }
};

__device__ __forceinline__ float sigmoid_(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

}  // namespace ema
#endif
