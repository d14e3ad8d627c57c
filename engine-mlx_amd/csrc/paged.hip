// Paged KV cache for gfx950: append with norm and rotation, and attention over pages.
//
// The pages are a pool [n_pages, Hkv, P, D] (an ema_kvcache_desc of n_pages rows of P
// positions, P a power of two >= 16); sequence b's position p lies in slot p % P of page
// table[b][p / P]. A table entry outside [0, n_pages) is never followed: nothing is written
// there, and its positions read as zero rows. A batch is ragged: sequence b's query rows are
// packed rows [starts[b], starts[b + 1]).
#include <type_traits>

#include "ema_common.hpp"
#include "paged.hpp"

namespace ema {
namespace {

// ------------------------------------------------------------------ append
// One workgroup per packed row, its groups of 8 lanes over the row's heads, as in the static
// cache's pre-attention kernel (8 lanes hold a head: lane j elements jE.. of both halves, so a
// rotated pair sits in one lane). Everything up to the store is in 32 bits, and a value is
// rounded once, when it is stored (the static cache's kernel rounds after the norm and after
// the weight as well, as the reference's separate operators do). The angle pos * theta^(-2i/D)
// is formed and reduced to a fraction of a turn in 64 bits: in 32 bits it is off by 0.004 at
// position 100000, half a bf16 step of the result.
// HBM-bound: each byte of qkv is read once, q, k and v written once: 11435 rows of 48 heads, 281 MB,
// in 54 us (5.2 TB/s; a large device copy 4.9). Loads past the caches gain nothing (55.5 us).
template <int E>
__device__ __forceinline__ void load_row(const uint16_t* p, float (&x)[E]) {
  if constexpr (E == 4) {
    const u32x2 w = *(const u32x2*)p;
#pragma unroll
    for (int i = 0; i < 2; ++i) x[2 * i] = bf16_lo(w[i]), x[2 * i + 1] = bf16_hi(w[i]);
  } else {
#pragma unroll
    for (int c = 0; c < E / 8; ++c) {
      const u32x4 w = ((const u32x4*)p)[c];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[8 * c + 2 * i] = bf16_lo(w[i]), x[8 * c + 2 * i + 1] = bf16_hi(w[i]);
    }
  }
}
template <int E>
__device__ __forceinline__ void store_row(uint16_t* p, const float (&x)[E]) {
  if constexpr (E == 4) {
    *(u32x2*)p = u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
  } else {
#pragma unroll
    for (int c = 0; c < E / 8; ++c)
      ((u32x4*)p)[c] = u32x4{pack_bf16x2(x[8 * c], x[8 * c + 1]), pack_bf16x2(x[8 * c + 2], x[8 * c + 3]),
                             pack_bf16x2(x[8 * c + 4], x[8 * c + 5]), pack_bf16x2(x[8 * c + 6], x[8 * c + 7])};
  }
}

struct AppendArgs {
  const uint16_t* qkv;
  const uint16_t* qw;
  const uint16_t* kw;
  const int32_t* off;
  const int32_t* starts;  // null: T rows per sequence
  const int32_t* prefix;  // null: 0
  const int32_t* table;
  uint16_t* q_out;
  void* k;
  void* v;
  int8_t* kexp;
  int8_t* vexp;
  int64_t sb, sh, sp;  // elements (fp8: bytes)
  double log2_theta;
  float eps;
  int B, T, n_rows, Hq, Hkv, cols, shift, n_pages;
  uint32_t flags;
};

// Sequence of packed row r: the last b with starts[b] <= r (lane-parallel, at most two loads
// for up to 4096 sequences).
__device__ __forceinline__ int sequence_of(const int32_t* starts, int B, int r) {
  const int lane = threadIdx.x & 63;
  const int step = (B + 63) >> 6;
  const int i = lane * step;
  uint64_t le = __ballot(i < B && starts[i < B ? i : 0] <= r);
  int b = le ? (63 - __builtin_clzll(le)) * step : 0;
  if (step > 1) {
    const int j = b + lane;
    le = __ballot(lane < step && j < B && starts[j < B ? j : 0] <= r);
    b += le ? 63 - __builtin_clzll(le) : 0;
  }
  return __builtin_amdgcn_readfirstlane(b);
}

template <int D, bool kFp8>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
  constexpr int HALF = D / 2, E = D / 16;
  __shared__ float2 turn[HALF];  // (cos, sin) of the row's angles
  const int r = blockIdx.x;
  int b, t;
  if (a.starts) {
    b = sequence_of(a.starts, a.B, r);
    const int s0 = ld_uniform(a.starts, b), s1 = ld_uniform(a.starts, b + 1);
    if (r < s0 || r >= s1) return;  // a row behind the last sequence (uniform over the workgroup)
    t = r - s0;
  } else {
    b = r / a.T;
    t = r - b * a.T;
  }
  const int64_t pos = (int64_t)ld_uniform(a.off, b) + t;
  const bool rope = !(a.flags & EMA_PRE_NO_ROPE);
  if (rope && (int)threadIdx.x < HALF) {
    const int64_t at = pos + (a.prefix ? ld_uniform(a.prefix, 0) : 0);
    const double f = (double)at * exp2(-((double)threadIdx.x / HALF) * a.log2_theta) * 0.15915494309189533577;
    float sn, cs;
    sincospif(2.0f * (float)(f - rint(f)), &sn, &cs);
    turn[threadIdx.x] = make_float2(cs, sn);
  }
  int page = -1;
  if (pos >= 0 && (pos >> a.shift) < a.cols) page = ld_uniform(a.table, (int64_t)b * a.cols + (pos >> a.shift));
  const bool held = (uint32_t)page < (uint32_t)a.n_pages;
  const int slot = (int)(pos & ((1 << a.shift) - 1));
  const int64_t dst0 = (int64_t)page * a.sb + (int64_t)slot * a.sp;
  __syncthreads();

  const int j = threadIdx.x & 7;
  const int H = a.Hq + 2 * a.Hkv;
  for (int h = threadIdx.x >> 3; h < H; h += 32) {
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
    if (!is_q && !held) continue;
    const uint16_t* const src = a.qkv + ((int64_t)r * H + h) * D + j * E;
    float x[E], y[E];
    load_row<E>(src, x);
    load_row<E>(src + HALF, y);
    if (!is_v) {
      if (!(a.flags & (EMA_PRE_NO_NORM | (is_q ? EMA_PRE_NO_Q_NORM : EMA_PRE_NO_K_NORM)))) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss += x[e] * x[e] + y[e] * y[e];
        ss += __shfl_xor(ss, 4, 8);
        ss += __shfl_xor(ss, 2, 8);
        ss += __shfl_xor(ss, 1, 8);
        const float inv = 1.0f / sqrtf(ss / (float)D + a.eps);
        const uint16_t* const w = (is_q ? a.qw : a.kw) + j * E;
        float wx[E], wy[E];
        load_row<E>(w, wx);
        load_row<E>(w + HALF, wy);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] *= inv * wx[e], y[e] *= inv * wy[e];
      }
      if (rope) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float2 cs = turn[j * E + e];
          const float u = x[e] * cs.x - y[e] * cs.y;
          y[e] = x[e] * cs.y + y[e] * cs.x;
          x[e] = u;
        }
      }
    }
    if (is_q) {
      uint16_t* const dst = a.q_out + ((int64_t)r * a.Hq + h) * D + j * E;
      store_row<E>(dst, x);
      store_row<E>(dst + HALF, y);
      continue;
    }
    const int kh = h - a.Hq - (is_v ? a.Hkv : 0);
    const int64_t dst = dst0 + (int64_t)kh * a.sh;
    if constexpr (kFp8) {
      // the row as bf16, then quantised per 64-value block, as the static FP8 cache's rows are:
      // the 8 lanes' halves are the two blocks
      uint16_t lo[8], hi[8];
      float m0 = 0.f, m1 = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo[e] = (uint16_t)f32_to_bf16_bits(x[e]);
        hi[e] = (uint16_t)f32_to_bf16_bits(y[e]);
        m0 = fmaxf(m0, fabsf(bf16_to_f32(lo[e])));
        m1 = fmaxf(m1, fabsf(bf16_to_f32(hi[e])));
      }
      const int e0 = fp8_block_exp(m0), e1 = fp8_block_exp(m1);
      uint8_t* const row = (uint8_t*)(is_v ? a.v : a.k) + dst + j * 8;
      *(u32x2*)row = fp8_encode8(lo, e0);
      *(u32x2*)(row + HALF) = fp8_encode8(hi, e1);
      if (j == 0) {
        const int64_t er = (((int64_t)page * a.Hkv + kh) << a.shift) + slot;
        *(uint16_t*)((is_v ? a.vexp : a.kexp) + 2 * er) = (uint16_t)((uint8_t)e0 | ((uint32_t)(uint8_t)e1 << 8));
      }
    } else {
      uint16_t* const p = (uint16_t*)(is_v ? a.v : a.k) + dst + j * E;
      store_row<E>(p, x);
      store_row<E>(p + HALF, y);
    }
  }
}

// ------------------------------------------------------------------ attention, rows in blocks of 32
// A segment is 32 query rows of one (sequence, kv head): row i is token i / G, head i % G of
// the kv head's group, so a decode step's G heads and a few drafted tokens' share one pass over
// K and V. The keys of a segment are tiles of 32, four tiles a round, one or four rounds a unit;
// the units of all segments, laid end to end, are cut into equal slices, one per workgroup,
// whatever the lengths.
// The four waves of a workgroup take a round's tiles, each with its own softmax state and its own
// LDS slot for the tile, and no barrier until their states meet at the piece's end. A segment cut over
// several workgroups leaves partial states in the workspace; the last of them to arrive joins
// them.
//
//   S^T[key, row] = K . Q^T     MFMA 32x32x16, A = K rows from LDS, B = Q^T in registers
//   O^T[d, row] += V^T P^T      A = V^T by the transposing LDS read, B = P^T (the S^T
//                               accumulators after exp, unmoved)
// A lane owns one query row: its scores, its share of the row sum, 64 output accumulators.
// Softmax state in 32 bits; P is rounded to bf16 for the product with V, and the row sum is
// taken over the rounded P, so that the weights sum to one.
//
// Bound by HBM with few rows: at G = 4 a 16 KB tile costs a wave about 500 cycles of MFMA
// and as many of vector work, an eighth of the time in which HBM delivers a CU's eight tiles,
// so the 32-row product is used down to one row. 32 heads on 8: 8 sequences of about 32k keys
// (1031 MB) 160 us, 6.4 TB/s; 32 of up to 8k (541 MB) 90 us, FP8 (275 MB) 54; 16 heads on 8, one
// sequence of 1k keys 7.4 us, a chain of dependent reads. K and V that are read once pass the
// caches: 183 and 104 us without that.
//
// Made for few rows: a segment takes the tiles of all its sequence's keys, also those that only
// later rows see (masked), so a causal prompt without history costs twice the tiles that it needs,
// and each segment reads (and, FP8, decodes) K and V again: 4 prompts of 2048 tokens over FP8 pages
// 574 us against 167 for the blocks over bf16 ones.
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;
constexpr int kD = 128;
constexpr int kSlot = kPagedTile * kD * 2;     // one K or V tile as bf16: 8 KB

struct PagedArgs {
  const uint16_t* q;
  const uint8_t* k;
  const uint8_t* v;
  const uint16_t* kexp;  // fp8: exponent pairs [n_pages, Hkv, P]
  const uint16_t* vexp;
  const int32_t* table;
  const int32_t* starts;  // null: T rows per sequence
  const int32_t* rows_end;  // starts null, B 1: the rows end there, or null
  const int32_t* len;
  uint16_t* out;
  int32_t* cnt;     // arrival counters, one per worker
  float* part;      // partial states, slots of [32][kPagedState]
  const float* carry_in;  // states of the rows over a shared prefix [chunk][n_rows, Hq][kPagedState], or null
  float* carry_out;       // leave the rows' states there instead of their output, or null
  const int32_t* prefix_len;      // null: no shared prefix
  const int32_t* prefix_table;    // its pages, where the segments take them themselves (else null)
  int prefix_cols;
  int carry_blocks;       // 64-key blocks of a chunk of the prefix (0: one state, always there)
  int prefix_cap;         // most positions of the prefix (the call's bound)
  int64_t sh;       // bytes
  uint32_t page_bytes, row_bytes;
  uint32_t magic;   // paged_magic(G)
  float qk_scale;   // scale * log2(e): scores live in the log2 domain
  int B, T, n_rows, Hq, Hkv, G, cols, shift, n_pages, W, causal;
  int cap;          // most positions of a sequence: what its table row holds
  int few, max_q;   // sequences of few < n <= max_q rows are prefill_kernel's
};

__device__ __forceinline__ u32x4 rsrc_words(const void* base, uint32_t bytes) {
  const uint64_t addr = (uint64_t)base;
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)addr),
               (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(addr >> 32) & 0xffffu),
               (uint32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}
// 16 bytes per lane from buffer offset voff straight into LDS at lds + 16 lane (zeros past the
// resource's range). Asm, so that the compiler does not track it; the s_nop gives the wait
// states that the DMA needs after the write of M0 (one) and, in the first load over a resource,
// after a vector instruction (a spill's reload) wrote the resource's scalar registers (five).
// kOnce: the bytes are read once in the call (non-temporal).
template <bool kFirst, bool kOnce>
__device__ __forceinline__ void dma16(u32x4 rs, uint32_t voff, uint32_t lds) {
  if constexpr (kOnce)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop %3\n\tbuffer_load_dwordx4 %0, %1, 0 offen nt lds"
                 :
                 : "v"(voff), "s"(rs), "s"(__builtin_amdgcn_readfirstlane(lds)), "i"(kFirst ? 4 : 0)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %2\n\ts_nop %3\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                 :
                 : "v"(voff), "s"(rs), "s"(__builtin_amdgcn_readfirstlane(lds)), "i"(kFirst ? 4 : 0)
                 : "memory", "m0");
}

// Partial states cross XCDs as device-coherent stores and loads (past the XCDs' own L2s).
__device__ __forceinline__ void put2(float* p, float x, float y) {
  const uint64_t w = (uint64_t)__float_as_uint(x) | ((uint64_t)__float_as_uint(y) << 32);
  __hip_atomic_store((uint64_t*)p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float* p) {
  const uint64_t w = __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((uint32_t)w), __uint_as_float((uint32_t)(w >> 32)));
}

// The kernel's arguments, read again from where they came: through a pointer that the compiler
// cannot see into, so that what a piece needs before or after its tiles is not held in scalar
// registers over them (with every argument live the kernels spilled 55 to 79 of them to vector
// lanes and reloaded some in each tile).
__device__ __forceinline__ PagedArgs args_again() {
#if defined(__HIP_DEVICE_COMPILE__)
  auto p = (const __attribute__((address_space(4))) PagedArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
#else
  return {};
#endif
}

struct State4 {  // four dims of a row: running max, row sum, unnormalised output
  float m, l;
  f32x4 o;
};
__device__ __forceinline__ float weight(float m, float M) { return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M); }

// A row's final state: joined with those over the prefix's chunks, then stored as output or
// carried on.
template <bool kFp8>
__device__ __forceinline__ void finish4(const PagedArgs& a, int n_carry, bool keys, int64_t row, int h, int d, State4 s) {
  const int64_t rh = row * a.Hq + h;
  if (a.carry_in) {
    constexpr int kChunk = 16;  // states whose loads are in flight together
    for (int c0 = 0; c0 < n_carry; c0 += kChunk) {
      float2 cm[kChunk];
      f32x4 co[kChunk];
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        const int c = c0 + i < n_carry ? c0 + i : n_carry - 1;
        const float* const p = a.carry_in + ((int64_t)c * a.n_rows * a.Hq + rh) * kPagedState;
        cm[i] = *(const float2*)p;
        co[i] = *(const f32x4*)(p + 4 + d);
      }
      float M = s.m;
#pragma unroll
      for (int i = 0; i < kChunk; ++i) M = fmaxf(M, cm[i].x);
      const float f = weight(s.m, M);
      s.l *= f;
      s.o *= f;
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        const float g = weight(cm[i].x, M);
        if (c0 + i < n_carry && (g > 0.f || cm[i].y != cm[i].y)) {  // (a row that is not finite stays so)
          s.l += cm[i].y * g;
          s.o += co[i] * g;
        }
      }
      s.m = M;
    }
  }
  if (kFp8 && a.carry_out) {  // (bf16: prefill_kernel leaves the states)
    float* const c = a.carry_out + rh * kPagedState;
    if (d == 0) *(float2*)c = make_float2(s.m, s.l);
    *(f32x4*)(c + 4 + d) = s.o;
    return;
  }
  const float inv = keys ? 1.0f / s.l : 0.f;  // no key: zeros; keys and no finite score: NaN, as the softmax is
  *(u32x2*)(a.out + rh * kD + d) = u32x2{pack_bf16x2(s.o[0] * inv, s.o[1] * inv), pack_bf16x2(s.o[2] * inv, s.o[3] * inv)};
}

__device__ __forceinline__ PagedRows own_rows(const PagedArgs& a, PagedRows r) {
  if (r.n > a.few && r.n <= a.max_q) r.n = 0;
  return r;
}
__device__ __forceinline__ PagedRows rows_of(const PagedArgs& a, int b) {
  if (!a.starts) return a.rows_end ? paged_rows(0, ld_uniform(a.rows_end, 0), a.T) : PagedRows{b * a.T, a.T};
  return own_rows(a, paged_rows(ld_uniform(a.starts, b), ld_uniform(a.starts, b + 1), a.n_rows));
}
__device__ __forceinline__ int clamp_len(const PagedArgs& a, int L) {
  return L < 0 ? 0 : (L > a.cap ? a.cap : L);
}
__device__ __forceinline__ int blocks_of(const PagedArgs& a, int T) {
  return (int)(((uint32_t)T * (uint32_t)a.G + kPagedRows - 1) / kPagedRows);
}

// kDirect: the segments take a shared prefix's tiles before their own.
template <bool kFp8, bool kOnce, bool kDirect>
__global__ __launch_bounds__(64 * kPagedWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_kernel(PagedArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t slots[kPagedWaves][2 * kSlot];
  __shared__ float2 ml[kPagedWaves][kPagedRows];
  __shared__ int32_t pre[kPagedMaxB + 64];
  __shared__ int arrived;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // a shared prefix: its keys, the states of the rows over it (one per chunk that holds keys), or
  // its tiles, which then come before each segment's own
  int n_carry = 1, prefix = 0, prefix_tiles = 0;
  if (a.prefix_len) {
    prefix = ld_uniform(a.prefix_len, 0);
    prefix = prefix < 0 ? 0 : (prefix > a.prefix_cap ? a.prefix_cap : prefix);
    if (a.carry_blocks) n_carry = ((prefix + 63) / 64 + a.carry_blocks - 1) / a.carry_blocks;
    if (kDirect) prefix_tiles = paged_tiles(prefix);
  }
  const bool shared_keys = prefix > 0;

  // Units of work before each sequence, by every wave for itself: lane l takes sequences
  // l step .. +step-1 (up to 64 sequences: one each, kept in the lane's registers; more: their
  // starts go to LDS, where all waves write the same values), and the lanes' sums are scanned.
  const int step = (a.B + 63) >> 6;
  const PagedRows all_rows = a.starts ? PagedRows{0, 0} : rows_of(a, 0);
  auto rows_at = [&](int b) __attribute__((always_inline)) {
    if (a.starts) return own_rows(a, paged_rows(a.starts[b], a.starts[b + 1], a.n_rows));
    return PagedRows{b * all_rows.n, all_rows.n};
  };
  PagedRows lane_rows = {0, 0};
  int lane_len = 0, sum1 = 0, sum_long = 0, sum_segs = 0;
  for (int i = 0; i < step; ++i) {
    const int b = lane * step + i;
    if (b < a.B) {
      lane_rows = rows_at(b);
      lane_len = clamp_len(a, a.len[b]);
      const int nr = paged_rounds(prefix_tiles + paged_tiles(lane_len)), segs = blocks_of(a, lane_rows.n) * a.Hkv;
      sum1 += segs * paged_units(nr, 1);
      sum_long += segs * paged_units(nr, kPagedLongUnit);
      sum_segs += nr ? segs : 0;
    }
  }
  const int pre1 = sum_up_to_lane(sum1), pre_long = sum_up_to_lane(sum_long);
  const int unit = paged_unit(__builtin_amdgcn_readlane(pre1, 63), __builtin_amdgcn_readlane(sum_up_to_lane(sum_segs), 63), a.W);
  const int total = __builtin_amdgcn_readlane(unit == 1 ? pre1 : pre_long, 63);
  const int lane_pre = unit == 1 ? pre1 - sum1 : pre_long - sum_long;
  if (step > 1) {
    int run = lane_pre;
    for (int i = 0; i < step; ++i) {
      const int b = lane * step + i;
      if (b < a.B) {
        pre[b] = run;
        const int nr = paged_rounds(prefix_tiles + paged_tiles(clamp_len(a, a.len[b])));
        run += blocks_of(a, rows_at(b).n) * a.Hkv * paged_units(nr, unit);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }

  // rows of sequences that see nothing: no unit visits them
  for (int i = 0; i < step && prefix_tiles == 0; ++i) {
    const int bl = lane * step + i;
    uint64_t none = __ballot(bl < a.B && (step == 1 ? lane_len : a.len[bl < a.B ? bl : 0]) <= 0);
    for (; none; none &= none - 1) {
      const int b = __builtin_ctzll(none) * step + i;
      if (b % (int)gridDim.x != (int)blockIdx.x) continue;
      const PagedRows rw = rows_of(a, b);
      const State4 empty = {-INFINITY, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}};
      for (int64_t e = tid; e < (int64_t)rw.n * a.Hq * 32; e += 64 * kPagedWaves)
        finish4<kFp8>(a, n_carry, shared_keys, rw.begin + e / (a.Hq * 32), (int)(e / 32 % a.Hq), (int)(e % 32) * 4, empty);
    }
  }

  const int W = paged_active_workers(total, a.W);
  if (total == 0 || (int)blockIdx.x >= W) return;
  const int w = xcd_rank(blockIdx.x, W);
  const PagedSplit split = paged_split(total, W);
  int t = paged_begin(split, w);
  const int t_end = paged_begin(split, w + 1);

  const int hh = lane >> 5, r4 = lane >> 4, p16 = lane & 15;
  uint8_t* const Kt = slots[wave];
  uint8_t* const Vt = Kt + kSlot;
  const uint32_t kdst = (uint32_t)(uintptr_t)(lds_void*)Kt, vdst = (uint32_t)(uintptr_t)(lds_void*)Vt;
  // LDS tiles are 32 unpadded 256-byte rows, 16-byte chunks swizzled against bank conflicts:
  // chunk p of K row r holds chunk p ^ (r & 15), of V row r chunk p ^ 4 (r & 3). bf16: loads of
  // 4 whole rows; source offset of position p16 in row 4 i + r4 of a 16-row half
  uint32_t koff[4], voff[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    koff[i] = (uint32_t)(4 * i + r4) * a.row_bytes + (uint32_t)(p16 ^ (4 * i + r4)) * 16;
    voff[i] = (uint32_t)(4 * i + r4) * a.row_bytes + (uint32_t)(p16 ^ (4 * r4)) * 16;
  }
  // operand reads: K row lane & 31, column chunk 2 s + hh; V^T by the transposing read
  const uint16_t* const kp = (const uint16_t*)Kt + (lane & 31) * kD + 8 * (hh ^ (lane & 1));
  const int k_x = 16 * ((lane & 15) >> 1);
  const int grp = lane >> 4, s16 = lane & 15;
  const int tr_row = 4 * (grp >> 1) + (s16 >> 2);
  int v_col[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) v_col[dt] = tr_row * kD + 16 * (grp & 1) + 4 * (s16 & 3) + 32 * (dt ^ (s16 >> 2));

  while (t < t_end) {
    const PagedArgs a = args_again();
    // the segment of unit t: the last b whose units begin at or before it
    const uint64_t le = __ballot(lane * step < a.B && lane_pre <= t);
    const int at = 63 - __builtin_clzll(le);
    int b = at, L, pre_b;
    PagedRows rw;
    if (step == 1) {
      rw = PagedRows{__builtin_amdgcn_readlane(lane_rows.begin, at), __builtin_amdgcn_readlane(lane_rows.n, at)};
      L = __builtin_amdgcn_readlane(lane_len, at);
      pre_b = __builtin_amdgcn_readlane(lane_pre, at);
    } else {
      const int bi = at * step + lane;
      b = at * step + 63 - __builtin_clzll(__ballot(lane < step && bi < a.B && pre[bi < a.B ? bi : 0] <= t));
      rw = rows_of(a, b);
      L = clamp_len(a, ld_uniform(a.len, b));
      pre_b = __builtin_amdgcn_readfirstlane(pre[b]);
    }
    const int tile_end = prefix_tiles + paged_tiles(L);
    const int nu = paged_units(paged_rounds(tile_end), unit), nrb = blocks_of(a, rw.n);
    const uint32_t seg = (uint32_t)(t - pre_b) / (uint32_t)nu;
    const int unit0 = (int)((uint32_t)(t - pre_b) - seg * (uint32_t)nu);
    const int kh = nrb == 1 ? (int)seg : (int)(seg / (uint32_t)nrb), rb = (int)(seg - (uint32_t)kh * (uint32_t)nrb);
    if (kh >= a.Hkv) break;  // (row starts that do not ascend can overflow the count of units)
    const int seg_begin = t - unit0, seg_end = seg_begin + nu;
    const int piece_end = t_end < seg_end ? t_end : seg_end;
    const int tile0 = unit0 * unit * kPagedWaves;
    const int tile1 = min(tile0 + (piece_end - t) * unit * kPagedWaves, tile_end);
    const int row0 = rb * kPagedRows;                     // the segment's first row (token * G + head)
    const int n_seg = rw.n * a.G - row0 < kPagedRows ? rw.n * a.G - row0 : kPagedRows;

    // this lane's query row, and the last key it sees
    const int i_row = row0 + ((lane & 31) < n_seg ? (lane & 31) : n_seg - 1);
    const int tok = paged_div(i_row, a.magic), head = i_row - tok * a.G;
    const int last_key = a.causal ? L - rw.n + tok : L - 1;
    const int first_limit = a.causal ? L - rw.n + paged_div(row0, a.magic) : L - 1;

    // tile of the segment's list: the prefix's first, then its own
    const int32_t* const own_table = a.table + (int64_t)b * a.cols;
    auto is_own = [&](int tile) __attribute__((always_inline)) { return !kDirect || tile >= prefix_tiles; };
    auto place = [&](int tile) __attribute__((always_inline)) { return kDirect && is_own(tile) ? tile - prefix_tiles : tile; };
    // table entry of the page that holds position 16 half of the tile (any entry past the tiles)
    auto entry = [&](int tile, int half) __attribute__((always_inline)) {
      const int c = (int)(((uint32_t)place(tile) * kPagedTile + 16u * half) >> a.shift);
      const int cols = is_own(tile) ? a.cols : a.prefix_cols;
      return ld_uniform(is_own(tile) ? own_table : a.prefix_table, c < cols ? c : cols - 1);
    };
    // The two 16-row halves of a tile: where their rows begin, in bytes from the kv head's first
    // row in either pool, and how many are held (none past the piece, past the keys or on an entry
    // outside the pool)
    struct Halves {
      int64_t at[2];
      uint32_t n[2];
    };
    const uint8_t* const kb = a.k + (int64_t)kh * a.sh;
    const uint8_t* const vb = a.v + (int64_t)kh * a.sh;
    auto halves = [&](int tile, int e0, int e1) __attribute__((always_inline)) {
      Halves r;
      const int left = (is_own(tile) ? L : prefix) - place(tile) * kPagedTile;
      const uint32_t slot = ((uint32_t)place(tile) * kPagedTile) & ((1u << a.shift) - 1u);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t page = (uint32_t)(half ? e1 : e0);
        const bool in = tile < tile1 && page < (uint32_t)a.n_pages;
        const int n = left - 16 * half;
        r.n[half] = in && n > 0 ? (uint32_t)(n < 16 ? n : 16) : 0u;
        // (a 16-position page begins anew with the second half)
        const uint32_t row = half ? (slot + 16u) & ((1u << a.shift) - 1u) : slot;
        r.at[half] = (int64_t)((uint64_t)(in ? page : 0u) * a.page_bytes + (uint64_t)row * a.row_bytes);
      }
      return r;
    };
    // bf16: a tile by eight loads of four whole rows each, straight into the slot
    auto dma_tile = [&](bool k, const Halves& hv) __attribute__((always_inline)) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const u32x4 r = rsrc_words((k ? kb : vb) + hv.at[half], hv.n[half] * a.row_bytes);
        const uint32_t dst = (k ? kdst : vdst) + 4096 * half;
        dma16<true, kOnce>(r, k ? koff[0] : voff[0], dst);
#pragma unroll
        for (int i = 1; i < 4; ++i) dma16<false, kOnce>(r, k ? koff[i] : voff[i], dst + 1024 * i);
      }
    };
    // fp8: a tile's codes into registers (row 8 i + lane / 8, codes 16 (lane % 8) .. +15), with
    // the exponent of the row's 64-code block; decoded into the slot as bf16 before use
    struct Codes {
      u32x4 w[4];
      int e[4];
    };
    auto load_codes = [&](bool k, int tile, const Halves& hv, int e0, int e1) __attribute__((always_inline)) {
      Codes c;
      const uint32_t slot = ((uint32_t)place(tile) * kPagedTile) & ((1u << a.shift) - 1u);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t n = hv.n[half], at = half ? (slot + 16u) & ((1u << a.shift) - 1u) : slot;
        const uint16_t* const eb = (k ? a.kexp : a.vexp) +
            (n ? (((int64_t)(half ? e1 : e0) * a.Hkv + kh) << a.shift) + at : 0);
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>((k ? kb : vb) + hv.at[half]), (short)0, (int)(n * a.row_bytes), 0x00020000);
        const __amdgpu_buffer_rsrc_t re =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(eb), (short)0, (int)(2 * n), 0x00020000);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t row = 8 * i + (lane >> 3);
          c.w[2 * half + i] = __builtin_amdgcn_raw_buffer_load_b128(r, row * a.row_bytes + 16 * (lane & 7), 0, kOnce ? 2 : 0);
          c.e[2 * half + i] = (int8_t)__builtin_amdgcn_raw_buffer_load_b8(re, 2 * row + ((lane >> 2) & 1), 0, 0);
        }
      }
      return c;
    };
    auto decode_codes = [&](bool k, const Codes& c) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 8 * i + (lane >> 3), p = 2 * (lane & 7);
        const int sw = k ? row & 15 : 4 * (row & 3);
        u32x4* const dst = (u32x4*)((k ? Kt : Vt) + 256 * row);
        dst[p ^ sw] = fp8_decode8(u32x2{c.w[i][0], c.w[i][1]}, c.e[i]);
        dst[(p + 1) ^ sw] = fp8_decode8(u32x2{c.w[i][2], c.w[i][3]}, c.e[i]);
      }
    };

    const int first = tile0 + wave;
    int e0 = entry(first, 0), e1 = entry(first, 1);
    // Q^T as B operand: step s covers dims 16 s + 8 hh .. +7 of the lane's row
    bf16x8 qop[8];
    {
      const u32x4* const qp = (const u32x4*)(a.q + (((int64_t)rw.begin + tok) * a.Hq + kh * a.G + head) * kD) + hh;
#pragma unroll
      for (int s = 0; s < 8; ++s) qop[s] = as_bf16x8(qp[2 * s]);
    }
    Halves hv = halves(first, e0, e1);
    Codes kc, vc;
    if constexpr (kFp8) {
      kc = load_codes(true, first, hv, e0, e1);
      vc = load_codes(false, first, hv, e0, e1);
    } else if (first < tile1) {
      dma_tile(true, hv);
      dma_tile(false, hv);
    }

    float m = -INFINITY, l = 0.f;  // of the lane's row; l over this lane's half of the keys
    f32x16 o[4];
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;

    for (int tile = first; tile < tile1; tile += kPagedWaves) {
      e0 = entry(tile + kPagedWaves, 0);
      e1 = entry(tile + kPagedWaves, 1);
      if constexpr (kFp8) {
        decode_codes(true, kc);
        hv = halves(tile + kPagedWaves, e0, e1);
        kc = load_codes(true, tile + kPagedWaves, hv, e0, e1);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      } else {
        asm volatile("s_waitcnt vmcnt(8)" ::: "memory");  // K of this tile
      }
      f32x16 sc, sc2;  // two chains of products
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i] = sc2[i] = 0.f;
#pragma unroll
      for (int s = 0; s < 8; s += 2) {
        sc = mfma32(as_bf16x8(*(const u32x4*)(kp + (k_x ^ (16 * s)))), qop[s], sc);
        sc2 = mfma32(as_bf16x8(*(const u32x4*)(kp + (k_x ^ (16 * s + 16)))), qop[s + 1], sc2);
      }
      sc += sc2;
      const bool more = tile + kPagedWaves < tile1;
      if (!kFp8 && more) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot has been read
        hv = halves(tile + kPagedWaves, e0, e1);
        dma_tile(true, hv);
      }
      // key of score i: 32 place + (i % 4) + 8 (i / 4) + 4 hh
      const int key0 = place(tile) * kPagedTile;
      if (key0 + kPagedTile - 1 > (is_own(tile) ? first_limit : prefix - 1)) {
        const int room = (is_own(tile) ? last_key : prefix - 1) - key0 - 4 * hh;
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = (i & 3) + 8 * (i >> 2) <= room ? sc[i] : -INFINITY;
      }
      float mx = sc[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sc[i]);
      mx = fmaxf(wave_max_xor(mx, 32) * a.qk_scale, m);
      if (__any(mx > m)) {  // some row's max grew: rescale what was accumulated
        const float alpha = weight(m, mx);
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) o[dt] *= alpha;
        m = mx;
      }
      const float base = m == -INFINITY ? 0.f : m;
      u32x4 pw[2];
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 8 * st + 2 * e;
          pw[st][e] = pack_bf16x2(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], a.qk_scale, -base)),
                                  __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i + 1], a.qk_scale, -base)));
          l = dot2_bf16(pw[st][e], 0x3F803F80u, l);
        }
      if constexpr (kFp8) {
        decode_codes(false, vc);
        vc = load_codes(false, tile + kPagedWaves, hv, e0, e1);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      } else {
        if (more) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");  // V of this tile, and not K of the next
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) {
          const uint16_t* const p0 = (const uint16_t*)Vt + 16 * st * kD + v_col[dt];
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p0);
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p0 + 8 * kD));
          typedef short s16x8 __attribute__((ext_vector_type(8)));
          const s16x8 av = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          o[dt] = mfma32(__builtin_bit_cast(bf16x8, av), as_bf16x8(pw[st]), o[dt]);
        }
      if constexpr (!kFp8) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (more) dma_tile(false, hv);
      } else {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      }
    }
    // (from here on, arguments read again)
    const PagedArgs z = args_again();
    // the waves' states meet: o of wave w in its own slots, [row][d / 4] with unit d4 of row r
    // at d4 ^ r
    f32x4* const os = (f32x4*)Kt;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const int d4 = 8 * dt + 2 * i4 + hh, r = lane & 31;
        os[r * 32 + (d4 ^ r)] = f32x4{o[dt][4 * i4], o[dt][4 * i4 + 1], o[dt][4 * i4 + 2], o[dt][4 * i4 + 3]};
      }
    l += __shfl_xor(l, 32, 64);
    if (lane < 32) ml[wave][lane] = make_float2(m, l);
    __syncthreads();
    const int w0 = paged_worker_of(split, seg_begin), w1 = paged_worker_of(split, seg_end - 1);
    const int units = n_seg * 32;
    for (int u = tid; u < units; u += 64 * kPagedWaves) {
      const int r = u >> 5, d4 = u & 31;
      State4 s = {-INFINITY, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int v = 0; v < kPagedWaves; ++v) s.m = fmaxf(s.m, ml[v][r].x);
#pragma unroll
      for (int v = 0; v < kPagedWaves; ++v) {
        const float f = weight(ml[v][r].x, s.m);
        s.l += ml[v][r].y * f;
        s.o += ((const f32x4*)slots[v])[r * 32 + (d4 ^ r)] * f;
      }
      if (w0 == w1) {
        const int ir = row0 + r, tk = paged_div(ir, z.magic);
        finish4<kFp8>(z, n_carry, shared_keys || !z.causal || L - rw.n + tk >= 0, (int64_t)rw.begin + tk, kh * z.G + ir - tk * z.G, 4 * d4, s);
      } else {
        float* const p = z.part + ((int64_t)paged_slot(w, w0) * kPagedRows + r) * kPagedState;
        if (d4 == 0) put2(p, s.m, s.l);
        put2(p + 4 + 4 * d4, s.o[0], s.o[1]);
        put2(p + 6 + 4 * d4, s.o[2], s.o[3]);
      }
    }
    if (w0 != w1) {
      // arrival: every wave's stores have reached the device-coherent level before its
      // workgroup is counted in; the last of the segment's workgroups returns the counter to
      // zero and joins the pieces
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (tid == 0) {
        int i = w0;
        asm volatile("" : "+v"(i));
        const int old = __hip_atomic_fetch_add(z.cnt + i, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const int last = old == w1 - w0;
        if (last) __hip_atomic_store(z.cnt + i, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        arrived = last;
      }
      __syncthreads();
      if (arrived) {
        auto join = [&](auto chunk_tag) __attribute__((always_inline)) {
          constexpr int kChunk = decltype(chunk_tag)::value;  // pieces whose loads are in flight together
          for (int u = tid; u < units; u += 64 * kPagedWaves) {
            const int r = u >> 5, d4 = u & 31;
            State4 s = {-INFINITY, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}};
            for (int c0 = w0; c0 <= w1; c0 += kChunk) {
              float2 pm[kChunk], pa[kChunk], pb[kChunk];
#pragma unroll
              for (int i = 0; i < kChunk; ++i) {
                const int ww = c0 + i <= w1 ? c0 + i : w1;
                const float* const p = z.part + ((int64_t)paged_slot(ww, w0) * kPagedRows + r) * kPagedState;
                pm[i] = get2(p);
                pa[i] = get2(p + 4 + 4 * d4);
                pb[i] = get2(p + 6 + 4 * d4);
              }
              float M = s.m;
#pragma unroll
              for (int i = 0; i < kChunk; ++i) M = fmaxf(M, pm[i].x);
              const float f = weight(s.m, M);
              s.l *= f;
              s.o *= f;
#pragma unroll
              for (int i = 0; i < kChunk; ++i)
                if (c0 + i <= w1) {
                  const float g = weight(pm[i].x, M);
                  s.l += pm[i].y * g;
                  s.o += f32x4{pa[i].x, pa[i].y, pb[i].x, pb[i].y} * g;
                }
              s.m = M;
            }
            const int ir = row0 + r, tk = paged_div(ir, z.magic);
            finish4<kFp8>(z, n_carry, shared_keys || !z.causal || L - rw.n + tk >= 0, (int64_t)rw.begin + tk,
                    kh * z.G + ir - tk * z.G, 4 * d4, s);
          }
        };
        if (w1 - w0 < 3) join(std::integral_constant<int, 3>{});
        else if (w1 - w0 < 8) join(std::integral_constant<int, 8>{});
        else join(std::integral_constant<int, 16>{});
      }
    }
    __syncthreads();  // the slots and ml are reused by the next piece
    t = piece_end;
  }
}

// max_q: most rows of a sequence. Where all are one segment, K and V are read once.
int32_t launch_rows(hipStream_t s, const PagedArgs& a, bool fp8, int max_q, const char* what) {
  const bool once = (int64_t)max_q * a.G <= kPagedRows;
  const dim3 grid(a.W), block(64 * kPagedWaves);
  if (a.prefix_table) {  // (several sequences' segments read the prefix)
    if (fp8) hipLaunchKernelGGL((paged_kernel<true, false, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((paged_kernel<false, false, true>), grid, block, 0, s, a);
  } else if (fp8 && once) {
    hipLaunchKernelGGL((paged_kernel<true, true, false>), grid, block, 0, s, a);
  } else if (fp8) {
    hipLaunchKernelGGL((paged_kernel<true, false, false>), grid, block, 0, s, a);
  } else if (once) {
    hipLaunchKernelGGL((paged_kernel<false, true, false>), grid, block, 0, s, a);
  } else {
    hipLaunchKernelGGL((paged_kernel<false, false, false>), grid, block, 0, s, a);
  }
  return check_hip(hipGetLastError(), what);
}

}  // namespace

int32_t launch_paged_append(hipStream_t s, const PagedAppend& p, const ema_kvcache_desc& c) {
  AppendArgs a;
  a.qkv = (const uint16_t*)p.qkv;
  a.qw = (const uint16_t*)p.q_norm_w;
  a.kw = (const uint16_t*)p.k_norm_w;
  a.off = p.offsets;
  a.starts = p.q_starts;
  a.prefix = p.prefix_len;
  a.table = p.table;
  a.q_out = (uint16_t*)p.q_out;
  a.k = c.k;
  a.v = c.v;
  a.kexp = (int8_t*)c.k_exp;
  a.vexp = (int8_t*)c.v_exp;
  a.sb = c.stride_batch;
  a.sh = c.stride_head;
  a.sp = c.stride_pos;
  a.log2_theta = log2((double)p.theta);
  a.eps = p.eps;
  a.B = p.batch;
  a.T = p.q_starts ? 1 : p.n_rows / p.batch;
  a.n_rows = p.n_rows;
  a.Hq = p.n_heads;
  a.Hkv = c.n_kv_heads;
  a.cols = p.table_cols;
  a.shift = paged_shift(c.capacity);
  a.n_pages = c.batch;
  a.flags = p.flags;
  const dim3 grid((unsigned)p.n_rows), block(256);
  if (c.dtype == EMA_DTYPE_FP8_E4M3) hipLaunchKernelGGL((paged_append_kernel<128, true>), grid, block, 0, s, a);
  else if (c.head_dim == 64) hipLaunchKernelGGL((paged_append_kernel<64, false>), grid, block, 0, s, a);
  else if (c.head_dim == 128) hipLaunchKernelGGL((paged_append_kernel<128, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((paged_append_kernel<256, false>), grid, block, 0, s, a);
  return check_hip(hipGetLastError(), "ema_paged_append launch");
}

// More query rows than kFewRows per (sequence, kv head) run in prefill_kernel's 128-row blocks
// (bf16 pages) where these, were every sequence as long as the longest, are at least 3/8 of the CUs;
// the others in paged_kernel's 32-row segments, whose keys are split. Segments / blocks, us, 32
// heads on 8. Blocks taken: 16 sequences of 192 rows 54.7 / 25.7 after 1000 keys and 12.7 / 10.1
// without history, 4 of 512 rows after 8000 keys 122 / 108, one of 2048 rows 131 / 109. Segments
// taken: after 8000 keys 4 sequences of 256 rows 82 / 104 (64 workgroups of blocks), one 42 / 100.
// The rule knows neither the history nor the rows that the sequences really have, and takes the
// slower way in these: segments, 16 sequences after 8000 keys, 64 rows 121 / 111, 96 rows 293 / 114
// (their segments read K and V out of phase, each from HBM), 128 rows 147 / 116, after 1000 keys
// 96 rows 42.9 / 22.5, and 4 of 192 rows after 8000 keys 129 / 103; blocks, a chunk of 64 tokens
// (256 rows) after 8000 keys beside single tokens after 2000 keys, 7 of them 46.9 / 118, 31
// 77.7 / 146 (a caller's way out is max_q 1: 55 and 85).
constexpr int kFewRows = 128;
bool paged_blocks(int64_t rows, int B, int Hkv, int cus) {
  return rows > kFewRows && (rows + 127) / 128 * B * Hkv * 8 >= (int64_t)cus * 3;
}
// A shared prefix whose tiles are no more rounds than this when every segment takes them itself:
// one launch over the prefix's and the own tiles together, K and V of the prefix from the L2s. Against
// the prefix in a launch of its own, us, 32 heads on 8 / 16 on 2. bf16 (in 128-row blocks): 416 rounds
// 10.1 : 16.2 / 11.6 : 17.5, 832 14.6 : 16.9 / 12.0 : 18.2, 1664 17.0 : 17.7 / -, 2048 25.9 : 20.1 /
// 17.0 : 22.7, 4032 45.8 : 27.3 / 47.1 : 41.6. FP8 (in segments): 1664 16.5 : 26.7, 2048 19.1 : 26.6 /
// 17.9 : 26.8, 4096 26.4 : 26.6. Near the limit the layouts differ (a prefix on 2 kv heads is read by
// fewer segments at a time), and rounds alone do not tell them apart: at 2048 rounds the limit is
// right for 2 kv heads and for FP8 and 6 us too high for bf16 on 8.
constexpr int kDirectRounds = 4 * kPagedMaxWorkers;

// Workspace: the arrival counters, the partial states of the workers' shared segments, then
// the rows' states over a shared prefix.
PagedPlan plan_paged(int B, int n_rows, int Hq, int Hkv, int max_q, int max_len, int max_prefix) {
  PagedPlan p;
  const int G = Hq / Hkv;
  const int64_t nrb = paged_row_blocks(B, n_rows, max_q, G);
  p.workers = paged_plan_workers(nrb, Hkv, paged_tiles(max_len));
  p.prefix_workers = 0;
  p.chunks = p.chunk_blocks = 0;
  p.carry_bytes = 0;
  p.direct = max_prefix > 0 && nrb * Hkv * paged_rounds(paged_tiles(max_prefix) + paged_tiles(max_len)) <= kDirectRounds;
  if (p.direct) {
    p.workers = paged_plan_workers(nrb, Hkv, paged_tiles(max_prefix) + paged_tiles(max_len));
  } else if (max_prefix > 0) {
    p.prefix_workers = paged_plan_workers(paged_row_blocks(1, n_rows, n_rows, G), Hkv, paged_tiles(max_prefix));
    const PagedChunks c = paged_chunks((int64_t)n_rows * G, Hkv, max_prefix, device_cus());
    p.chunks = c.n;
    p.chunk_blocks = c.blocks;
    p.carry_bytes = (uint64_t)c.n * n_rows * Hq * kPagedState * sizeof(float);
  }
  const int w = p.workers > p.prefix_workers ? p.workers : p.prefix_workers;
  p.part_bytes = (uint64_t)2 * w * kPagedRows * kPagedState * sizeof(float);
  p.bytes = kDecodeCounterBytes + p.part_bytes + p.carry_bytes;
  return p;
}

// The plans' bytes are not monotone (fewer rows are more chunks of a prefix, and the ways to take
// it differ), so the size told to a caller is a bound of all of them up to the bounds: workgroups
// over the most tiles of any way, and states of one chunk's rows or of what fills the chip, 128 rows
// on each CU.
uint64_t paged_workspace_bytes(int B, int n_rows, int Hq, int Hkv, int max_q, int max_len, int max_prefix) {
  const int G = Hq / Hkv;
  const int own = paged_plan_workers(paged_row_blocks(B, n_rows, max_q, G), Hkv,
                                     paged_tiles(max_prefix) + paged_tiles(max_len));
  const int all = paged_plan_workers(paged_row_blocks(1, n_rows, n_rows, G), Hkv, paged_tiles(max_prefix));
  const uint64_t rows = (uint64_t)n_rows * Hq, fill = (uint64_t)device_cus() * 128;
  const uint64_t most = rows * (((uint64_t)max_prefix + 127) / 128);  // a chunk holds 128 keys at least
  uint64_t states = most < fill ? most : fill;
  if (states < rows) states = rows;
  return kDecodeCounterBytes + (uint64_t)2 * (own > all ? own : all) * kPagedRows * kPagedState * sizeof(float) +
         (max_prefix > 0 ? states * kPagedState * sizeof(float) : 0);
}

int32_t launch_paged_attention(hipStream_t s, const PagedAttention& p, const ema_kvcache_desc& c, const PagedPlan& plan,
                               void* ws) {
  const bool fp8 = c.dtype == EMA_DTYPE_FP8_E4M3;
  const int es = fp8 ? 1 : 2;  // bytes per element of the strides
  PagedArgs a;
  a.q = (const uint16_t*)p.q;
  a.k = (const uint8_t*)c.k;
  a.v = (const uint8_t*)c.v;
  a.kexp = (const uint16_t*)c.k_exp;
  a.vexp = (const uint16_t*)c.v_exp;
  a.table = p.table;
  a.starts = p.q_starts;
  a.rows_end = nullptr;
  a.len = p.lengths;
  a.out = (uint16_t*)p.out;
  a.cnt = (int32_t*)ws;
  a.part = (float*)((char*)ws + kDecodeCounterBytes);
  a.carry_in = nullptr;
  a.carry_out = nullptr;
  a.prefix_len = p.prefix_len;
  a.prefix_table = nullptr;
  a.prefix_cols = p.prefix_cols;
  a.carry_blocks = 0;
  a.prefix_cap = p.max_prefix;
  a.sh = c.stride_head * es;
  a.page_bytes = (uint32_t)(c.stride_batch * es);
  a.row_bytes = (uint32_t)(c.stride_pos * es);
  a.qk_scale = p.scale * kLog2e;
  a.B = p.batch;
  a.T = p.q_starts ? 1 : p.n_rows / p.batch;
  a.n_rows = p.n_rows;
  a.Hq = p.n_heads;
  a.Hkv = c.n_kv_heads;
  a.G = p.n_heads / c.n_kv_heads;
  a.magic = paged_magic(a.G);
  a.cols = p.table_cols;
  a.shift = paged_shift(c.capacity);
  a.n_pages = c.batch;
  a.causal = p.causal;
  a.cap = p.table_cols << a.shift;  // (at most 2^30: host)
  a.few = INT32_MAX;
  a.max_q = 0;
  if (p.prefix_table && plan.direct) {
    a.prefix_table = p.prefix_table;
  } else if (p.prefix_table) {
    float* const carry = (float*)((char*)ws + kDecodeCounterBytes + plan.part_bytes);
    if (!fp8) {  // in blocks of 128 rows over chunks of the prefix
      const int32_t rc = launch_prefix_rows(s, p, c, plan.chunks, plan.chunk_blocks, carry);
      if (rc) return rc;
      a.carry_blocks = plan.chunk_blocks;
    } else {
      PagedArgs x = a;  // all rows of the batch as one sequence over the shared pages
      x.table = p.prefix_table;
      x.cols = p.prefix_cols;
      x.cap = p.max_prefix;
      x.len = p.prefix_len;
      x.prefix_len = nullptr;
      x.starts = nullptr;
      x.rows_end = p.q_starts ? p.q_starts + p.batch : nullptr;
      x.B = 1;
      x.T = p.n_rows;
      x.causal = 0;
      x.carry_out = carry;
      x.W = plan.prefix_workers;
      const int32_t rc = launch_rows(s, x, fp8, p.n_rows, "ema_prefix_attention prefix launch");
      if (rc) return rc;
    }
    a.carry_in = carry;
  } else if (!fp8 && paged_blocks((int64_t)p.max_q * a.G, p.batch, a.Hkv, device_cus())) {
    const int few = kFewRows / a.G;
    const int32_t rc = launch_paged_prefill(s, p, c, few);
    if (rc || !p.q_starts) return rc;  // (the same rows for all: every sequence is done)
    a.few = few;  // the sequences of few rows, and of more than the bound says, are left
    a.max_q = p.max_q;
  }
  a.W = plan.workers;
  return launch_rows(s, a, fp8, p.max_q, "ema_paged_attention launch");
}

}  // namespace ema
