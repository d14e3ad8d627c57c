// Shared pieces of the paged-cache kernels: how packed rows, pages and work are addressed.
//
// A page pool is a ema_kvcache_desc of n_pages "sequences" of page_size "positions"; row b of
// the block table names the pages of sequence b. The integer parts are host/device functions,
// checked on the CPU (tests/cpp/test_paged.cpp).
#pragma once

#include "ema_schedule.hpp"

namespace ema {

constexpr int kPagedMaxB = 1024;    // sequences of one call (the kernels' tables in LDS)
constexpr int kPagedRows = 32;      // query rows of a segment: (token, head of the kv group) pairs
constexpr int kPagedTile = 32;      // keys per tile
constexpr int kPagedWaves = 4;      // waves per workgroup, each with tiles of its own
constexpr int kPagedMaxWorkers = 512;
constexpr int kPagedState = 128 + 4;  // floats of a row's partial state: m, l, pad, pad, o[128]
constexpr int kPagedMinPage = 16;   // a wave's 1 KB loads (4 rows) never straddle two pages

// Query rows of sequence b: packed rows [begin, begin + n). Row starts from the device are
// taken as given only inside [0, n_rows].
struct PagedRows {
  int begin, n;
};
EMA_HD PagedRows paged_rows(int s0, int s1, int n_rows) {
  s0 = s0 < 0 ? 0 : (s0 > n_rows ? n_rows : s0);
  s1 = s1 < s0 ? s0 : (s1 > n_rows ? n_rows : s1);
  return PagedRows{s0, s1 - s0};
}

// Key tiles of L positions, and rounds of n tiles: a round is one tile for each wave of a workgroup.
EMA_HD int paged_tiles(int L) { return (int)(((uint32_t)L + kPagedTile - 1) / kPagedTile); }
EMA_HD int paged_rounds(int tiles) { return (tiles + kPagedWaves - 1) / kPagedWaves; }

// Units of a segment: one round each, or kPagedLongUnit rounds where the rounds are more than the
// workgroups, or more than 16 for a segment, and no more than kPagedLongUnit for each workgroup.
// A piece costs a workgroup about as much as three rounds before and after its tiles, and the
// joining workgroup a load's round trip per 16 pieces, so short segments (own tokens behind a
// prefix) are better whole and long ones better in fewer pieces than there are rounds: one
// sequence's 32 rows after 8000 keys (32 heads on 8) 47 us in pieces of one round, 24 of four.
constexpr int kPagedLongUnit = 4;
EMA_HD int paged_units(int rounds, int unit) { return (rounds + unit - 1) / unit; }
EMA_HD int paged_unit(int rounds, int segments, int W) {
  return (rounds > W || rounds > 16 * (int64_t)segments) && rounds <= kPagedLongUnit * W ? kPagedLongUnit : 1;
}

// The units of all segments, laid end to end, cut into W slices that differ by at most one
// unit; 32-bit arithmetic without products of the two (total < 2^31).
struct PagedSplit {
  uint32_t base, rem;  // every slice has base units, the first rem of them one more
};
EMA_HD int paged_active_workers(int total, int W) { return total < W ? (total < 1 ? 1 : total) : W; }
EMA_HD PagedSplit paged_split(int total, int W) {
  if (total == W) return PagedSplit{1u, 0u};  // (no division on the small calls' path)
  const uint32_t base = (uint32_t)total / (uint32_t)W;
  return PagedSplit{base, (uint32_t)total - base * (uint32_t)W};
}
EMA_HD int paged_begin(PagedSplit s, int w) { return (int)((uint32_t)w * s.base + ((uint32_t)w < s.rem ? (uint32_t)w : s.rem)); }
EMA_HD int paged_worker_of(PagedSplit s, int t) {
  if (s.base == 1 && s.rem == 0) return t;
  const uint32_t cut = s.rem * (s.base + 1);
  return (int)((uint32_t)t < cut ? (uint32_t)t / (s.base + 1) : s.rem + ((uint32_t)t - cut) / s.base);
}
// Partial-state slot of worker w's piece of a segment that several workers share. A slice
// shares at most two segments: the one it begins inside (slot 2 w) and the one that begins
// inside it and runs on (slot 2 w + 1, w then being the segment's first worker w0).
EMA_HD int paged_slot(int w, int w0) { return 2 * w + (w == w0 ? 1 : 0); }

// r / G for r < 2^23 by a product: magic = ceil(2^32 / G), exact while r * G < 2^32 (G <= 256).
constexpr int kPagedMaxGroup = 256;
EMA_HD uint32_t paged_magic(int G) { return G == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + G - 1) / (uint64_t)G); }
EMA_HD int paged_div(int r, uint32_t magic) { return magic ? (int)(((uint64_t)(uint32_t)r * magic) >> 32) : r; }

// Workers the plan sizes the workspace for, from the host's bounds: nrb row blocks per kv head
// (all sequences), max_tiles key tiles each.
EMA_HD int paged_plan_workers(int64_t nrb, int Hkv, int max_tiles) {
  const int64_t want = nrb * Hkv * paged_rounds(max_tiles);
  return (int)(want < 1 ? 1 : (want < kPagedMaxWorkers ? want : kPagedMaxWorkers));
}
// log2 of a page size.
EMA_HD int paged_shift(int page) {
  int s = 0;
  while ((1 << s) < page) ++s;
  return s;
}
// Row blocks of a batch whose sequences have at most max_q rows and n_rows together (a bound of
// none, which any row is past, counts as one).
EMA_HD int64_t paged_row_blocks(int B, int64_t n_rows, int64_t max_q, int G) {
  if (max_q < 1) max_q = 1;
  const int64_t each = (int64_t)B * ((max_q * G + kPagedRows - 1) / kPagedRows);
  const int64_t all = n_rows * G / kPagedRows + B;
  return each < all ? each : all;
}

// A shared prefix cut into chunks of 64-key blocks for its row blocks of 128 over all kv heads:
// as many chunks as give the chip one workgroup per CU, of two blocks at least (one for each
// half of a workgroup).
struct PagedChunks {
  int n, blocks;  // chunks, and 64-key blocks of each
};
EMA_HD PagedChunks paged_chunks(int64_t rows, int Hkv, int max_prefix, int cus) {
  const int64_t wgs = (rows > 0 ? (rows + 127) / 128 : 1) * Hkv;
  const int total = (int)(((int64_t)max_prefix + 63) / 64);
  int64_t n = cus / wgs;
  if (n > (total + 1) / 2) n = (total + 1) / 2;
  if (n < 1) n = 1;
  PagedChunks c;
  c.blocks = (int)((total + n - 1) / n);
  c.n = (total + c.blocks - 1) / c.blocks;
  return c;
}

#if defined(__HIPCC__)
// Constant-address-space loads: table entries, lengths and row starts are uniform over a wave
// and not written by the kernels, so they come as scalar loads.
typedef const __attribute__((address_space(4))) int32_t paged_cint;
__device__ __forceinline__ int ld_uniform(const int32_t* p, int64_t i) { return ((paged_cint*)p)[i]; }
// Sum of v over this lane and those before it, by DPP: within rows of 16, then across them.
__device__ __forceinline__ int sum_up_to_lane(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);  // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);  // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);  // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return v;
}
#endif

}  // namespace ema
