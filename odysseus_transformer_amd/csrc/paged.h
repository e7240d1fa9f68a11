// A key / value cache in pages, as the kernels that fill and read it see it, and the division of attention over it among blocks.
#pragma once
#include "attn_params.h"

struct PageStrides {
  int64_t p, r, h;  // page, row of a page, head: elements; head_dim stride is 1
};

struct PagedCache {
  void* k;              // (pages, page size, Hkv, D)
  void* v;
  const int* table;     // (S, width): page of rows [c << shift, (c + 1) << shift) of a sequence; outside [0, pages): none
  const int* lengths;   // (S): tokens of the sequence, the new ones included
  PageStrides sk, sv;
  int64_t table_stride;
  int pages, shift, width;
};

struct PagedAttnParams {
  const void* q;        // (S, n, Hq, D)
  void* out;            // (S, n, Hq, D)
  float* lse;           // (S, Hq, n)
  AttnStrides sq, so;
  int S, n, Hq, Hkv, group;
  float scale_log2e;
  int row_tiles;        // of one (sequence, kv head): its rows, token i, query head g of the group as row i * group + g, in tiles of `tile`
  int tile;
  float* part;          // [block][2][tile][D]: results of the first and the last unit of a block's range, where they are not whole
  float2* part_ml;      // [block][2][tile]: their maxima (of scores times log2 e) and sums
};

#ifdef __HIPCC__
// ---- Division of the work.  A unit is a row tile of one (sequence, kv head); its work is a row of steps of STEP keys, up to the last key
// that its last row sees, one at least.  All steps of all units, in the order (sequence, row tile, kv head, step), are cut into gridDim.x
// ranges of equal length (to a step), so that blocks finish together whatever the lengths are; a unit that a cut goes through has its
// results joined by a second kernel.  Fewer steps than blocks: a step each, for as many as there are.  Every block finds its range by itself from the lengths on the device: a captured graph replays with
// the lengths of that time, and there is no plan to be kept.
struct PagedUnit {
  int s, rt;        // sequence, row tile
  int steps;
};

// Tokens of a sequence; less than nothing is nothing.
__device__ __forceinline__ int paged_length(const PagedCache& c, int s) { return max(0, c.lengths[s]); }
// Keys that the last row of a row tile sees: places behind the table's last column have no page (the host checks width << shift < 2^31).
__device__ __forceinline__ int paged_keys(const PagedAttnParams& p, const PagedCache& c, int length, int rt) {
  const int64_t last_row = min((int64_t)(rt + 1) * p.tile, (int64_t)p.n * p.group) - 1;
  return max(0, min(c.width << c.shift, length - p.n + (int)(last_row / p.group) + 1));
}
template <int STEP>
__device__ __forceinline__ int paged_steps(const PagedAttnParams& p, const PagedCache& c, int e) {
  const int s = e / p.row_tiles, keys = paged_keys(p, c, paged_length(c, s), e - s * p.row_tiles);
  return max(1, (int)(((int64_t)keys + STEP - 1) / STEP));
}

// Every lane of a wavefront: inclusive sums over its lanes.
__device__ __forceinline__ int paged_wave_scan(int x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  return x;
}
// Steps of all (sequence, row tile) pairs of one kv head.
template <int STEP>
__device__ __forceinline__ int64_t paged_total(const PagedAttnParams& p, const PagedCache& c, int lane) {
  const int entries = p.S * p.row_tiles;
  int64_t total = 0;
  for (int at = 0; at < entries; at += 64) {
    const int x = paged_wave_scan(at + lane < entries ? paged_steps<STEP>(p, c, at + lane) : 0, lane);
    total += __builtin_amdgcn_readlane(x, 63);
  }
  return total;
}
// The pair that step `pos` (of all kv heads together) belongs to, and the first step of it.
template <int STEP>
__device__ __forceinline__ int paged_find(const PagedAttnParams& p, const PagedCache& c, int lane, int64_t pos, int64_t& first, int& steps) {
  const int entries = p.S * p.row_tiles;
  int64_t before = 0;
  for (int at = 0;; at += 64) {
    const int mine = at + lane < entries ? paged_steps<STEP>(p, c, at + lane) : 0, x = paged_wave_scan(mine, lane);
    const int all = __builtin_amdgcn_readlane(x, 63);
    if (pos < (before + all) * p.Hkv || at + 64 >= entries) {
      const int k = min(__popcll(__ballot((before + x) * p.Hkv <= pos)), min(63, entries - 1 - at));
      steps = __builtin_amdgcn_readlane(mine, k);
      first = (before + __builtin_amdgcn_readlane(x, k) - steps) * p.Hkv;
      return at + k;
    }
    before += all;
  }
}
__device__ __forceinline__ int64_t paged_cut(int64_t total, int block, int blocks) { return total / blocks * block + total % blocks * block / blocks; }
// The block whose range holds step `pos`.
__device__ __forceinline__ int paged_block_of(int64_t total, int64_t pos, int blocks) {
  int b = (int)min((int64_t)blocks - 1, (int64_t)((double)pos * blocks / (double)total));
  while (b > 0 && paged_cut(total, b, blocks) > pos) b--;
  while (b + 1 < blocks && paged_cut(total, b + 1, blocks) <= pos) b++;
  return b;
}
#endif

// Host side: the checks that both entry points share.
int paged_check(const char* who, int S, int n, int Hq, int Hkv, int D, int dtype, const PagedCache& c, int page_size);
static inline bool paged_rows_aligned(const void* ptr, int64_t a, int64_t b, int64_t c, int dtype) {
  const int q = dtype == ODY_BF16 ? 8 : 4;
  return ody_aligned16(ptr) && a % q == 0 && b % q == 0 && c % q == 0;
}
static inline int paged_shift(int page_size) { return page_size > 0 ? __builtin_ctz((unsigned)page_size) : 0; }
