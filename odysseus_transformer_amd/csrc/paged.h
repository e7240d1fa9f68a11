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
  const int* fresh;     // (S): how many of the n new ones it has, the last ones; null: all
  PageStrides sk, sv;
  int64_t table_stride;
  int pages, shift, width;
  unsigned k_page, k_row, v_page, v_row;   // bytes from page to page and from row to row (paged_check: rows of a page lie within 4 GiB, as pages' starts do)
  PagedCache(void* k_, void* v_, const int* table_, const int* lengths_, const int* fresh_, PageStrides sk_, PageStrides sv_, int64_t table_stride_, int pages_, int page_size,
             int width_, int dtype);
};

struct PagedAttnParams {
  const void* q;        // (S, n, Hq, D)
  void* out;            // (S, n, Hq, D)
  float* lse;           // (S, Hq, n)
  AttnStrides sq, so;
  int S, n, Hq, Hkv, group;
  float scale_log2e;    // above 0: a negative scale is the queries' sign, of a scale of 0 the queries are 0
  unsigned q_keep, q_flip;   // 32 bits of a query, two values or one: kept, then flipped
  int row_tiles;        // of one (sequence, kv head): its rows, token i, query head g of the group as row i * group + g, in tiles of `tile`
  int tile;
  float* part;          // [block][2][tile][D]: results of the first and the last unit of a block's range, where they are not whole
  float2* part_ml;      // [block][2][tile]: their maxima (of scores times log2 e) and sums
#ifdef __HIPCC__
  template <typename V> __device__ __forceinline__ V signed_query(V q) const {
    i32x4 x = __builtin_bit_cast(i32x4, q);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = (x[e] & q_keep) ^ q_flip;
    return __builtin_bit_cast(V, x);
  }
#endif
};

// The kernels of many rows (paged_attn_chunk.hip, paged_attn_wide.hip): rows of a tile, keys of a step
constexpr int PAGED_CHUNK_ROWS = 128, PAGED_WIDE_ROWS = 256, PAGED_CHUNK_KEYS = 64;

// How far the kernels count past a sequence's last key, in 32 bits, before they cut off what is behind it: the places of tiles whose page numbers go out ahead
// (paged_attn_wide.hip: 64 groups of 8 keys at a time, at most 1 080 past a key; paged_attn_chunk.hip: four tiles, 248) and a tile's or a step's end.  A table may hold
// 2^31 less so many places.
constexpr int PAGED_AHEAD = 4096;

// What a unit costs the kernels of many rows besides its steps, in steps: the latencies in front of the first products, queries in and results out.  It counts as
// so many steps at the unit's start, of which nothing comes.  (0 / 2 / 4 / 6 / 8: a prompt of 4096 tokens, 32 heads on 8, 253 / 232 / 204 / 187 / 188 us; 512
// tokens behind 8192 keys 95 / 95 / 90 / 87 / 88.)
constexpr int PAGED_EXTRA = 6;
__host__ __device__ constexpr int paged_extra(int tile) { return tile >= PAGED_CHUNK_ROWS ? PAGED_EXTRA : 0; }
#ifdef __HIPCC__
// Ranges that so many steps are cut into, one for a block, of which there are `most`.  With many rows four steps each at least (4 / 8 / 16, 32 heads on 8 behind 2000
// keys: 48 tokens 21 / 26 / 32 us, 128 tokens 26 / 28 / 34); 128 rows two blocks a compute unit only with 16 steps each (512 tokens behind 8192 keys 96 us, 111
// with one block; 17 behind 32768 with two blocks of 8 steps 52, with one 48).  A multiple of the units, where they are few: no range has parts of two of them if
// they are alike (3 sequences of 5000 keys, 40 heads on 10: 24.2 -> 22.6 us).
__device__ __forceinline__ int paged_blocks(const PagedAttnParams& p, int steps, int most) {
  int blocks = most;
  if (p.tile >= PAGED_CHUNK_ROWS && !(p.tile == PAGED_CHUNK_ROWS && steps >= 16 * most))
    blocks = max(1, min(p.tile == PAGED_CHUNK_ROWS ? most / 2 : most, steps / 4));
  const int units = p.S * p.row_tiles * p.Hkv;
  if (4 * units <= blocks) blocks -= blocks % units;
  return blocks;
}
#endif
int ody_launch_paged_wide(const PagedAttnParams& p, const PagedCache& c, int blocks, hipStream_t st);
int ody_launch_paged_chunk(const PagedAttnParams& p, int D, const PagedCache& c, int blocks, hipStream_t st);

#ifdef __HIPCC__
// ---- Division of the work.  A unit is a row tile of one (sequence, kv head); its work is a row of steps of STEP keys, up to the last key
// that its last row sees, one at least.  All steps of all units, in the order (kv head, sequence, row tile, step), are cut into gridDim.x
// ranges of equal length (to a step), so that blocks finish together whatever the lengths are; a unit that a cut goes through has its
// results joined by a second kernel.  Fewer steps than blocks: a step each, for as many as there are.  Every block finds its range by itself from the lengths on the device: a captured graph replays with
// the lengths of that time, and there is no plan to be kept.
// Tokens of a sequence; less than nothing is nothing.
__device__ __forceinline__ int paged_length(const PagedCache& c, int s) { return max(0, c.lengths[s]); }
// New tokens of sequence s, of n.
__device__ __forceinline__ int paged_fresh(const PagedCache& c, int s, int n) { return c.fresh ? max(0, min(c.fresh[s], n)) : n; }
// The arguments' cache lines at once, in front of everything: one after the other, where they are first needed, they are a latency each
// (one sequence of 8 192 tokens, 32 heads on 8, D=128: 14.2 -> 14.0 us; three of 500 to 2 048 in fp32, 8 heads, D=64: 13.3 -> 13.0;
// five new tokens of eight of 700 to 5 000, 16 heads on 4, D=64: 17.2 -> 16.9).
__device__ __forceinline__ void paged_arguments(const PagedAttnParams& p, const PagedCache& c) {
  asm volatile("" ::"s"(p.q), "s"(p.S), "s"(c.k), "s"(c.width), "s"((int)gridDim.x));
}
// Keys that the last row of a row tile sees, none if it has no token: places behind the table's last column have no page (the host checks width << shift <= 2^31 - PAGED_AHEAD).
__device__ __forceinline__ int paged_keys(const PagedAttnParams& p, const PagedCache& c, int length, int fresh, int rt) {
  const int last_row = min((rt + 1) * p.tile, p.n * p.group) - 1;   // rows, and a row tile more, are below 2^31 (paged_check)
  const int last = p.row_tiles == 1 ? p.n - 1 : last_row / p.group;
  return last < p.n - fresh ? 0 : max(0, min(c.width << c.shift, length - p.n + last + 1));
}
// Inclusive sums over the lanes of a wavefront, within rows of 16 lanes and then from row to row.
__device__ __forceinline__ int paged_wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // row_shr:1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, true);   // row_bcast:15 into rows 1 and 3, row_bcast:31 into 2 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, true);
  return x;
}

// The range that a block takes, of `blocks`: blocks of one XCD, which share its L2, take ranges in a row, so that row tiles of one (sequence, kv head) meet
// there.  Behind the last range: none.
__device__ __forceinline__ int paged_range(int block, int blocks) {
  const int each = (blocks + 7) / 8, range = (block & 7) * each + (block >> 3);
  return block >> 3 < each ? range : blocks;
}

// Where the cuts are: `total` steps (below 2^31, which the host checks) over as many of the blocks as there are steps for; the ranges that are a step longer lie evenly
// among the others.
struct PagedCuts {
  int total, blocks, base, more;
  __device__ __forceinline__ PagedCuts(int steps, int most_blocks) : total(steps), blocks(min(most_blocks, steps)) {
    base = (unsigned)total / (unsigned)blocks, more = total - base * blocks;
  }
  __device__ __forceinline__ int at(int range) const { return range * base + (int)((unsigned)(range * more) / (unsigned)blocks); }
  __device__ __forceinline__ int range_of(int step) const {
    int r = min(blocks - 1, (int)((float)step * (float)blocks / (float)total));   // at most one off
    if (at(r) > step) r--;
    if (at(r + 1) <= step) r++;
    return r;
  }
};

// A walk over the (sequence, row tile) pairs by a wavefront, a chunk of 64 of them at a time: a lane has the length of its pair's sequence, the pair's
// steps and the sum of steps so far.  Where there are more pairs, total() first sums up 64 equal shares of them, a lane each, whose loads do not wait for one another,
// and find() starts with the share that a step is in (1024 sequences of 100 keys, 8 kv heads: 112 -> 106 us).
template <int STEP>
struct PagedWalk {
  const PagedAttnParams& p;
  const PagedCache& c;
  int lane, entries, at = 0, before = 0, length = 0, fresh = 0, mine = 0, sums = 0;   // sums: inclusive, of this chunk
  int share = 1, share_mine = 0, share_sums = 0;
  __device__ __forceinline__ PagedWalk(const PagedAttnParams& p_, const PagedCache& c_, int lane_) : p(p_), c(c_), lane(lane_), entries(p_.S * p_.row_tiles) { chunk(); }
  __device__ __forceinline__ int steps_of(int e, int& len, int& new_) const {
    const int s = p.row_tiles == 1 ? e : e / p.row_tiles;
    len = paged_length(c, s), new_ = paged_fresh(c, s, p.n);
    return max(1, (paged_keys(p, c, len, new_, e - s * p.row_tiles) - 1) / STEP + 1) + paged_extra(p.tile);
  }
  __device__ __forceinline__ void chunk() {
    mine = at + lane < entries ? steps_of(at + lane, length, fresh) : 0;
    sums = paged_wave_scan(mine);
  }
  __device__ __forceinline__ int all() const { return __builtin_amdgcn_readlane(sums, 63); }
  __device__ __forceinline__ bool next() {
    if (at + 64 >= entries) return false;
    before += all(), at += 64;
    chunk();
    return true;
  }
  __device__ __forceinline__ int total() {   // of one kv head
    if (entries <= 64) return all();
    share = (entries + 63) / 64;
    const int end = min(entries, (lane + 1) * share);
#pragma unroll 8
    for (int e = lane * share; e < end; e++) {
      int len, new_;
      share_mine += steps_of(e, len, new_);
    }
    share_sums = paged_wave_scan(share_mine);
    return __builtin_amdgcn_readlane(share_sums, 63);
  }
  __device__ __forceinline__ void start(int k) {   // with share k
    at = k * share, before = __builtin_amdgcn_readlane(share_sums, k) - __builtin_amdgcn_readlane(share_mine, k);
    chunk();
  }
  // behind total(): the chunk that step `pos` is in, or pair `entry`
  __device__ __forceinline__ void find(int pos) {
    if (entries > 64) start(__popcll(__ballot(share_sums <= pos)));
    while (before + all() <= pos && next()) {}
  }
  __device__ __forceinline__ void find_entry(int entry) {
    if (entries > 64) start(entry / share);
    while (entry >= at + 64) next();
  }
  __device__ __forceinline__ void rewind() {
    if (at == 0) return;
    at = before = 0;
    chunk();
  }
};

// A place in the order of all steps: kv head, pair (sequence, row tile), step of it.
template <int STEP>
struct PagedPlace {
  int hk, entry, s, rt, length, fresh, steps, step;
  // that of step `pos`, `each` of every kv head
  __device__ __forceinline__ PagedPlace(PagedWalk<STEP>& w, int pos, int each) {
    hk = (int)((unsigned)pos / (unsigned)each);
    pos -= hk * each;
    w.find(pos);
    entry = w.at + __popcll(__ballot(w.before + w.sums <= pos));
    take(w);
    step = pos - (w.before + __builtin_amdgcn_readlane(w.sums, entry - w.at) - steps);
  }
  // the first step of the next unit
  __device__ __forceinline__ void next_unit(PagedWalk<STEP>& w) {
    if (++entry == w.entries) {
      entry = 0, hk++;
      w.rewind();
    } else if (entry == w.at + 64) {
      w.next();
    }
    take(w);
    step = 0;
  }

 private:
  __device__ __forceinline__ void take(const PagedWalk<STEP>& w) {
    const int k = entry - w.at;
    steps = __builtin_amdgcn_readlane(w.mine, k), length = __builtin_amdgcn_readlane(w.length, k), fresh = __builtin_amdgcn_readlane(w.fresh, k);
    s = w.p.row_tiles == 1 ? entry : entry / w.p.row_tiles, rt = entry - s * w.p.row_tiles;
  }
};
#endif

// Host side: the checks that both entry points share.
int paged_check(const char* who, int S, int n, int Hq, int Hkv, int D, int dtype, const PagedCache& c, int page_size);
static inline bool paged_rows_aligned(const void* ptr, int64_t a, int64_t b, int64_t c, int dtype) {
  const int q = dtype == ODY_BF16 ? 8 : 4;
  return ody_aligned16(ptr) && a % q == 0 && b % q == 0 && c % q == 0;
}
static inline int paged_shift(int page_size) { return page_size > 0 ? __builtin_ctz((unsigned)page_size) : 0; }
