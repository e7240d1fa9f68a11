// The second kernel of attention over a cache in pages: joins the results of units that a cut between blocks goes through.
#pragma once
#include <algorithm>
#include "paged.h"

namespace {

// The parts of the units that a cut goes through, weighted by their sums, with D / 4 threads on a row: the parts of a lone row are read by all threads of a block, of
// several each is a group's of them.
// BY_CUTS, where those are fewer blocks: a block takes PAGED_JOIN_ROWS rows of a row tile (which are a divisor of it) at a cut, and the cuts through a unit
// share its rows.  Else it takes R rows of a unit.  (8 tokens of 256 sequences of up to 1000 keys, 32 heads on 8: 158 us in all, 191 with a block for each row of
// each unit; 512 tokens of one behind 8192 keys by cuts 103, by units 91, 131 with R = 1; 17 behind 16000, more than 16 parts, 31, 36 with all threads on the
// rows in turn.)
constexpr int PAGED_JOIN_ROWS = 8;
template <typename T, int D, int STEP, int R, bool BY_CUTS>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedAttnParams p, const PagedCache cache, int most_blocks) {
  constexpr int C4 = D / 4, GROUPS = 256 / C4, U = 4;
  static_assert(GROUPS >= R, "a group of threads for each of a block's rows");
  __shared__ f32x4 red[GROUPS][C4];
  __shared__ float2 red_ml[GROUPS];
  paged_arguments(p, cache);
  const int tid = threadIdx.x, lane = tid & 63, all_rows = p.n * p.group, extra = paged_extra(p.tile);
  PagedWalk<STEP> walk(p, cache, lane);
  const int each = walk.total();
  const PagedCuts cuts(each * p.Hkv, paged_blocks(p, each * p.Hkv, most_blocks));
  // the unit's place, its first step, how many it has; the block's rows are row0 + mine, row0 + mine + through .. of the kv head's, R of them for through = 1
  int hk, s, rt, row0, first, steps, mine = 0, through = 1;
  if (BY_CUTS) {   // blockIdx.x: (cut, R rows of a row tile)
    const int row_blocks = (min(p.tile, all_rows) + R - 1) / R, cut = 1 + blockIdx.x / row_blocks;
    if (cut >= cuts.blocks) return;
    const PagedPlace<STEP> at(walk, cuts.at(cut), each);
    if (at.step <= extra) return;   // between two units, or in what one costs besides its steps
    hk = at.hk, s = at.s, rt = at.rt, steps = at.steps, first = cuts.at(cut) - at.step, row0 = rt * p.tile + blockIdx.x % row_blocks * R, mine = cut;
  } else {         // (sequence, R rows of a kv head, kv head)
    const int row_blocks = (all_rows + R - 1) / R;
    hk = blockIdx.x % p.Hkv, row0 = blockIdx.x / p.Hkv % row_blocks * R, s = blockIdx.x / p.Hkv / row_blocks;
    rt = row0 / p.tile;
    const int entry = s * p.row_tiles + rt;
    walk.find_entry(entry);
    steps = __builtin_amdgcn_readlane(walk.mine, entry - walk.at);
    first = hk * each + walk.before + __builtin_amdgcn_readlane(walk.sums, entry - walk.at) - steps;
  }
  const int b0 = cuts.range_of(first + extra), b1 = cuts.range_of(first + steps - 1), parts = b1 - b0 + 1;   // ranges with keys of the unit
  if (parts == 1) return;
  if (BY_CUTS) mine -= b0 + 1, through = parts - 1;
  // part k is in slot 2 (b0 + k), but for the first where that block's range begins with another unit
  const int first_slot = 2 * b0 + (first > cuts.at(b0));
  const int d4 = tid % C4, g = tid / C4;
  auto write = [&](int row, float m, float l, f32x4 acc) {
    const int i = row / p.group, h = hk * p.group + row - i * p.group;
    typedef T out4 __attribute__((ext_vector_type(4)));
    acc *= l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<out4*>(static_cast<T*>(p.out) + s * p.so.b + i * p.so.l + h * p.so.h + 4 * d4) = out4{(T)acc[0], (T)acc[1], (T)acc[2], (T)acc[3]};
    if (d4 == 0) p.lse[((int64_t)s * p.Hq + h) * p.n + i] = l == 0.f ? -INFINITY : (m + __log2f(l)) * ODY_LN2;
  };
  // parts from .. in steps of `by`, U at a time
  auto sum = [&](int row, int from, int by, float& m, float& l, f32x4& acc) {
    const int r = row - rt * p.tile;
    m = -INFINITY, l = 0.f, acc = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = from; k < parts; k += U * by) {
      float2 ml[U];
      f32x4 o[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int part = min(k + u * by, parts - 1);
        const int64_t at = (int64_t)(part == 0 ? first_slot : 2 * (b0 + part)) * p.tile + r;
        ml[u] = p.part_ml[at];
        o[u] = *reinterpret_cast<const f32x4*>(p.part + at * D + 4 * d4);
      }
      float now = m;
#pragma unroll
      for (int u = 0; u < U; u++)
        if (u == 0 || k + u * by < parts) now = fmaxf(now, ml[u].x);
      const float ref = now == -INFINITY ? 0.f : now, old = ody_exp2(m - ref);
      m = now, l *= old, acc *= old;
#pragma unroll
      for (int u = 0; u < U; u++)
        if (u == 0 || k + u * by < parts) {
          const float w = ody_exp2(ml[u].x - ref);
          l += ml[u].y * w, acc += o[u] * w;
        }
    }
  };
  float m, l;
  f32x4 acc;
  if (through < R) {
    const int row = row0 + mine + through * g;
    if (mine + through * g < R && row < all_rows) {
      sum(row, 0, 1, m, l, acc);
      write(row, m, l, acc);
    }
    return;
  }
  const int row = row0 + mine;
  if (mine >= R || row >= all_rows) return;
  sum(row, g, GROUPS, m, l, acc);
  red[g][d4] = acc;
  if (d4 == 0) red_ml[g] = make_float2(m, l);
  __syncthreads();
  if (g == 0) {
    m = -INFINITY, l = 0.f, acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < GROUPS; k++) m = fmaxf(m, red_ml[k].x);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int k = 0; k < GROUPS; k++) {
      const float w = ody_exp2(red_ml[k].x - ref);
      l += red_ml[k].y * w, acc += red[k][d4] * w;
    }
    write(row, m, l, acc);
  }
}

template <typename T, int D, int STEP, int R>
int paged_join(const PagedAttnParams& p, const PagedCache& c, bool joined, int blocks, hipStream_t st) {
  if (!joined) return ODY_OK;
  const int64_t rows = (int64_t)p.n * p.group, by_units = p.S * ((rows + R - 1) / R) * p.Hkv,
                by_cuts = (blocks - 1) * ((std::min(rows, (int64_t)p.tile) + PAGED_JOIN_ROWS - 1) / PAGED_JOIN_ROWS);
  if (by_cuts < by_units) ODY_LAUNCH("paged_join", st, (paged_join_kernel<T, D, STEP, PAGED_JOIN_ROWS, true>), dim3((unsigned)by_cuts), dim3(256), 0, p, c, blocks);
  else ODY_LAUNCH("paged_join", st, (paged_join_kernel<T, D, STEP, R, false>), dim3((unsigned)by_units), dim3(256), 0, p, c, blocks);
  return ody_check_launch("paged_join");
}

}  // namespace
