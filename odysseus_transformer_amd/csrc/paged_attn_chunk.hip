// Attention of many new tokens over a key / value cache in pages, bf16: a chunk of a prompt, more than 64 rows of a kv head (its query heads
// times the tokens).
//
// Bound by the matrix cores and, as much, by the vector work of the softmax between the two products.  A block of four wavefronts takes 128 rows of one
// (sequence, kv head), 32 a wavefront, and streams the keys in tiles of 64, which direct loads bring to LDS a tile ahead (the page numbers two).  Both
// products are computed transposed, so that a row's maximum, sum and rescaling belong to one lane and the one 32 lanes away:
//
//      S^T (keys x rows) = K Q^T        A: K rows from LDS      B: this lane's query row, in registers
//      O^T (D x rows) += V^T P^T        B: P^T as the accumulators of S^T hold it      A: V^T by transposing LDS reads
//
// on v_mfma_f32_32x32x16_bf16, tiles laid out and read as attn_rowtile.h has it.
#include <cmath>
#include <type_traits>
#include "attn_rowtile.h"
#include "paged.h"

namespace {

using namespace rowtile;

constexpr int KEYS = PAGED_CHUNK_KEYS, BLOCK_ROWS = PAGED_CHUNK_ROWS, WAVES = 4;
static_assert(KEYS == ROWS && BLOCK_ROWS == 32 * WAVES, "a tile of keys, 32 rows a wavefront");

__device__ const bf16x8 no_key[16] = {};   // the row that a key without a page, or behind the last one, is read from

template <int D>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_chunk_kernel(const PagedAttnParams p, const PagedCache cache) {
  constexpr int KS = D / 16, DT = D / 32, TILE = KEYS * D, STAGE = 2 * TILE;         // elements
  constexpr int LANES = D / 8, PER = 64 / LANES, STEP = PER * WAVES, LOADS = KEYS / STEP;   // of a direct load: lanes on a row, rows; of a tile
  static_assert(STEP % 16 == 0, "swz of the rows of the other loads");
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  bf16* stages = reinterpret_cast<bf16*>(smem);   // [2][K tile | V tile]

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 5, i = lane & 31;
  PagedWalk<KEYS> walk(p, cache, lane);
  const PagedCuts cuts(walk.total() * p.Hkv, gridDim.x);
  const int block = blockIdx.x;
  if (block >= cuts.blocks) return;
  const int begin = cuts.at(block), end = cuts.at(block + 1);
  int pos = begin, hk, step, steps, entry = walk.find(pos, hk, step, steps);
  const int lrow = PER * wave + lane / LANES, lcol = 8 * ((lane % LANES) ^ swz<D>(lrow));   // of this lane in the first direct load
  const int64_t lk = lane / LANES * cache.sk.r + lcol, lv = lane / LANES * cache.sv.r + lcol;
  const float c2 = p.scale_log2e;
  Readers<D> rd;
  rd.init(stages, g, i);

  while (pos < end) {
    const int s = p.row_tiles == 1 ? entry : entry / p.row_tiles, rt = entry - s * p.row_tiles, row0 = rt * BLOCK_ROWS;
    const int rows = min(BLOCK_ROWS, p.n * p.group - row0), length = paged_length(cache, s);
    const int keys = paged_keys(p, cache, length, rt), steps_here = min(steps - step, end - pos), tiles = keys > 0 ? steps_here : 0;
    const bf16* kp = static_cast<const bf16*>(cache.k) + hk * cache.sk.h;
    const bf16* vp = static_cast<const bf16*>(cache.v) + hk * cache.sv.h;
    const int* table = cache.table + s * cache.table_stride;

    // ---- lane n % 8 holds the page of the tile's n-th group of 8 keys; the rows of a direct load are in one of them
    auto lookup = [&](int t) { return table[min((step + t) * KEYS + 8 * (lane & 7), keys - 1) >> cache.shift]; };
    auto load = [&](int t, int pages, unsigned have) {
      bf16* stage = stages + (t & 1) * STAGE;
#pragma unroll
      for (int j = 0; j < LOADS; j++) {
        const int first = STEP * j + PER * wave, key = (step + t) * KEYS + first, row = key & ((1 << cache.shift) - 1);
        const int page = __builtin_amdgcn_readlane(pages, first / 8);
        const bf16* ks = kp + page * cache.sk.p + row * cache.sk.r + lk;
        const bf16* vs = vp + page * cache.sv.p + row * cache.sv.r + lv;
        if (key + PER > keys || (have >> (first / 8) & 1) == 0) {
          const bool none = key + lane / LANES >= keys || (have >> (first / 8) & 1) == 0;
          const bf16* zero = reinterpret_cast<const bf16*>(no_key) + lcol;
          ks = none ? zero : ks, vs = none ? zero : vs;
        }
        __builtin_amdgcn_global_load_lds((global_ptr)ks, (lds_ptr)(stage + (WAVES * j + wave) * 512), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((global_ptr)vs, (lds_ptr)(stage + TILE + (WAVES * j + wave) * 512), 16, 0, 0);
      }
    };
    auto have_pages = [&](int pages) { return (unsigned)__builtin_amdgcn_ballot_w64((unsigned)pages < (unsigned)cache.pages) & 0xff; };
    int next = 0;
    unsigned have = 0;
    if (tiles > 0) {
      next = lookup(0);
      have = have_pages(next);
      load(0, next, have);
      next = lookup(1);
    }

    // ---- this lane's row: token ri, query head h
    const int r = row0 + min(32 * wave + i, rows - 1), ri = r / p.group, h = hk * p.group + r - ri * p.group;
    bf16x8 qf[KS];
    {
      const bf16* qp = static_cast<const bf16*>(p.q) + s * p.sq.b + ri * p.sq.l + h * p.sq.h + 8 * g;
#pragma unroll
      for (int ks = 0; ks < KS; ks++) qf[ks] = p.signed_query(*reinterpret_cast<const bf16x8*>(qp + 16 * ks));
    }
    const int lim = min(keys - 1, length - p.n + ri);   // last key that it sees
    const int first_row = min(32 * wave, rows - 1), last_row = min(32 * wave + 31, rows - 1);
    const int safe = __builtin_amdgcn_readfirstlane(min(keys - 1, length - p.n + (row0 + first_row) / p.group));   // ... that all of the wavefront's see
    const int seen = 32 * wave < rows ? __builtin_amdgcn_readfirstlane(min(keys - 1, length - p.n + (row0 + last_row) / p.group)) : -1;

    f32x16 o[DT];
    clear(o);
    float ref = -INFINITY, l4[4] = {0.f, 0.f, 0.f, 0.f};
    auto tile = [&](int n0, unsigned have) {
      f32x16 x[2];
#pragma unroll
      for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int kt = 0; kt < 2; kt++) x[kt] = mfma32(row_frag(rd, 32 * kt, ks), qf[ks], ks == 0 ? f32x16{0} : x[kt]);
      if (n0 + KEYS - 1 > safe || have != 0xff) {
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
          for (int e = 0; e < 16; e++)
            if (n0 + 32 * kt + acc_row(e, g) > lim || (have >> (4 * kt + (e >> 2)) & 1) == 0) x[kt][e] = -INFINITY;
      }
      float top = fmaxf(x[0][0], x[1][0]);
#pragma unroll
      for (int e = 1; e < 16; e++) top = fmaxf(top, fmaxf(x[0][e], x[1][e]));
      top = half_swap_max(top) * c2;
      if (__builtin_amdgcn_ballot_w64(top > ref) != 0) {   // somebody's maximum has grown
        const float now = fmaxf(ref, top), alpha = now == -INFINITY ? 1.f : ody_exp2(ref - now);
        ref = now;
#pragma unroll
        for (int e = 0; e < 4; e++) l4[e] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
          for (int e = 0; e < 16; e++) o[dt][e] *= alpha;
      }
      const float minus = ref == -INFINITY ? 0.f : -ref;
      auto half = [&](auto which) {
        constexpr int kt = decltype(which)::value;
        bf16x8 pb[2], vf[2];
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const float w = ody_exp2(fmaf(x[kt][e], c2, minus));
          l4[e & 3] += w;
          pb[e >> 3][e & 7] = (bf16)w;
        }
        auto product = [&](auto slice) {   // 16 keys, 64 columns
          constexpr int ss = decltype(slice)::value & 1, hf = decltype(slice)::value >> 1;
          tr_frags<ROWS + 32 * kt + 16 * ss, hf>(vf, rd);
#pragma unroll
          for (int dt = 0; dt < 2; dt++) o[2 * hf + dt] = mfma32(vf[dt], pb[ss], o[2 * hf + dt]);
        };
        product(std::integral_constant<int, 0>{});
        if constexpr (D == 128) product(std::integral_constant<int, 2>{});
        product(std::integral_constant<int, 1>{});
        if constexpr (D == 128) product(std::integral_constant<int, 3>{});
      };
      half(std::integral_constant<int, 0>{});
      half(std::integral_constant<int, 1>{});
    };
    for (int t = 0; t < tiles; t++) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();   // the tile has landed, and everyone is done with the one before
      const unsigned now = have;
      if (t + 1 < tiles) {
        have = have_pages(next);
        load(t + 1, next, have);
        next = lookup(t + 2);
      }
      const int n0 = (step + t) * KEYS;
      if (n0 <= seen) tile(n0, now);
      rd.move(t & 1 ? -(int)(STAGE * sizeof(bf16)) : (int)(STAGE * sizeof(bf16)));
    }
    if (tiles & 1) rd.move(-(int)(STAGE * sizeof(bf16)));
    __syncthreads();   // everyone is done with the stages

    const float sum = half_swap_sum((l4[0] + l4[1]) + (l4[2] + l4[3]));
    if (32 * wave + i < rows) {
      if (steps_here == steps) {
        store_row(static_cast<bf16*>(p.out) + s * p.so.b + ri * p.so.l + h * p.so.h, o, sum == 0.f ? 0.f : 1.f / sum, g);
        if (g == 0) p.lse[((int64_t)s * p.Hq + h) * p.n + ri] = sum == 0.f ? -INFINITY : (ref + __log2f(sum)) * ODY_LN2;
      } else {
        const int64_t at = (int64_t)(2 * block + (pos > begin)) * BLOCK_ROWS + 32 * wave + i;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
          for (int a = 0; a < 4; a++)
            *reinterpret_cast<f32x4*>(p.part + at * D + 32 * dt + 8 * a + 4 * g) = f32x4{o[dt][4 * a], o[dt][4 * a + 1], o[dt][4 * a + 2], o[dt][4 * a + 3]};
        if (g == 0) p.part_ml[at] = make_float2(ref, sum);
      }
    }
    pos += steps_here;
    step = 0;
    if (++hk == p.Hkv && pos < end) hk = 0, steps = paged_steps<KEYS>(p, cache, ++entry);
  }
}

template <int D>
int launch(const PagedAttnParams& p, const PagedCache& c, int blocks, hipStream_t st) {
  constexpr size_t smem = (size_t)4 * KEYS * D * sizeof(bf16);
  if (int rc = ody_allow_dynamic_lds(reinterpret_cast<const void*>(&paged_chunk_kernel<D>), smem, "ody_paged_attn")) return rc;
  ODY_LAUNCH("paged_chunk", st, (paged_chunk_kernel<D>), dim3(blocks), dim3(64 * WAVES), smem, p, c);
  return ody_check_launch("paged_chunk");
}

}  // namespace

int ody_launch_paged_chunk(const PagedAttnParams& p, int D, const PagedCache& c, int blocks, hipStream_t st) {
  return D == 64 ? launch<64>(p, c, blocks, st) : launch<128>(p, c, blocks, st);
}
