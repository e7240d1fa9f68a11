// Attention of long chunks over a key / value cache in pages that holds its values in 8 bits, bf16 queries, heads of 128: row tiles of 256, of which
// paged_q8_chunk.hip takes 128.
//
// The pipeline over row tiles of 256 of paged_attn_wide.hip, which says how its phases and references work: a wavefront a SIMD, 64 rows each.  Tiles come through registers here: a wavefront
// takes two groups of eight keys of K and of V, whose scale is one number each, converts them -- exactly, 16 products' operands a turn and not 128, as where each wavefront
// converts what it multiplies -- and writes them to LDS as bf16, in the order in which the products read them:
//
//      under S^T(t + 1), first 32 keys        K of tile t + 2 is converted
//      under O^T += P(t), first 32 keys       V of tile t + 1 is converted; K of tile t + 3 and V of tile t + 2 are asked for
//
// A turn has one form, for whole tiles and others: with a second one the compiler runs out of registers, and one with reloads from memory takes seven times as long.
//
// Bound by the wavefront's instructions, 440 besides 64 products a turn; the matrix cores are busy for 45 % of it, 36 % of the kernel.  512 tokens behind 8191 keys, 32 heads on 8: 93.7 us, of which the
// join takes 10 (760 TFLOP/s; tiles of 128 106 us, the cache in 16 bits 87); behind 32768 290 us (960 TFLOP/s; 337 and 258).
#include <cmath>
#include "attn_rowtile.h"
#include "paged_q8.h"

namespace {

using namespace rowtile;

constexpr int D = 128, KS = D / 16, DT = D / 32, KEYS = PAGED_CHUNK_KEYS, WAVES = 4, HALVES = 2, BLOCK_ROWS = PAGED_WIDE_ROWS, SLOTS = 4, TILE = KEYS * D;
static_assert(KEYS == ROWS && BLOCK_ROWS == 32 * HALVES * WAVES, "a tile of keys, 64 rows a wavefront");
constexpr float SLACK = 8.f;   // in powers of two: as in paged_attn_chunk.hip
constexpr int SMEM = 2 * SLOTS * TILE * (int)sizeof(bf16);
#define FENCE() __builtin_amdgcn_sched_barrier(0)   // the compiler's order of instructions ends here
#define INLINE __attribute__((always_inline))

typedef const u32x4 __attribute__((address_space(1))) * global_row;
typedef const uint8_t __attribute__((address_space(1))) * global_byte;
typedef u32x4 __attribute__((address_space(3))) * lds_row;

// (as assembly: results of score_onto would first be multiplied by 1 each, for all that the compiler knows of them)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(a), "v"(b), "v"(c));
  return m;
}
__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Products with the second operand in accumulation registers, where the queries wait; see mfma32_new and mfma32_onto of attn_tile.h
__device__ __forceinline__ void score_new(f32x16& d, bf16x8 a, bf16x8 b) { asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(d) : "v"(a), "a"(b)); }
__device__ __forceinline__ void score_onto(f32x16& d, bf16x8 a, bf16x8 b) { asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "a"(b)); }


__global__ __launch_bounds__(64 * WAVES, 1) void paged_wide_q8_kernel(const PagedAttnParams p, const PagedCache cache, const PagedScales z) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const unsigned k_places = (unsigned)(uintptr_t)(lds_ptr)smem, v_places = k_places + SLOTS * TILE * 2;   // LDS addresses of [SLOTS][KEYS][D]

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 5, i = lane & 31;
  PagedWalk<KEYS> walk(p, cache, lane);
  const int each = walk.total();   // steps of a kv head
  const PagedCuts cuts(each * p.Hkv, paged_blocks(p, each * p.Hkv, gridDim.x));
  const int block = paged_range(blockIdx.x, cuts.blocks);
  if (block >= cuts.blocks) return;
  const int begin = cuts.at(block), end = cuts.at(block + 1);
  int pos = begin;
  PagedPlace<KEYS> at(walk, pos, each);
  // Of this lane in a load of eight rows: in the cache; in LDS, row and first chunk, of which the other one is 16 bytes to either side.  16 lanes in a row have rows 4 apart, whose swz
  // differ in bit 0: they write to 16 different 16 bytes of 256.
  const int lrow = lane >> 4 | (lane >> 3 & 1) << 2;
  const unsigned lk = lrow * cache.k_row + 16 * (lane & 7), lv = lrow * cache.v_row + 16 * (lane & 7);
  const unsigned put = (8 * wave + lrow) * (2 * D) + 16 * ((2 * (lane & 7)) ^ swz<D>(8 * wave + lrow));
  const float c2 = p.scale_log2e;
  unsigned krow, vtr[KS];   // of fragments, in the slots in turn; of K of columns 16 n on at krow ^ 32 n
  {
    Readers<D> rd;
    rd.init(reinterpret_cast<const bf16*>(smem), g, i);
#pragma unroll
    for (int n = 0; n < KS; n++) vtr[n] = rd.tr[n] + SLOTS * TILE * 2;
    krow = rd.row[0];
  }
  auto step_of = [](int from, int to) { return (unsigned)((to & (SLOTS - 1)) - (from & (SLOTS - 1))) * (TILE * 2); };
  auto k_to_slot = [&](int from, int to) INLINE { krow += step_of(from, to); };
  auto v_to_slot = [&](int from, int to) INLINE {
#pragma unroll
    for (int n = 0; n < KS; n++) vtr[n] += step_of(from, to);
  };

  while (pos < end) {
    const int s = at.s, rt = at.rt, hk = at.hk, length = at.length, row0 = rt * BLOCK_ROWS;
    const int span = min(at.steps - at.step, end - pos), step = max(0, at.step - PAGED_EXTRA), steps_here = at.step + span - PAGED_EXTRA - step;
    const bool whole = step == 0 && at.step + span == at.steps;
    if (steps_here <= 0) break;   // the range ends with what a unit costs besides its steps
    const int rows = min(BLOCK_ROWS, p.n * p.group - row0);
    const int none = p.n - at.fresh;   // the first tokens, which are none
    const int keys = paged_keys(p, cache, length, at.fresh, rt), tiles = keys > 0 ? steps_here : 0;
    const int key0 = KEYS * step, last = max(tiles - 1, 0);
    const uint8_t *kp = static_cast<const uint8_t*>(cache.k) + hk * cache.sk.h, *vp = static_cast<const uint8_t*>(cache.v) + hk * cache.sv.h;
    const uint8_t *kz = z.k + hk * z.sk.h, *vz = z.v + hk * z.sv.h;
    const int* table = cache.table + s * cache.table_stride;

    // this lane's row of each half: token, query head
    struct Row { int token, head; };
    auto row_of = [&](int qt) {
      const int r = row0 + min(64 * wave + 32 * qt + i, rows - 1), token = r / p.group;
      return Row{token, hk * p.group + r - token * p.group};
    };
    f32x16 o[HALVES][DT];
#pragma unroll
    for (int qt = 0; qt < HALVES; qt++) clear(o[qt]);
    float ref[HALVES] = {-INFINITY, -INFINITY}, minus[HALVES] = {0.f, 0.f}, alpha[HALVES] = {1.f, 1.f}, l4[HALVES][4] = {};
    bool pending = false;   // O is to be rescaled by alpha

    if (tiles > 0) {
      const int first_token = (row0 + min(64 * wave, rows - 1)) / p.group;
      const int safe = __builtin_amdgcn_readfirstlane(first_token < none ? -1 : min(keys - 1, length - p.n + first_token));   // last key that all rows see

      int lim[HALVES];   // last key that the row sees

      // ---- lane n % 8 holds the page of a tile's n-th group of 8 keys
      const int in_page = (1 << cache.shift) - 1;
      auto lookup = [&](int t) INLINE { return table[min(key0 + KEYS * t + 8 * (lane & 7), keys - 1) >> cache.shift]; };
      auto with_page = [&](int pages) INLINE { return (unsigned)__builtin_amdgcn_ballot_w64((unsigned)pages < (unsigned)cache.pages) & 0xff; };
      // A wavefront's groups wave and wave + 4 of a tile, 16 bytes a lane, and their scales.  Rows behind the last key lie in its page; without a page they are page 0's.
      struct Part {
        u32x4 x[2];
        unsigned scale[2];
      };
      auto ask = [&](Part& a, int j, int t, int pages, const uint8_t* base, unsigned of_page, unsigned of_row, unsigned of_lane, const uint8_t* scales, const PageStrides& sz) INLINE {
        const int row = (key0 + KEYS * t + 8 * (wave + 4 * j)) & in_page;
        unsigned page = __builtin_amdgcn_readlane(pages, wave + 4 * j);
        page = page < (unsigned)cache.pages ? page : 0;
        asm("" : "+v"(of_lane));   // (it stays one register)
        a.x[j] = *(global_row)(base + (uint64_t)page * of_page + (uint64_t)((unsigned)row * of_row) + of_lane);
        a.scale[j] = *(global_byte)(scales + (int64_t)page * sz.p + (row >> z.shift) * sz.r);
      };
      auto ask_k = [&](Part& a, int j, int t, int pages) INLINE { ask(a, j, t, pages, kp, cache.k_page, cache.k_row, lk, kz, z.sk); };
      auto ask_v = [&](Part& a, int j, int t, int pages) INLINE { ask(a, j, t, pages, vp, cache.v_page, cache.v_row, lv, vz, z.sv); };
      // what is not there is 0
      auto only_there = [&](Part& a, int t, unsigned have) INLINE {
        if (have == 0xff && key0 + KEYS * (t + 1) <= keys) return;
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const int left = (have >> (wave + 4 * j) & 1) ? keys - (key0 + KEYS * t + 8 * (wave + 4 * j)) : 0;   // keys from the group's first on
          if (lrow >= left) a.x[j] = u32x4{0, 0, 0, 0}, a.scale[j] = 127;
        }
      };
      // eight values of each lane to LDS, item 0 .. 3: group item / 2, half item % 2
      auto convert = [&](const Part& a, int item, int t, unsigned place) INLINE {
        const int j = item >> 1, h = item & 1;
        *(lds_row)(uintptr_t)((put ^ 16 * h) + place + (t & (SLOTS - 1)) * (TILE * 2) + j * (32 * 2 * D)) =
            __builtin_bit_cast(u32x4, q8_operand(a.x[j][2 * h], a.x[j][2 * h + 1], q8_scale(a.scale[j])));
      };
      Part rk, rv;                        // on their way: of K of tile t + 2 and V of tile t + 1, in turn t
      int p2 = 0, p3 = 0;                 // pages of tiles t + 2 and t + 3
      unsigned have0 = 0, h1 = 0, h2 = 0;   // groups that have a page: of tile 0, of tiles t + 1 and t + 2

      // ---- the rows' queries beside the first pages; K of tiles 0 and 1, V of tile 0
      bf16x8 qf[HALVES][KS];
      {
        const int pages0 = lookup(0), pages1 = lookup(1);
        p2 = lookup(2), p3 = lookup(3);
#pragma unroll
        for (int qt = 0; qt < HALVES; qt++) {
          const Row r = row_of(qt);
          lim[qt] = r.token < none ? -1 : min(keys - 1, length - p.n + r.token);
          const bf16* qp = static_cast<const bf16*>(p.q) + s * p.sq.b + r.token * p.sq.l + r.head * p.sq.h + 8 * g;
#pragma unroll
          for (int ks = 0; ks < KS; ks++) qf[qt][ks] = *reinterpret_cast<const bf16x8*>(qp + 16 * ks);
        }
#pragma unroll
        for (int j = 0; j < 2; j++) ask_k(rk, j, 0, pages0), ask_v(rv, j, 0, pages0);
        have0 = with_page(pages0), h1 = with_page(pages1), h2 = with_page(p2);
#pragma unroll
        for (int qt = 0; qt < HALVES; qt++)
#pragma unroll
          for (int ks = 0; ks < KS; ks++) {
            qf[qt][ks] = p.signed_query(qf[qt][ks]);
            asm volatile("" : "+a"(qf[qt][ks]));   // in one piece, and there
          }
        only_there(rk, 0, have0), only_there(rv, 0, have0);
#pragma unroll
        for (int item = 0; item < 4; item++) convert(rk, item, 0, k_places), convert(rv, item, 0, v_places);
#pragma unroll
        for (int j = 0; j < 2; j++) ask_k(rk, j, 1, pages1), ask_v(rv, j, 1, pages1);
        only_there(rk, 1, h1);
#pragma unroll
        for (int item = 0; item < 4; item++) convert(rk, item, 1, k_places);
#pragma unroll
        for (int j = 0; j < 2; j++) ask_k(rk, j, 2, p2);
        FENCE();
      }
      f32x16 y[2][HALVES];        // scores of half tile 0 / 1
      bf16x8 pb[2][HALVES][2];    // P of a half tile
      float ex = 0.f, x1 = 0.f, x2 = 0.f;   // the exponent of the element due; the two elements before it
      // element e = 0 .. 31 of half tile kt: rows qt = e / 16, accumulator register e % 16
      auto exponent = [&](int kt, int e) INLINE { return fmaf(y[kt][e >> 4][e & 15], c2, minus[e >> 4]); };
      auto take = [&](int kt, int e) INLINE {
        const int qt = e >> 4, r = e & 15;
        l4[qt][r & 3] += x1;
        asm volatile("" : "+v"(l4[qt][r & 3]));
        if (r & 1) pb[kt][qt][r >> 3][(r & 7) - 1] = (bf16)x2, pb[kt][qt][r >> 3][r & 7] = (bf16)x1;
        if ((r & 7) == 7) asm volatile("" : "+v"(pb[kt][qt][r >> 3]));
      };
      auto weight = [&](int kt, int e) INLINE {
        float x = ody_exp2(ex);
        asm volatile("" : "+v"(x));   // (empty assembly keeps these where they stand: the compiler would move them behind the branches, to where they are used)
        if (e < 31) ex = exponent(kt, e + 1);
        if (e > 0) take(kt, e - 1);
        x2 = x1, x1 = x;
        if (e == 31) take(kt, e);
      };
      float top[HALVES];    // a row's largest score of the half tile at hand, in powers of two
      bool above = false;   // one of them is too far above its reference
      auto rescale = [&]() INLINE {
        if (pending) {
#pragma unroll
          for (int qt = 0; qt < HALVES; qt++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
              for (int r = 0; r < 16; r++) o[qt][dt][r] *= alpha[qt];
          pending = false;
        }
      };
      auto largest = [&](int kt, int qt) INLINE {
        float m = y[kt][qt][0];
#pragma unroll
        for (int r = 1; r < 15; r += 2) m = max3(m, y[kt][qt][r], y[kt][qt][r + 1]);
        return half_swap_max(max3(m, m, y[kt][qt][15])) * c2;
      };
      // the scores of half tile kt, keys n0 .., are complete, top and above are theirs
      auto decide = [&](int kt, int n0, unsigned ok) INLINE {
        rescale();
        if (n0 + KEYS / 2 - 1 > safe || ok != 15) {
#pragma unroll
          for (int qt = 0; qt < HALVES; qt++) {
#pragma unroll
            for (int r = 0; r < 16; r++)
              if (n0 + acc_row(r, g) > lim[qt] || (ok >> (r >> 2) & 1) == 0) y[kt][qt][r] = -INFINITY;
            top[qt] = largest(kt, qt);
          }
          above = top[0] > ref[0] + SLACK || top[1] > ref[1] + SLACK;
        }
        if (__builtin_amdgcn_ballot_w64(above) != 0) {
#pragma unroll
          for (int qt = 0; qt < HALVES; qt++) {
            const float now = fmaxf(ref[qt], top[qt]);
            alpha[qt] = now == -INFINITY ? 1.f : ody_exp2(ref[qt] - now);
            ref[qt] = now, minus[qt] = now == -INFINITY ? 0.f : -now;
#pragma unroll
            for (int e = 0; e < 4; e++) l4[qt][e] *= alpha[qt];
          }
          pending = true;
        }
        ex = exponent(kt, 0);
      };

      constexpr int PF = 8;   // a phase's fragments; each is loaded again, for the next phase, behind its products
      bf16x8 fr[PF];
      auto kfrag = [&](int kt, int n) INLINE {
        typedef const bf16x8 __attribute__((address_space(3))) * ptr;
        return *(ptr)(uintptr_t)((krow ^ 32 * n) + 2 * 32 * kt * D);
      };
      auto vfrag = [&](int kt, int n) INLINE {   // n = 4 * (16 keys) + (32 columns)
        typedef s16x4 __attribute__((address_space(3))) * ptr;
        const int dt = n & 3, first = 32 * kt + 16 * (n >> 2);
        return concat4(__builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(uintptr_t)(vtr[2 * dt] + 2 * first * D))),
                       __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(uintptr_t)(vtr[2 * dt + 1] + 2 * (first + 8) * D))));
      };
      // The reads that may be under way: those of a phase's second half, of fragments that are one read each (K) or two (V)
      constexpr int LGKM_4 = 0xc47f, LGKM_8 = 0xc87f;
      auto s_phase = [&](int kt, int of, int e0, auto under) INLINE {   // S of half tile kt; elements e0 .. of P of half tile `of`; what `under` has for the n-th pair of products
#pragma unroll
        for (int n = 0; n < 8; n++)
#pragma unroll
          for (int qt = 0; qt < HALVES; qt++) {
            if (n == 0 && qt == 0) __builtin_amdgcn_s_waitcnt(LGKM_4);
            if (n == 4 && qt == 0) __builtin_amdgcn_s_waitcnt(LGKM_8);
            if (n == 0) score_new(y[kt][qt], fr[n], qf[qt][n]);
            else score_onto(y[kt][qt], fr[n], qf[qt][n]);
            FENCE();
            if (qt == 0) under(n);
            if (qt == 1) fr[n] = vfrag(kt, n);
            weight(of, e0 + 2 * n + qt);
            FENCE();
          }
      };
      // O with half tile kt; ...; the largest scores of half tile kt (of the next tile), which s_phase formed
      auto pv_phase = [&](int kt, int of, int e0, auto under) INLINE {
#pragma unroll
        for (int n = 0; n < 8; n++)
#pragma unroll
          for (int qt = 0; qt < HALVES; qt++) {
            if (n == 0 && qt == 0) __builtin_amdgcn_s_waitcnt(LGKM_8);
            if (n == 4 && qt == 0) __builtin_amdgcn_s_waitcnt(LGKM_4);
            o[qt][n & 3] = mfma32(fr[n], pb[kt][qt][n >> 2], o[qt][n & 3]);
            FENCE();
            if (qt == 0) under(n);
            if (qt == 1) fr[n] = kfrag(kt ^ 1, n);
            weight(of, e0 + 2 * n + qt);
            if (n >= 2 && n < 6) {   // two registers of each half's scores (complete three products behind s_phase)
              const int r = 4 * (n - 2) + 2 * qt;
#pragma unroll
              for (int z = 0; z < HALVES; z++) top[z] = max3(r == 0 ? y[kt][z][0] : top[z], y[kt][z][r], y[kt][z][r + 1]);
            }
            if (n == 6) top[qt] = half_swap_max(top[qt]) * c2;
            if (n == 7 && qt == 0) above = top[0] > ref[0] + SLACK || top[1] > ref[1] + SLACK;
            FENCE();
          }
      };

      __syncthreads();
      // S of the first tile, P of its first half
#pragma unroll
      for (int kt = 0; kt < 2; kt++)
#pragma unroll
        for (int n = 0; n < 8; n++) {
          const bf16x8 f = kfrag(kt, n);
#pragma unroll
          for (int qt = 0; qt < HALVES; qt++)
            if (n == 0) score_new(y[kt][qt], f, qf[qt][n]);
            else score_onto(y[kt][qt], f, qf[qt][n]);
        }
      asm volatile("s_nop 15\n\ts_nop 7" : "+v"(y[0][0]), "+v"(y[0][1]), "+v"(y[1][0]), "+v"(y[1][1]));
#pragma unroll
      for (int qt = 0; qt < HALVES; qt++) top[qt] = largest(0, qt);
      above = top[0] > ref[0] + SLACK || top[1] > ref[1] + SLACK;
      decide(0, key0, have0 & 15);
#pragma unroll
      for (int e = 0; e < 32; e++) weight(0, e);
#pragma unroll
      for (int qt = 0; qt < HALVES; qt++) top[qt] = largest(1, qt);
      above = top[0] > ref[0] + SLACK || top[1] > ref[1] + SLACK;
      decide(1, key0 + 32, have0 >> 4);
      k_to_slot(0, 1);
#pragma unroll
      for (int n = 0; n < PF; n++) fr[n] = kfrag(0, n);   // (of a lone tile: of whatever lies there, not used)
      FENCE();

      for (int t = 0; t + 1 < tiles; t++) {
        const int n0 = key0 + KEYS * (t + 1);
        only_there(rk, t + 2, h2), only_there(rv, t + 1, h1);
        s_phase(0, 1, 0, [&](int n) INLINE {
          if (n & 1) convert(rk, n >> 1, t + 2, k_places);
        });
        pv_phase(0, 1, 16, [&](int n) INLINE {
          if (n < 4) convert(rv, n, t + 1, v_places);
          else if (n < 6) ask_k(rk, n - 4, t + 3, p3);
          else ask_v(rv, n - 6, t + 2, p2);
        });
        const unsigned ok = h1;
        decide(0, n0, ok & 15);
        // K of t + 2 and V of t + 1 are written (behind them four reads of fragments and more); everyone is done with K of t and V of t - 1
        __builtin_amdgcn_s_waitcnt(LGKM_4);
        barrier();
        s_phase(1, 0, 0, [](int) {});
        pv_phase(1, 0, 16, [&](int n) INLINE {
          if (n == 0) {
            k_to_slot(t + 1, t + 2);
            h1 = h2, h2 = with_page(p3), p2 = p3;
            p3 = lookup(t + 4);
          }
          if (n == 3) v_to_slot(t, t + 1);
        });
        decide(1, n0 + 32, ok >> 4);
      }
      // the last tile: P of its second half, the products
#pragma unroll
      for (int e = 0; e < 32; e++) weight(1, e);
#pragma unroll
      for (int kt = 0; kt < 2; kt++) {
#pragma unroll
        for (int n = 0; n < 8; n++) {
          const bf16x8 f = vfrag(kt, n);
#pragma unroll
          for (int qt = 0; qt < HALVES; qt++) o[qt][n & 3] = mfma32(f, pb[kt][qt][n >> 2], o[qt][n & 3]);
        }
        if (kt == 0) rescale();
      }
      k_to_slot(tiles, 0);
      v_to_slot(last, 0);
    }
    __syncthreads();   // everyone is done with the tiles

#pragma unroll
    for (int qt = 0; qt < HALVES; qt++) {
      const int row = 64 * wave + 32 * qt + i;
      const float sum = half_swap_sum((l4[qt][0] + l4[qt][1]) + (l4[qt][2] + l4[qt][3]));
      if (row >= rows) continue;
      const Row r = row_of(qt);
      if (whole) {
        store_row(static_cast<bf16*>(p.out) + s * p.so.b + r.token * p.so.l + r.head * p.so.h, o[qt], sum == 0.f ? 0.f : 1.f / sum, g);
        if (g == 0) p.lse[((int64_t)s * p.Hq + r.head) * p.n + r.token] = sum == 0.f ? -INFINITY : (ref[qt] + __log2f(sum)) * ODY_LN2;
      } else {
        const int64_t slot = (int64_t)(2 * block + (pos > begin)) * BLOCK_ROWS + row;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
          for (int a = 0; a < 4; a++)
            *reinterpret_cast<f32x4*>(p.part + slot * D + 32 * dt + 8 * a + 4 * g) =
                f32x4{o[qt][dt][4 * a], o[qt][dt][4 * a + 1], o[qt][dt][4 * a + 2], o[qt][dt][4 * a + 3]};
        if (g == 0) p.part_ml[slot] = make_float2(ref[qt], sum);
      }
    }
    pos += span;
    if (pos < end) at.next_unit(walk);
  }
}

}  // namespace

int ody_launch_paged_wide_q8(const PagedAttnParams& p, const PagedCache& c, const PagedScales& z, int blocks, hipStream_t st) {
  if (int rc = ody_allow_dynamic_lds(reinterpret_cast<const void*>(&paged_wide_q8_kernel), SMEM, "ody_paged_attn_q8")) return rc;
  ODY_LAUNCH("paged_wide_q8", st, paged_wide_q8_kernel, dim3(blocks), dim3(64 * WAVES), SMEM, p, c, z);
  return ody_check_launch("paged_wide_q8");
}
