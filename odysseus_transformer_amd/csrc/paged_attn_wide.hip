// Attention of long chunks over a key / value cache in pages, bf16, heads of 128: row tiles of 256, of which paged_attn_chunk.hip takes 128.
//
// The same two products, transposed, over the same tiles of 64 keys as there.  Here one block has a compute unit and a wavefront a SIMD with all of its registers:
// 64 rows each, as two halves that share every fragment read from LDS and every scalar instruction, of which the kernel of 128 rows has twice as many.  A
// turn of the loop forms O^T of tile t and S^T of tile t + 1 in four phases of 16 products, and under each product one element of P, of the half
// tile whose scores are complete and whose turn as an operand is next:
//
//      S^T(t + 1), first 32 keys      P(t), second 32 keys, rows 0 .. 31
//      O^T += P(t), first 32 keys     P(t), second 32 keys, rows 32 .. 63;  the largest of the scores just formed
//      S^T(t + 1), second 32 keys     P(t + 1), first 32 keys, rows 0 .. 31
//      O^T += P(t), second 32 keys    P(t + 1), first 32 keys, rows 32 .. 63;  the largest of the scores just formed
//
// Between a phase of O^T and the next one of S^T the half tile just formed is masked, where a row does not see all of it, and a row's reference follows its
// largest score where that is more than SLACK above (seldom).  P of the half tile before is in the old reference's scale then and not yet in O: the row sums
// are rescaled at once, O one half tile later.
//
// Measured against tiles of 128 rows, 32 heads on 8: 2048 tokens behind 8192 keys 354 -> 312 us (990 TFLOP/s; the kernel without a cache, attn_fwd_pipe.hip, 1 220 to
// 1 320), 512 behind 32768 301 -> 258 (1 060), 512 behind 8191 97 -> 87, of which the join takes 10.  The matrix cores are busy half of the time.  Of a turn's
// 4 090 cycles the loads cost 9 %, the exponentials 5, the LDS reads of K and of V 2 each, sums 3, maxima and the references 2 (left out in turn); nothing of it alone.
#include <cmath>
#include "attn_rowtile.h"
#include "paged.h"

namespace {

using namespace rowtile;

constexpr int D = 128, KS = D / 16, DT = D / 32, KEYS = PAGED_CHUNK_KEYS, WAVES = 4, HALVES = 2, BLOCK_ROWS = PAGED_WIDE_ROWS, SLOTS = 4, TILE = KEYS * D;
static_assert(KEYS == ROWS && BLOCK_ROWS == 32 * HALVES * WAVES, "a tile of keys, 64 rows a wavefront");
constexpr float SLACK = 8.f;   // in powers of two: as in paged_attn_chunk.hip
constexpr int PAGE_TILES = 8;  // tiles whose pages 64 lanes look up at once
constexpr int SMEM = 2 * SLOTS * TILE * (int)sizeof(bf16) + WAVES * 2 * 64 * (int)sizeof(int);
#define FENCE() __builtin_amdgcn_sched_barrier(0)   // the compiler's order of instructions ends here
#define INLINE __attribute__((always_inline))

__device__ const bf16x8 no_key[16] = {};   // the row that a key without a page, or behind the last one, is read from

// Direct loads, 16 bytes a lane or 4, to LDS address `to` on; as assembly without results: see paged_attn_chunk.hip
__device__ __forceinline__ void direct_load(const char* from, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}
__device__ __forceinline__ void direct_load(const char* from, unsigned of_lane, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(of_lane), "s"(from) : "memory");
}
__device__ __forceinline__ void direct_load_dword(const int* from, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(from) : "memory");
}
// (as assembly: results of score_onto would first be multiplied by 1 each, for all that the compiler knows of them)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(a), "v"(b), "v"(c));
  return m;
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Products with the second operand in accumulation registers, where the queries wait; see mfma32_new and mfma32_onto of attn_tile.h
__device__ __forceinline__ void score_new(f32x16& d, bf16x8 a, bf16x8 b) { asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(d) : "v"(a), "a"(b)); }
__device__ __forceinline__ void score_onto(f32x16& d, bf16x8 a, bf16x8 b) { asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "a"(b)); }

// SPREAD: a tile's keys lie in several pages, of 8 keys and more, and a load's address is formed for it; else a tile's is formed once (2048 tokens behind 8192 keys 346
// us against 337 on one card).
template <bool SPREAD>
__global__ __launch_bounds__(64 * WAVES, 1) void paged_wide_kernel(const PagedAttnParams p, const PagedCache cache) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const unsigned k_places = (unsigned)(uintptr_t)(lds_ptr)smem, v_places = k_places + SLOTS * TILE * 2;   // LDS addresses of [SLOTS][KEYS][D]

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 5, i = lane & 31;
  const unsigned page_place = k_places + 2 * SLOTS * TILE * 2 + wave * 512;   // [2][64]: this wavefront's page numbers of 8 tiles each
  PagedWalk<KEYS> walk(p, cache, lane);
  const int each = walk.total();   // steps of a kv head
  const PagedCuts cuts(each * p.Hkv, paged_blocks(p, each * p.Hkv, gridDim.x));
  const int block = paged_range(blockIdx.x, cuts.blocks);
  if (block >= cuts.blocks) return;
  const int begin = cuts.at(block), end = cuts.at(block + 1);
  int pos = begin;
  PagedPlace<KEYS> at(walk, pos, each);
  const int lrow = 4 * wave + (lane >> 4), lcol = 8 * ((lane & 15) ^ swz<D>(lrow));   // of this lane in its first direct load of a tile; 16 rows from one to the next
  const float c2 = p.scale_log2e;
  unsigned krow[KS], vtr[KS];   // of fragments, in the slots in turn
  {
    Readers<D> rd;
    rd.init(reinterpret_cast<const bf16*>(smem), g, i);
#pragma unroll
    for (int n = 0; n < KS; n++) krow[n] = rd.row[n], vtr[n] = rd.tr[n] + SLOTS * TILE * 2;
  }
  auto to_slot = [&](unsigned (&a)[KS], int from, int to) INLINE {
    const unsigned by = ((to & (SLOTS - 1)) - (from & (SLOTS - 1))) * (TILE * 2);
#pragma unroll
    for (int n = 0; n < KS; n++) a[n] += by;
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
    const char* kp = reinterpret_cast<const char*>(static_cast<const bf16*>(cache.k) + hk * cache.sk.h);
    const char* vp = reinterpret_cast<const char*>(static_cast<const bf16*>(cache.v) + hk * cache.sv.h);
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

      // ---- loads: pages of 64 groups of 8 keys at a time, those of a tile in lanes n % 8; a tile in four instructions a wavefront
      auto entry = [&](int b) { return table + (min(key0 + 8 * (64 * b + lane), keys - 1) >> cache.shift); };
      const int in_page = (1 << cache.shift) - 1;
      const unsigned lk = (unsigned)lrow * cache.k_row + 2 * lcol, lv = (unsigned)lrow * cache.v_row + 2 * lcol;
      struct Source {   // of a tile's rows
        int first, pages;   // first key; lane n % 8: page of its n-th group
        unsigned have;      // groups that have one
        bool whole;         // all of its keys are there and in one page, which begins at
        const char* from;
      };
      auto source = [&](int t, int pages, const char* base, unsigned of_page, unsigned of_row) INLINE {
        Source x;
        x.first = key0 + KEYS * t, x.pages = pages;
        x.have = (unsigned)__builtin_amdgcn_ballot_w64((unsigned)pages < (unsigned)cache.pages) & 0xff;
        x.whole = x.have == 0xff && x.first + KEYS <= keys;
        x.from = base + (uint64_t)(unsigned)__builtin_amdgcn_readlane(pages, 0) * of_page + (uint64_t)(unsigned)(x.first & in_page) * of_row;
        return x;
      };
      auto load = [&](auto plain, const Source& x, int j, const char* base, unsigned of_page, unsigned of_row, unsigned of_lane, unsigned place) INLINE {
        const unsigned to = place + (WAVES * j + wave) * 1024;
        const int row = 16 * j + 4 * wave, group = row / 8, first = x.first + row, page = __builtin_amdgcn_readlane(x.pages, group);
        if (decltype(plain)::value && SPREAD) {
          direct_load(base + (uint64_t)(unsigned)page * of_page + (uint64_t)((unsigned)(first & in_page) * of_row), of_lane - 4 * wave * of_row, to);
        } else if (decltype(plain)::value) {
          direct_load(x.from, of_lane + 16 * j * of_row, to);
        } else {
          const char* src = base + (uint64_t)(unsigned)page * of_page + (uint64_t)(unsigned)(first & in_page) * of_row + (of_lane - 4 * wave * of_row);
          const bool zero = first + (lane >> 4) >= keys || (x.have >> group & 1) == 0;
          direct_load(zero ? reinterpret_cast<const char*>(no_key) + 2 * lcol : src, to);
        }
      };
      std::true_type yes;
      std::false_type no;
      int tk = 0, tv = 0;   // the tiles being brought; the last one again where there are no more
      Source sk, sv;
      unsigned have0 = 0, have[2] = {};   // of tile 0; of the tiles before sk's: of t + 1 and t + 2 in turn t
      auto load_k = [&](auto plain, int j) INLINE { load(plain, sk, j, kp, cache.k_page, cache.k_row, lk, k_places + (tk & (SLOTS - 1)) * (TILE * 2)); };
      auto load_v = [&](auto plain, int j) INLINE { load(plain, sv, j, vp, cache.v_page, cache.v_row, lv, v_places + (tv & (SLOTS - 1)) * (TILE * 2)); };
      // pages of a tile from this wavefront's numbers in LDS
      auto pages_of = [&](int t) INLINE {
        typedef const int __attribute__((address_space(3))) * ptr;
        return *(volatile ptr)(uintptr_t)(page_place + (t / PAGE_TILES & 1) * 256 + (t % PAGE_TILES * 8 + (lane & 7)) * 4);
      };

      // ---- the rows' queries beside the first pages; then K of tiles 0 .. 2, V of 0 and 1, and a quarter each of the next ones, which the loop goes on with
      bf16x8 qf[HALVES][KS];
      {
        const int pages0 = *entry(0);
#pragma unroll
        for (int qt = 0; qt < HALVES; qt++) {
          const Row r = row_of(qt);
          lim[qt] = r.token < none ? -1 : min(keys - 1, length - p.n + r.token);
          const bf16* qp = static_cast<const bf16*>(p.q) + s * p.sq.b + r.token * p.sq.l + r.head * p.sq.h + 8 * g;
#pragma unroll
          for (int ks = 0; ks < KS; ks++) qf[qt][ks] = *reinterpret_cast<const bf16x8*>(qp + 16 * ks);
        }
#pragma unroll
        for (int qt = 0; qt < HALVES; qt++)
#pragma unroll
          for (int ks = 0; ks < KS; ks++) {
            qf[qt][ks] = p.signed_query(qf[qt][ks]);
            asm volatile("" : "+a"(qf[qt][ks]));   // in one piece, and here: in front of the direct loads, whose number the waits below go by
          }
        FENCE();
        direct_load_dword(entry(0), page_place);
        direct_load_dword(entry(1), page_place + 256);
        auto of_tile = [&](int t) INLINE { return __shfl(pages0, 8 * t + (lane & 7)); };
#pragma unroll
        for (int a = 0; a < 4; a++) {
          tk = min(a, last);
          sk = source(tk, of_tile(tk), kp, cache.k_page, cache.k_row);
          if (a == 0) have0 = sk.have;
          else if (a < 3) have[a - 1] = sk.have;
#pragma unroll
          for (int j = 0; j < (a < 3 ? 4 : 1); j++) load_k(no, j);
          if (a > 0) {
            tv = min(a - 1, last);
            sv = source(tv, of_tile(tv), vp, cache.v_page, cache.v_row);
#pragma unroll
            for (int j = 0; j < (a < 3 ? 4 : 1); j++) load_v(no, j);
          }
        }
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
      auto decide = [&](auto plain, int kt, int n0, unsigned ok) INLINE {
        rescale();
        if (!decltype(plain)::value) if (n0 + KEYS / 2 - 1 > safe || ok != 15) {
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
        return *(ptr)(uintptr_t)(krow[n] + 2 * 32 * kt * D);
      };
      auto vfrag = [&](int kt, int n) INLINE {   // n = 4 * (16 keys) + (32 columns)
        typedef s16x4 __attribute__((address_space(3))) * ptr;
        const int dt = n & 3, first = 32 * kt + 16 * (n >> 2);
        return concat4(__builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(uintptr_t)(vtr[2 * dt] + 2 * first * D))),
                       __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(uintptr_t)(vtr[2 * dt + 1] + 2 * (first + 8) * D))));
      };
      // The reads that may be under way: those of a phase's second half, of fragments that are one read each (K) or two (V)
      constexpr int LGKM_4 = 0xc47f, LGKM_8 = 0xc87f;
      auto s_phase = [&](int kt, int of, int e0) INLINE {   // S of half tile kt; elements e0 .. of P of half tile `of`
#pragma unroll
        for (int n = 0; n < 8; n++)
#pragma unroll
          for (int qt = 0; qt < HALVES; qt++) {
            if (n == 0 && qt == 0) __builtin_amdgcn_s_waitcnt(LGKM_4);
            if (n == 4 && qt == 0) __builtin_amdgcn_s_waitcnt(LGKM_8);
            if (n == 0) score_new(y[kt][qt], fr[n], qf[qt][n]);
            else score_onto(y[kt][qt], fr[n], qf[qt][n]);
            FENCE();
            if (qt == 1) fr[n] = vfrag(kt, n);
            weight(of, e0 + 2 * n + qt);
            FENCE();
          }
      };
      // O with half tile kt; ...; the largest scores of half tile kt (of the next tile), which s_phase formed; what `under` has for the n-th pair of products.  The
      // direct loads go out here, where half as many LDS reads do: three quarters of a tile's with half tile 0, the first of the next one's with half tile 1
      // (pages of 16: 343 -> 328 us than with one in each phase, 512 tokens behind 32488 keys 267 -> 258).
      auto pv_phase = [&](auto plain, int kt, int of, int e0, auto under) INLINE {
#pragma unroll
        for (int n = 0; n < 8; n++)
#pragma unroll
          for (int qt = 0; qt < HALVES; qt++) {
            if (n == 0 && qt == 0) __builtin_amdgcn_s_waitcnt(LGKM_8);
            if (n == 4 && qt == 0) __builtin_amdgcn_s_waitcnt(LGKM_4);
            o[qt][n & 3] = mfma32(fr[n], pb[kt][qt][n >> 2], o[qt][n & 3]);
            FENCE();
            if (qt == 0) under(n);
            if (qt == 0 && kt == 0 && n >= 1 && n <= 3) load_k(plain, n);
            if (qt == 0 && kt == 0 && n >= 4 && n <= 6) load_v(plain, n - 3);
            if (qt == 0 && kt == 1 && n == 2) load_k(plain, 0);
            if (qt == 0 && kt == 1 && n == 5) load_v(plain, 0);
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

      wait_loads<18>();   // for K of tile 0
      barrier();
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
      decide(no, 0, key0, have0 & 15);
#pragma unroll
      for (int e = 0; e < 32; e++) weight(0, e);
#pragma unroll
      for (int qt = 0; qt < HALVES; qt++) top[qt] = largest(1, qt);
      above = top[0] > ref[0] + SLACK || top[1] > ref[1] + SLACK;
      decide(no, 1, key0 + 32, have0 >> 4);
      to_slot(krow, 0, 1);
      wait_loads<10>();   // for V of tile 0 and K of tile 1
      barrier();
#pragma unroll
      for (int n = 0; n < PF; n++) fr[n] = kfrag(0, n);   // (of a lone tile: of whatever lies there, not used)
      FENCE();

      int pages = pages_of(min(4, last));   // of tile t + 4
      auto all_there = [&](int pages) INLINE { return ((unsigned)__builtin_amdgcn_ballot_w64((unsigned)pages < (unsigned)cache.pages) & 0xff) == 0xff; };
      bool next_there = all_there(pages);
      // turn t.  PLAIN: all rows see all of tile t + 1, and tiles t + 2 .. t + 4 are whole
      auto turn = [&](auto plain, int t) INLINE {
        const int n0 = key0 + KEYS * (t + 1);
        s_phase(0, 1, 0);
        pv_phase(plain, 0, 1, 16, [](int) {});
        decide(plain, 0, n0, have[0] & 15);
        // K of t + 2 and V of t + 1 have landed (behind them the 8 loads of the tiles after); everyone is done with K of t and V of t - 1
        wait_loads<8>();
        barrier();
        s_phase(1, 0, 0);
        if ((t & (PAGE_TILES - 1)) == PAGE_TILES - 2) direct_load_dword(entry(t / PAGE_TILES + 2), page_place + (t / PAGE_TILES & 1) * 256);
        const unsigned ok = have[0] >> 4;
        pv_phase(plain, 1, 0, 16, [&](int n) INLINE {
          if (n == 0) {
            to_slot(krow, t + 1, t + 2);
            const int before = sk.pages;
            have[0] = have[1], have[1] = sk.have;
            tv = tk, tk = min(t + 4, last);
            sk = source(tk, pages, kp, cache.k_page, cache.k_row);
            sv = source(tv, before, vp, cache.v_page, cache.v_row);
            pages = pages_of(min(t + 5, last));
          }
          if (n == 3) to_slot(vtr, t, t + 1);
          if (n == 6) next_there = all_there(pages);
        });
        decide(plain, 1, n0 + 32, ok);
      };
      int t = 0;
      const int seen = safe < key0 ? 0 : (safe + 1 - key0) / KEYS;   // tiles that all rows see all of
      auto is_plain = [&](int t) INLINE {
        return t + 4 < min(tiles, seen) && sk.whole && sv.whole && have[0] == 0xff && next_there;
      };
      for (; is_plain(t); t++) turn(yes, t);
      for (; t + 1 < tiles; t++) turn(no, t);
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
      to_slot(krow, tiles, 0);
      to_slot(vtr, last, 0);
      wait_loads<0>();
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

template <bool SPREAD>
int launch(const PagedAttnParams& p, const PagedCache& c, int blocks, hipStream_t st) {
  if (int rc = ody_allow_dynamic_lds(reinterpret_cast<const void*>(&paged_wide_kernel<SPREAD>), SMEM, "ody_paged_attn")) return rc;
  ODY_LAUNCH("paged_wide", st, paged_wide_kernel<SPREAD>, dim3(blocks), dim3(64 * WAVES), SMEM, p, c);
  return ody_check_launch("paged_wide");
}

}  // namespace

int ody_launch_paged_wide(const PagedAttnParams& p, const PagedCache& c, int blocks, hipStream_t st) {
  return 1 << c.shift >= KEYS ? launch<false>(p, c, blocks, st) : launch<true>(p, c, blocks, st);
}
