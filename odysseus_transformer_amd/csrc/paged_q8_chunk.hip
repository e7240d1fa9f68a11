// Attention of many new tokens over a key / value cache in pages that holds its values in 8 bits, bf16 queries: a chunk of a prompt, or many rows of a kv head; the
// rule is in paged_q8_attn.hip.
//
// Bound by the vector work of the softmax and the matrix cores, as paged_attn_chunk.hip, whose halves these are: a block of four wavefronts takes 128 rows, 32 a
// wavefront, over tiles of 64 keys; S of the next half tile is formed under the softmax of the present one.  Tiles lie in LDS as the cache has them, half as large as there:
// direct loads bring them two turns ahead into four places, and a turn has one barrier.
//
//      S^T = K Q^T        A: K rows, 16 bytes a lane for two products, converted in registers    B: this lane's query row, in the same order of columns
//      O^T += V^T P^T     A: V^T by transposing reads of 8 bits, converted in registers         B: P^T as the accumulators of S^T hold it
//
// on v_mfma_f32_32x32x16_bf16.  The conversions are exact and apply a block's power of two for nothing.  (The product of e4m3 values with scales of their own,
// v_mfma_scale_f32_32x32x64_f8f6f4, would take K as it is and a query as the sum of two such rows, which is exact; but its sums of 64 come out 2^-18.7 of the sum of
// their sizes off, root mean square, where this one's are at 2^-27: for rows of unit size less than the 2^-8 by which P is rounded, but all of what lse is off by.  Not taken up.)
//
// Each of a block's wavefronts converts all of a tile, half of the vector work: 512 tokens behind 8191 keys, 32 heads on 8 of 128, 106 us (670 TFLOP/s; paged_q8_wide.hip, which converts a value once, 94);
// heads of 64 65 us; 128 tokens 43.
// Of heads of 128, 47 registers go to memory: the loop of plain turns has two accesses a turn, whose wait is one for the direct loads before them too, the other one twelve.
//
// P is rounded to bf16 for its product and summed up in fp32 unrounded, as in the attention over contiguous keys.
#include <cmath>
#include <type_traits>
#include "attn_rowtile.h"
#include "paged_q8.h"

namespace {

using namespace rowtile;

constexpr int KEYS = PAGED_CHUNK_KEYS, BLOCK_ROWS = PAGED_CHUNK_ROWS, WAVES = 4, SLOTS = 4;
static_assert(KEYS == ROWS && BLOCK_ROWS == 32 * WAVES, "a tile of keys, 32 rows a wavefront");
// How far, in powers of two, a score may be above its row's reference before the reference follows: P is up to 2^8 then, as exact in bf16 as below 1,
// and sums of 2^31 of them are far from what fp32 holds.
constexpr float SLACK = 8.f;
#define FENCE() __builtin_amdgcn_sched_barrier(0)   // the compiler's order of instructions ends here

__device__ const u32x4 no_key[8] = {};   // the row that a key without a page, or behind the last one, is read from

// A direct load, 16 bytes a lane, to LDS address `to` on.  As assembly, for behind the builtin the compiler makes transposing reads wait for it.  It has no result that the
// compiler could use too early, and nothing else in these kernels uses m0.
__device__ __forceinline__ void direct_load(const uint8_t* from, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}
__device__ __forceinline__ void barrier() {   // ... behind which all that was loaded by then has landed
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A row of a tile is D / 16 chunks of 16 bytes; chunk c of row r sits at position c ^ swizzle(r).  The 16 rows of a 16-byte read, and the eight rows of two chunks in a row that half a
// wavefront's transposing read takes (bit 2 of r fixed), lie in 16 different 16 bytes of 256.
template <int D> __device__ __forceinline__ int swizzle(int r) {
  if constexpr (D == 128) return ((r & 8) >> 1) | (r & 2) | ((r & 4) >> 2);
  else return ((r & 8) >> 2) | ((r & 4) >> 2);
}

template <int D>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_chunk_q8_kernel(const PagedAttnParams p, const PagedCache cache, const PagedScales z) {
  constexpr int KM = D / 32, DT = D / 32, TILE = KEYS * D;                  // pairs of products of S over D; tiles of O; bytes of a tile
  constexpr int LANES = D / 16, PER = 64 / LANES, LOADS = KEYS / PER / WAVES;   // of a direct load: lanes on a row, rows; of a tile and wavefront
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const unsigned places = (unsigned)(uintptr_t)(lds_ptr)smem;   // LDS address of [K | V][SLOTS][KEYS][D]

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 5, i = lane & 31;
  PagedWalk<KEYS> walk(p, cache, lane);
  const int each = walk.total();   // steps of a kv head
  const PagedCuts cuts(each * p.Hkv, paged_blocks(p, each * p.Hkv, gridDim.x));
  const int block = paged_range(blockIdx.x, cuts.blocks);
  if (block >= cuts.blocks) return;
  const int begin = cuts.at(block), end = cuts.at(block + 1);
  int pos = begin;
  PagedPlace<KEYS> at(walk, pos, each);
  const float c2 = p.scale_log2e;
  // where a lane reads, in slot 0 at the start of a unit: K rows i, chunk 2 m + g; V rows 4 g + .., columns 32 dt ..
  unsigned krow[KM], vtr[DT];
  {
    const int e = (lane & 15) >> 1, rr = e < 4 ? 4 * g + e : 4 + 4 * g + e, c = (lane >> 4) & 1;
#pragma unroll
    for (int m = 0; m < KM; m++) krow[m] = places + i * D + 16 * ((2 * m + g) ^ swizzle<D>(i));
#pragma unroll
    for (int dt = 0; dt < DT; dt++) vtr[dt] = places + SLOTS * TILE + rr * D + 16 * ((2 * dt + c) ^ swizzle<D>(rr)) + 8 * (lane & 1);
  }
  int kslot = 0, vslot = 0;
  auto k_to = [&](int t) {
    const unsigned by = ((t & (SLOTS - 1)) - kslot) * TILE;
    kslot = t & (SLOTS - 1);
#pragma unroll
    for (int m = 0; m < KM; m++) krow[m] += by;
  };
  auto v_to = [&](int t) {
    const unsigned by = ((t & (SLOTS - 1)) - vslot) * TILE;
    vslot = t & (SLOTS - 1);
#pragma unroll
    for (int dt = 0; dt < DT; dt++) vtr[dt] += by;
  };

  while (pos < end) {
    const int s = at.s, rt = at.rt, hk = at.hk, length = at.length, row0 = rt * BLOCK_ROWS;
    const int span = min(at.steps - at.step, end - pos), step = max(0, at.step - PAGED_EXTRA), steps_here = at.step + span - PAGED_EXTRA - step;
    const bool whole = step == 0 && at.step + span == at.steps;
    if (steps_here <= 0) break;   // the range ends with what a unit costs besides its steps
    const int rows = min(BLOCK_ROWS, p.n * p.group - row0);
    const int none = p.n - at.fresh;   // the first tokens, which are none
    const int keys = paged_keys(p, cache, length, at.fresh, rt), tiles = keys > 0 ? steps_here : 0;
    const int key0 = KEYS * step;
    const uint8_t *kp = static_cast<const uint8_t*>(cache.k) + hk * cache.sk.h, *vp = static_cast<const uint8_t*>(cache.v) + hk * cache.sv.h;
    // of lane n % 16: the scales of K in lanes 0 .. 7, of V in lanes 8 .. 15
    const uint8_t* zp = lane & 8 ? z.v + hk * z.sv.h : z.k + hk * z.sk.h;
    const int64_t z_page = lane & 8 ? z.sv.p : z.sk.p, z_line = lane & 8 ? z.sv.r : z.sk.r;
    const int* table = cache.table + s * cache.table_stride;
    const int in_page = (1 << cache.shift) - 1;

    // ---- lane n % 8 holds the page of a tile's n-th group of 8 keys
    auto lookup = [&](int t) { return table[min(key0 + KEYS * t + 8 * (lane & 7), keys - 1) >> cache.shift]; };
    auto with_page = [&](int pages) { return (unsigned)__builtin_amdgcn_ballot_w64((unsigned)pages < (unsigned)cache.pages) & 0xff; };
    auto scales_of = [&](int t, int pages) {   // of group n % 8; of one without a key or a page 2^0
      const int key = key0 + KEYS * t + 8 * (lane & 7), row = min(key, keys - 1) & in_page;
      const bool there = key < keys && (unsigned)pages < (unsigned)cache.pages;
      const unsigned byte = zp[(there ? pages : 0) * z_page + (row >> z.shift) * z_line];
      return there ? byte : 127u;
    };
    auto load = [&](int t, int pages) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < LOADS; j++) {
        const int row = PER * (WAVES * j + wave) + lane / LANES, key = key0 + KEYS * t + row, page = __shfl(pages, row / 8);
        const unsigned col = 16 * ((lane % LANES) ^ swizzle<D>(row)), r = min(key, keys - 1) & in_page;
        const bool there = key < keys && (unsigned)page < (unsigned)cache.pages;
        const uint8_t* zero = reinterpret_cast<const uint8_t*>(no_key) + col;
        const uint8_t *ks = kp + (uint64_t)(unsigned)page * cache.k_page + (uint64_t)(r * cache.k_row) + col, *vs = vp + (uint64_t)(unsigned)page * cache.v_page + (uint64_t)(r * cache.v_row) + col;
        const unsigned to = places + (t & (SLOTS - 1)) * TILE + 1024 * (WAVES * j + wave);
        direct_load(there ? ks : zero, to);
        direct_load(there ? vs : zero, to + SLOTS * TILE);
      }
    };

    // ---- this lane's row: token ri, query head h; of columns 32 m + 16 g .. + 15 two operands
    const int r = row0 + min(32 * wave + i, rows - 1), ri = r / p.group, h = hk * p.group + r - ri * p.group;
    bf16x8 qf[2 * KM];
    int pages2 = 0;
    unsigned have = 0, have1 = 0, sc = 127, sc1 = 127, sc2 = 127;   // of tiles t, t + 1 (and t + 2): groups with a page, scales
    {
      const bf16* qp = static_cast<const bf16*>(p.q) + s * p.sq.b + ri * p.sq.l + h * p.sq.h + 16 * g;
#pragma unroll
      for (int m = 0; m < KM; m++) qf[2 * m] = *reinterpret_cast<const bf16x8*>(qp + 32 * m), qf[2 * m + 1] = *reinterpret_cast<const bf16x8*>(qp + 32 * m + 8);
      if (tiles > 0) {
        const int pages0 = lookup(0), pages1 = lookup(1);
        pages2 = lookup(2);
        have = with_page(pages0), have1 = with_page(pages1);
        load(0, pages0), load(1, pages1);
        sc = scales_of(0, pages0), sc1 = scales_of(1, pages1);
      }
#pragma unroll
      for (int m = 0; m < 2 * KM; m++) qf[m] = p.signed_query(qf[m]);
    }
    const int lim = ri < none ? -1 : min(keys - 1, length - p.n + ri);   // last key that it sees
    const int first_token = (row0 + min(32 * wave, rows - 1)) / p.group;
    const int safe = __builtin_amdgcn_readfirstlane(first_token < none ? -1 : min(keys - 1, length - p.n + first_token));   // ... that all of the wavefront's see

    f32x16 o[DT];
    clear(o);
    float ref = -INFINITY, l4[4] = {0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY;   // the row's largest score of the half to come, where that is plain
    auto largest = [&](const f32x16& y) {
      float m = y[0];
#pragma unroll
      for (int e = 1; e < 16; e++) m = fmaxf(m, y[e]);
      return half_swap_max(m) * c2;
    };
    auto kraw = [&](int m, int first) {   // row first + i, columns 32 m + 16 g ..
      typedef const u32x4 __attribute__((address_space(3))) * ptr;
      return *(ptr)(uintptr_t)(krow[m] + first * D);
    };
    auto vraw = [&](int first, int dt) {   // column 32 dt + i of rows first + 4 g .. + 3, first + 8 + 4 g .. + 3
      typedef i32x2 __attribute__((address_space(3))) * ptr;
      return __builtin_amdgcn_ds_read_tr8_b64_v2i32((ptr)(uintptr_t)(vtr[dt] + first * D));
    };
    // A half: the softmax of y, the scores against keys n0 .., of which PLAIN says that every row sees all; S of the next half (K rows from NEXT on of its tile, whose scales
    // are in `ksc`), into z; P V with the V rows from VROW on, whose groups' scales lanes VROW / 8 .. of `vsc` have.
    auto half = [&](auto plain, f32x16& y, f32x16& zz, int n0, unsigned ok, auto next_, unsigned ksc, auto vrow_, unsigned vsc) __attribute__((always_inline)) {
      constexpr bool PLAIN = decltype(plain)::value;
      constexpr int NEXT = decltype(next_)::value, VROW = decltype(vrow_)::value;
      if constexpr (!PLAIN) {
        if (n0 + KEYS / 2 - 1 > safe || ok != 15) {
#pragma unroll
          for (int e = 0; e < 16; e++)
            if (n0 + acc_row(e, g) > lim || (ok >> (e >> 2) & 1) == 0) y[e] = -INFINITY;
        }
        top = largest(y);
      }
      if (__builtin_amdgcn_ballot_w64(top > ref + SLACK) != 0) {
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
      bf16x8 pb[2];
      u32x4 kf[KM];
      i32x2 vf[2][DT];
      float vs[4];
#pragma unroll
      for (int n = 0; n < 4; n++) vs[n] = q8_scale((unsigned)__builtin_amdgcn_readlane((int)vsc, 8 + VROW / 8 + n));
      auto weight = [&](int e) __attribute__((always_inline)) {
        const float w = ody_exp2(fmaf(y[e], c2, minus));
        l4[e & 3] += w;
        pb[e >> 3][e & 7] = (bf16)w;
      };
      auto values = [&](int n, int dt) __attribute__((always_inline)) {
        bf16x8 v;
        const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)vf[n][dt][0], vs[2 * n], false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)vf[n][dt][0], vs[2 * n], true);
        const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)vf[n][dt][1], vs[2 * n + 1], false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)vf[n][dt][1], vs[2 * n + 1], true);
        v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
        return v;
      };
      float scale = 0.f;
      if constexpr (NEXT >= 0) {
        scale = q8_scale((unsigned)__shfl((int)ksc, NEXT / 8 + (i >> 3)));
#pragma unroll
        for (int m = 0; m < KM; m++) kf[m] = kraw(m, NEXT);
      }
#pragma unroll
      for (int dt = 0; dt < DT; dt++) vf[0][dt] = vraw(VROW, dt);
      FENCE();
      // twelve of the sixteen weights under the scores
#pragma unroll
      for (int k = 0; k < 2 * KM; k++) {
        if constexpr (NEXT >= 0) {
          zz = mfma32(q8_operand(kf[k >> 1][2 * (k & 1)], kf[k >> 1][2 * (k & 1) + 1], scale), qf[k], k == 0 ? f32x16{0} : zz);
          FENCE();
        }
        if (k % 2 == 1) vf[1][k / 2] = vraw(VROW + 16, k / 2);
#pragma unroll
        for (int e = 12 * k / (2 * KM); e < 12 * (k + 1) / (2 * KM); e++) weight(e);
        FENCE();
      }
#pragma unroll
      for (int dt = 0; dt < DT; dt++) {
        o[dt] = mfma32(values(0, dt), pb[0], o[dt]);
        FENCE();
#pragma unroll
        for (int e = 12 + 4 * dt / DT; e < 12 + 4 * (dt + 1) / DT; e++) weight(e);
        FENCE();
      }
      if constexpr (PLAIN) top = largest(zz);
#pragma unroll
      for (int dt = 0; dt < DT; dt++) o[dt] = mfma32(values(1, dt), pb[1], o[dt]);
    };
    f32x16 x[2];
    // turn t.  PLAIN: a tile follows, of which all keys are there, as they are of this one, all of which every row of the wavefront sees
    auto turn = [&](auto plain, int t) __attribute__((always_inline)) {
      constexpr bool PLAIN = decltype(plain)::value;
      std::integral_constant<int, 0> first;
      std::integral_constant<int, 32> second;
      std::integral_constant<int, -1> no_k;
      const int n0 = key0 + KEYS * t;
      barrier();   // tile t + 1 is there, everyone is done with t - 1
      const int pages = pages2;
      if (t > 0) sc1 = sc2;
      load(t + 2, pages);
      sc2 = scales_of(t + 2, pages);
      pages2 = lookup(t + 3);
      v_to(t);
      half(plain, x[0], x[1], n0, have & 15, second, sc, first, sc);
      const unsigned rest = have >> 4;
      k_to(t + 1);
      if (PLAIN || t + 1 < tiles) half(plain, x[1], x[0], n0 + 32, rest, first, sc1, second, sc);
      else half(plain, x[1], x[0], n0 + 32, rest, no_k, sc1, second, sc);
      have = have1, have1 = with_page(pages), sc = sc1;
    };
    if (tiles > 0) {
      barrier();
      k_to(0);
      const float scale = q8_scale((unsigned)__shfl((int)sc, i >> 3));
#pragma unroll
      for (int m = 0; m < KM; m++) {
        const u32x4 k = kraw(m, 0);
        x[0] = mfma32(q8_operand(k[0], k[1], scale), qf[2 * m], m == 0 ? f32x16{0} : x[0]);
        x[0] = mfma32(q8_operand(k[2], k[3], scale), qf[2 * m + 1], x[0]);
      }
      top = largest(x[0]);
      std::true_type yes;
      std::false_type no;
      // plain turns, and from the first one on that is not, the others
      int t = 0;
      while (t + 1 < tiles && key0 + KEYS * (t + 2) <= keys && key0 + KEYS * (t + 1) - 1 <= safe && (have & have1) == 0xff) turn(yes, t++);
      while (t < tiles) turn(no, t++);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();   // everyone is done with the tiles, and nothing is on its way to them

    const float sum = half_swap_sum((l4[0] + l4[1]) + (l4[2] + l4[3]));
    if (32 * wave + i < rows) {
      if (whole) {
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
    pos += span;
    if (pos < end) at.next_unit(walk);
  }
}

template <int D>
int launch(const PagedAttnParams& p, const PagedCache& c, const PagedScales& z, int blocks, hipStream_t st) {
  constexpr size_t smem = (size_t)2 * SLOTS * KEYS * D;
  if (int rc = ody_allow_dynamic_lds(reinterpret_cast<const void*>(&paged_chunk_q8_kernel<D>), smem, "ody_paged_attn_q8")) return rc;
  ODY_LAUNCH("paged_chunk_q8", st, (paged_chunk_q8_kernel<D>), dim3(blocks), dim3(64 * WAVES), smem, p, c, z);
  return ody_check_launch("paged_chunk_q8");
}

}  // namespace

int ody_launch_paged_chunk_q8(const PagedAttnParams& p, int D, const PagedCache& c, const PagedScales& z, int blocks, hipStream_t st) {
  return D == 64 ? launch<64>(p, c, z, blocks, st) : launch<128>(p, c, z, blocks, st);
}
