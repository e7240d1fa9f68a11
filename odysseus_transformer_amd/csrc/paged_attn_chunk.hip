// Attention of many new tokens over a key / value cache in pages, bf16: a chunk of a prompt, or many rows of a kv head (its query heads times the
// tokens) by a few tokens of many sequences; the rule is in paged_attn.hip.
//
// Bound by the matrix cores and, as much, by the vector work of the softmax between the two products.  A block of four wavefronts takes 128 rows of one
// (sequence, kv head), 32 a wavefront, and walks over the keys in tiles of 64, two halves each.  Both products are computed transposed, so that a row's
// reference and sum belong to one lane and the one 32 lanes away:
//
//      S^T (keys x rows) = K Q^T        A: K rows from LDS      B: this lane's query row, in registers
//      O^T (D x rows) += V^T P^T        B: P^T as the accumulators of S^T hold it      A: V^T by transposing LDS reads
//
// on v_mfma_f32_32x32x16_bf16, LDS rows laid out and read as attn_rowtile.h has it.  S of the next half is formed under the softmax of the present one, whose
// P V follows; the other block on the compute unit fills what either leaves free.  Direct loads bring V a turn ahead and K one and a half, two places in
// LDS for each.
//
// P is rounded to bf16 for its product and summed up in fp32 unrounded, as in the attention over contiguous keys.
//
// Measured with the join, 32 heads on 8 of 128 in pages of 16: 128 tokens behind 2000 keys 25 us, 256 behind 8192 58 (590 TFLOP/s), behind 32768 158 (870); heads of 64,
// 512 behind 8191, 61 (580), 2048 behind 8192 222 (700).  Heads of 128 take 156 bytes of scratch memory: the loop of plain turns has none of it, a turn that is not plain
// reloads 20 registers, for which it waits until the direct loads in front of them have landed too.
#include <cmath>
#include <type_traits>
#include "attn_rowtile.h"
#include "paged.h"

namespace {

using namespace rowtile;

constexpr int KEYS = PAGED_CHUNK_KEYS, BLOCK_ROWS = PAGED_CHUNK_ROWS, WAVES = 4;
static_assert(KEYS == ROWS && BLOCK_ROWS == 32 * WAVES, "a tile of keys, 32 rows a wavefront");
// How far, in powers of two, a score may be above its row's reference before the reference follows: P is up to 2^8 then, as exact in bf16 as below 1,
// and sums of 2^31 of them are far from what fp32 holds.  (With 0 every second sub-tile of random scores rescales the accumulators.)
constexpr float SLACK = 8.f;
#define FENCE() __builtin_amdgcn_sched_barrier(0)   // the compiler's order of instructions ends here

__device__ const bf16x8 no_key[16] = {};   // the row that a key without a page, or behind the last one, is read from

// A direct load, 16 bytes a lane, to LDS address `to` on.  As assembly, for behind the builtin the compiler makes transposing reads wait for it (they could
// read what it writes, as far as it knows); the waits that there have to be stand in the loop.  It has no result that the compiler could use too early,
// and nothing else in these kernels uses m0 (a reserved register, which cannot be named as overwritten; a test looks through the generated code).
__device__ __forceinline__ void direct_load(const char* from, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}
__device__ __forceinline__ void direct_load(const char* from, unsigned of_lane, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(of_lane), "s"(from) : "memory");
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// A operand of the transposed V rows FIRST .. FIRST + 15, columns 32 dt .. + 31, as tr_frags of attn_rowtile.h reads it
template <int D>
__device__ __forceinline__ bf16x8 column_frag(const Readers<D>& r, int first, int dt) {
  typedef s16x4 __attribute__((address_space(3))) * lds_s16x4_ptr;
  return concat4(__builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(uintptr_t)(r.tr[2 * dt] + 2 * first * D))),
                 __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(uintptr_t)(r.tr[2 * dt + 1] + 2 * (first + 8) * D))));
}

template <int D>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_chunk_kernel(const PagedAttnParams p, const PagedCache cache) {
  constexpr int KS = D / 16, DT = D / 32, TILE = KEYS * D;                              // elements of a tile
  constexpr int LANES = D / 8, PER = 64 / LANES, STEP = PER * WAVES, LOADS = KEYS / STEP;   // of a direct load: lanes on a row, rows; of a tile
  static_assert(STEP % 16 == 0, "swz of the rows of the other loads");
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const unsigned places = (unsigned)(uintptr_t)(lds_ptr)smem;   // LDS address of [K | V][2][KEYS][D]

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 5, i = lane & 31;
  PagedWalk<KEYS> walk(p, cache, lane);
  const int each = walk.total();   // steps of a kv head
  const PagedCuts cuts(each * p.Hkv, paged_blocks(p, each * p.Hkv, gridDim.x));
  const int block = paged_range(blockIdx.x, cuts.blocks);
  if (block >= cuts.blocks) return;
  const int begin = cuts.at(block), end = cuts.at(block + 1);
  int pos = begin;
  PagedPlace<KEYS> at(walk, pos, each);
  const int lcol = 8 * ((lane % LANES) ^ swz<D>(PER * wave + lane / LANES));   // of this lane in its direct loads
  const unsigned lk = lane / LANES * cache.k_row + 2 * lcol, lv = lane / LANES * cache.v_row + 2 * lcol;   // bytes
  const float c2 = p.scale_log2e;
  Readers<D> rd;
  rd.init(reinterpret_cast<const bf16*>(smem), g, i);

  while (pos < end) {
    const int s = at.s, rt = at.rt, hk = at.hk, length = at.length, row0 = rt * BLOCK_ROWS;
    const int span = min(at.steps - at.step, end - pos), step = max(0, at.step - PAGED_EXTRA), steps_here = at.step + span - PAGED_EXTRA - step;
    const bool whole = step == 0 && at.step + span == at.steps;
    if (steps_here <= 0) break;   // the range ends with what a unit costs besides its steps
    const int rows = min(BLOCK_ROWS, p.n * p.group - row0);
    const int none = p.n - at.fresh;   // the first tokens, which are none
    const int keys = paged_keys(p, cache, length, at.fresh, rt), tiles = keys > 0 ? steps_here : 0;
    const int key0 = KEYS * step;
    const char* kp = reinterpret_cast<const char*>(static_cast<const bf16*>(cache.k) + hk * cache.sk.h);
    const char* vp = reinterpret_cast<const char*>(static_cast<const bf16*>(cache.v) + hk * cache.sv.h);
    const int* table = cache.table + s * cache.table_stride;

    // ---- lane n % 8 holds the page of a tile's n-th group of 8 keys; the rows of a direct load are in one of them
    auto lookup = [&](int t) { return table[min(key0 + KEYS * t + 8 * (lane & 7), keys - 1) >> cache.shift]; };
    auto with_page = [&](int pages) { return (unsigned)__builtin_amdgcn_ballot_w64((unsigned)pages < (unsigned)cache.pages) & 0xff; };
    // Load j of a tile's.  PLAIN: all of the tile's keys are there
    auto load = [&](auto plain, int j, int t, int pages, unsigned have, const char* base, unsigned of_page, unsigned of_row, unsigned of_lane, unsigned place) __attribute__((always_inline)) {
      const int first = key0 + KEYS * t + PER * wave + STEP * j, in_page = (1 << cache.shift) - 1;
      const int at = (STEP * j + PER * wave) / 8, page = __builtin_amdgcn_readlane(pages, at);
      const char* row = base + (uint64_t)(unsigned)page * of_page + (unsigned)(first & in_page) * of_row;
      const unsigned to = place + (WAVES * j + wave) * 1024;
      if constexpr (decltype(plain)::value) {
        direct_load(row, of_lane, to);
      } else {
        const bool none = first + lane / LANES >= keys || (have >> at & 1) == 0;
        unsigned l = of_lane;
        asm volatile("" : "+v"(l));   // 64 bits of it here, and not from turn to turn: the loops have no register to spare (that of plain turns went to scratch memory)
        direct_load(none ? reinterpret_cast<const char*>(no_key) + 2 * lcol : row + l, to);
      }
    };
    auto load_k = [&](auto plain, int j, int t, int pages, unsigned have) __attribute__((always_inline)) { load(plain, j, t, pages, have, kp, cache.k_page, cache.k_row, lk, places + (t & 1) * 2 * TILE); };
    auto load_v = [&](auto plain, int j, int t, int pages, unsigned have) __attribute__((always_inline)) { load(plain, j, t, pages, have, vp, cache.v_page, cache.v_row, lv, places + (2 + (t & 1)) * 2 * TILE); };
    std::true_type yes;
    std::false_type no;
    // of the tiles behind the present one: pages, and which groups have one
    int pages1 = 0, pages2 = 0, pages3 = 0;
    unsigned have = 0, have1 = 0;
    if (tiles > 0) {
      const int pages0 = lookup(0);
      pages1 = lookup(1), pages2 = lookup(2), pages3 = lookup(3);
      have = with_page(pages0);
#pragma unroll
      for (int j = 0; j < LOADS; j++) load_k(no, j, 0, pages0, have);
#pragma unroll
      for (int j = 0; j < LOADS; j++) load_v(no, j, 0, pages0, have);
      have1 = with_page(pages1);
      if (tiles > 1) {
#pragma unroll
        for (int j = 0; j < LOADS; j++) load_k(no, j, 1, pages1, have1);
      }
    }

    // ---- this lane's row: token ri, query head h
    const int r = row0 + min(32 * wave + i, rows - 1), ri = r / p.group, h = hk * p.group + r - ri * p.group;
    bf16x8 qf[KS];
    {
      const bf16* qp = static_cast<const bf16*>(p.q) + s * p.sq.b + ri * p.sq.l + h * p.sq.h + 8 * g;
#pragma unroll
      for (int ks = 0; ks < KS; ks++) qf[ks] = p.signed_query(*reinterpret_cast<const bf16x8*>(qp + 16 * ks));
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
    // A half: the softmax of y, the scores against keys n0 .., of which PLAIN says that every row sees all; S of the next half (with the K rows from NEXT on,
    // into z); P V with the V rows from VROW on.  `loads` (of j) go out under it.  Sixteen products, and with each of them what follows it here of the rest.
    auto half = [&](auto plain, f32x16& y, f32x16& z, int n0, unsigned ok, auto next_, auto vrow_, auto loads) __attribute__((always_inline)) {
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
      bf16x8 pb[2], kf[4], vf[2][DT];
      auto weight = [&](int e) __attribute__((always_inline)) {
        const float w = ody_exp2(fmaf(y[e], c2, minus));
        l4[e & 3] += w;
        pb[e >> 3][e & 7] = (bf16)w;
      };
      if constexpr (NEXT >= 0) {
#pragma unroll
        for (int ks = 0; ks < 4; ks++) kf[ks] = row_frag(rd, NEXT, ks);
      }
      FENCE();
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        if constexpr (NEXT >= 0) {
          z = mfma32(kf[ks % 4], qf[ks], ks == 0 ? f32x16{0} : z);
          FENCE();
          if (ks + 4 < KS) kf[ks % 4] = row_frag(rd, NEXT, ks + 4);
        }
        if (ks >= KS - DT) vf[0][ks - (KS - DT)] = column_frag(rd, VROW, ks - (KS - DT));
        if (ks % (KS / LOADS) == 0) loads(ks / (KS / LOADS));
        // twelve of the sixteen weights under the scores
#pragma unroll
        for (int e = 12 * ks / KS; e < 12 * (ks + 1) / KS; e++) weight(e);
        FENCE();
      }
#pragma unroll
      for (int dt = 0; dt < DT; dt++) {
        o[dt] = mfma32(vf[0][dt], pb[0], o[dt]);
        FENCE();
        vf[1][dt] = column_frag(rd, VROW + 16, dt);
#pragma unroll
        for (int e = 12 + 4 * dt / DT; e < 12 + 4 * (dt + 1) / DT; e++) weight(e);
        FENCE();
      }
      if constexpr (PLAIN) top = largest(z);
#pragma unroll
      for (int dt = 0; dt < DT; dt++) o[dt] = mfma32(vf[1][dt], pb[1], o[dt]);
    };
    f32x16 x[2];
    auto nothing = [](int) {};
    // turn t: P = t mod 2.  PLAIN: two tiles follow, of which all keys are there, as they are of this one, all of which every row of the wavefront sees
    auto turn = [&](auto plain, int t, auto parity) __attribute__((always_inline)) {
      constexpr int P = decltype(parity)::value;
      constexpr bool PLAIN = decltype(plain)::value;
      std::integral_constant<int, KEYS * P + 32> k_here;
      std::integral_constant<int, KEYS * (P ^ 1)> k_next;
      std::integral_constant<int, KEYS * (2 + P)> v_here;
      std::integral_constant<int, KEYS * (2 + P) + 32> v_half;
      std::integral_constant<int, -1> no_k;
      const int n0 = key0 + KEYS * t;
      const bool more = PLAIN || t + 1 < tiles;
      barrier();   // V of t is there, everyone is done with V of t - 1
      half(plain, x[0], x[1], n0, have & 15, k_here, v_here, [&](int j) __attribute__((always_inline)) { if (more) load_v(plain, j, t + 1, pages1, have1); });
      const unsigned second = have >> 4;
      have = have1;
      if (more) {
        wait_loads<LOADS>();
        barrier();   // K of t + 1 is there, everyone is done with K of t
        have1 = with_page(pages2);
        half(plain, x[1], x[0], n0 + 32, second, k_next, v_half, [&](int j) __attribute__((always_inline)) {
          if (PLAIN || t + 2 < tiles) load_k(plain, j, t + 2, pages2, have1);
        });
        pages1 = pages2, pages2 = pages3, pages3 = lookup(t + 4);
      } else {
        half(plain, x[1], x[0], n0 + 32, second, no_k, v_half, nothing);
      }
    };
    if (tiles > 0) {
      wait_loads<0>();
      barrier();
#pragma unroll
      for (int ks = 0; ks < KS; ks++) x[0] = mfma32(row_frag(rd, 0, ks), qf[ks], ks == 0 ? f32x16{0} : x[0]);
      top = largest(x[0]);
      // V of t has to be there; K of t + 1 and two page numbers may be under way
      auto wait_v = [&](int t) {
        if (t + 1 < tiles) wait_loads<LOADS + 1>();
        else wait_loads<0>();
      };
      auto is_plain = [&](int t) {
        return t + 2 < tiles && key0 + KEYS * (t + 3) <= keys && key0 + KEYS * (t + 1) - 1 <= safe && (have & have1 & with_page(pages2)) == 0xff;
      };
      std::integral_constant<int, 0> even;
      std::integral_constant<int, 1> odd;
      // plain turns, and from the first one on that is not, the others
      int t = 0;
      for (;; t++) {
        wait_v(t);
        if (!is_plain(t)) break;
        turn(yes, t, even);
        wait_v(++t);
        if (!is_plain(t)) break;
        turn(yes, t, odd);
      }
      for (bool at_odd = t & 1; t < tiles; at_odd = false) {
        if (!at_odd) {
          wait_v(t);
          turn(no, t++, even);
          if (t >= tiles) break;
        }
        wait_v(t);
        turn(no, t++, odd);
      }
    }
    __syncthreads();   // everyone is done with the tiles

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
