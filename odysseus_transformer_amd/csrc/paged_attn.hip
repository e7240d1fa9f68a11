// Attention of new tokens over a key / value cache in pages.
//
// Bound by reading K and V once.  A wavefront takes a tile of keys (32 in bf16, 16 in fp32) for all rows of a row tile (16 NT of them: the
// query heads that share a kv head, times the new tokens) at once, and nothing but registers lies between memory and the matrix cores:
//
//      S^T = K Q^T          A: K rows in operand order, 16 bytes a lane        B: Q^T, in registers
//      O^T += V^T P^T       A: V^T, the lane's own rows transposed in its registers   B: P^T = accumulator layout of S^T
//
// on v_mfma_f32_16x16x32_bf16 / v_mfma_f32_16x16x4_f32 (lane = 16 q + c: A row c / B column c; accumulator column c, rows 4 q .. 4 q + 3).  The key that
// row c of a K operand stands for is chosen so that a lane's scores are those of GK keys in a row, tile + GK q ..: its P is then the B operand for the very
// keys whose V rows this lane loads.  V rows are loaded GK at a time with 16 lanes on a row; component i of the vectors is row c of operand i, which
// stands for column c * DV + i of V, so the transposition is bytes exchanged within a lane (bf16) or nothing at all (fp32).
// In bf16 P is rounded for its product, as V is stored, and summed up in fp32 unrounded, as in the attention over contiguous keys: half a step of each weight.
// A tile's K goes out when the products have read that of the one before, and so does its V (two tiles in registers, the one under way while the products read
// the other: the same times to 1 %).  A group of GK keys lies within a page: two table entries a lane and tile.
//
// Measured, bf16, heads of 128, results joined: 64 sequences of up to 8192 keys, 32 heads on 8, in rows of all heads 196 to 200 us (5.4 TB/s of K and V; a copy runs
// at 5.1, a sum at 6.0 to 6.3), with heads outside of rows 171 to 177 (6.1); 16 of 4001, 32 heads, 125 us (5.5); one of 131072 100 us (5.4), of 8192 13.5, where launches
// and the chain length, table, keys, join are all.  One of 100 5.4 under a table of one step, 7.4 under a wider one, for which the join is launched too.
#include <algorithm>
#include <cmath>
#include "paged_join.h"

namespace {

// Two blocks on each of 256 compute units.  256 / 512 / 1024: 64 sequences of up to 8192 keys 218 / 202 / 203 us, one of 8192 13.7 / 14.0 / 14.0, chunks of
// 512 tokens behind 8192 (paged_attn_chunk.hip) 110 / 106 / 130.
constexpr int WAVES = 4, BLOCKS = 512;

template <typename T, int D> struct Tile;
template <int D> struct Tile<bf16, D> {
  static constexpr int KEYS = 32, GK = 8, KV = 2 * (D / 32), DV = D / 16;   // keys, keys of a group, K vectors and V columns a lane
  typedef bf16x8 kvec;
  typedef bf16 vvec __attribute__((ext_vector_type(DV)));
  // K vector j of a lane: operand row c stands for key 8 (c / 4) + 4 (j / (D / 32)) + c % 4
  __device__ static constexpr int key_row(int j) { return 4 * (j / (D / 32)); }
  __device__ static constexpr int key_col(int q, int j) { return 32 * (j % (D / 32)) + 8 * q; }
};
template <int D> struct Tile<float, D> {
  static constexpr int KEYS = 16, GK = 4, KV = D / 16, DV = D / 16;
  typedef f32x4 kvec;
  typedef float vvec __attribute__((ext_vector_type(DV)));
  __device__ static constexpr int key_row(int) { return 0; }
  __device__ static constexpr int key_col(int q, int j) { return 16 * j + 4 * q; }
};

// scores of the lane's GK keys against column c's query row
template <int D>
__device__ __forceinline__ void scores(const bf16x8 (&k)[D / 16], const bf16x8 (&qf)[D / 32], float (&x)[8]) {
#pragma unroll
  for (int st = 0; st < 2; st++) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < D / 32; ks++) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[st * (D / 32) + ks], qf[ks], s, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; r++) x[4 * st + r] = s[r];
  }
}
template <int D>
__device__ __forceinline__ void scores(const f32x4 (&k)[D / 16], const f32x4 (&qf)[D / 16], float (&x)[4]) {
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < D / 16; j++)
#pragma unroll
    for (int e = 0; e < 4; e++) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[j][e], qf[j][e], s, 0, 0, 0);
#pragma unroll
  for (int r = 0; r < 4; r++) x[r] = s[r];
}

// o[i], row c: column c * DV + i of the result
template <int D, int NT>
__device__ __forceinline__ void values(const typename Tile<bf16, D>::vvec (&rows)[8], const float (&w)[NT][8], f32x4 (&o)[NT][D / 16]) {
  bf16x8 pb[NT];
#pragma unroll
  for (int m = 0; m < NT; m++)
#pragma unroll
    for (int e = 0; e < 8; e++) pb[m][e] = (bf16)w[m][e];
  unsigned v[8][D / 32];
#pragma unroll
  for (int j = 0; j < 8; j++) __builtin_memcpy(v[j], &rows[j], sizeof(v[j]));
#pragma unroll
  for (int i = 0; i < D / 16; i++) {
    i32x4 a;
#pragma unroll
    for (int j = 0; j < 4; j++) a[j] = __builtin_amdgcn_perm(v[2 * j + 1][i / 2], v[2 * j][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
    const bf16x8 af = __builtin_bit_cast(bf16x8, a);
#pragma unroll
    for (int m = 0; m < NT; m++) o[m][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, pb[m], o[m][i], 0, 0, 0);
  }
}
template <int D, int NT>
__device__ __forceinline__ void values(const typename Tile<float, D>::vvec (&rows)[4], const float (&w)[NT][4], f32x4 (&o)[NT][D / 16]) {
#pragma unroll
  for (int r = 0; r < 4; r++)
#pragma unroll
    for (int i = 0; i < D / 16; i++)
#pragma unroll
      for (int m = 0; m < NT; m++) o[m][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(rows[r][i], w[m][r], o[m][i], 0, 0, 0);
}

template <bool STREAM, typename V>
__device__ __forceinline__ V load_vector(const char* p) {
  typedef unsigned raw __attribute__((ext_vector_type(sizeof(V) / 4)));
  if constexpr (STREAM) return __builtin_bit_cast(V, __builtin_nontemporal_load(reinterpret_cast<const raw*>(p)));
  else return *reinterpret_cast<const V*>(p);
}

// STREAM: keys that one row tile reads, in rows of whole cache lines, take no cache room (16 x 4001 keys of 32 heads 130 -> 124 us, 131072 of 8 heads 103 -> 100;
// in rows of 64 columns, of which a load takes half a line, 16.6 -> 17.7).
template <typename T, int D, int NT, bool STREAM>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_attn_kernel(const PagedAttnParams p, const PagedCache cache) {
  typedef Tile<T, D> G;
  constexpr int STEP = WAVES * G::KEYS, GK = G::GK, OP = D + 4;
  __shared__ __attribute__((aligned(16))) float Os[WAVES][16][OP];
  __shared__ float sm[WAVES][16 * NT], sl[WAVES][16 * NT];
  paged_arguments(p, cache);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c = lane & 15, q = lane >> 4;
  PagedWalk<STEP> walk(p, cache, lane);
  const int each = walk.total();   // steps of a kv head
  const PagedCuts cuts(each * p.Hkv, paged_blocks(p, each * p.Hkv, gridDim.x));
  const int block = paged_range(blockIdx.x, cuts.blocks);
  if (block >= cuts.blocks) return;
  const int begin = cuts.at(block), end = cuts.at(block + 1);
  int pos = begin;
  const unsigned of_lane_k = (c & 3) * cache.k_row + G::key_col(q, 0) * sizeof(T), of_lane_v = c * G::DV * sizeof(T);
  PagedPlace<STEP> at(walk, pos, each);

  while (pos < end) {
    const int s = at.s, rt = at.rt, hk = at.hk, length = at.length, step = at.step, steps = at.steps, row0 = rt * p.tile;
    const int rows = min(p.tile, p.n * p.group - row0);
    const int none = p.n - at.fresh;   // the first tokens, which are none
    const int keys = paged_keys(p, cache, length, at.fresh, rt), steps_here = min(steps - step, end - pos);
    const char* kp = reinterpret_cast<const char*>(static_cast<const T*>(cache.k) + hk * cache.sk.h) + of_lane_k;
    const char* vp = reinterpret_cast<const char*>(static_cast<const T*>(cache.v) + hk * cache.sv.h) + of_lane_v;
    const int* table = cache.table + s * cache.table_stride;
    const int in_page = (1 << cache.shift) - 1, last_group = max(keys - 1, 0) & -GK;

    // ---- row 16 m + c: token (row0 + ..) / group, query head hk * group + (row0 + ..) % group
    typename G::kvec qf[NT][D * sizeof(T) / 64];
    int lim[NT];   // last key the row sees
    int safe = keys - 1;
#pragma unroll
    for (int m = 0; m < NT; m++) {
      const int r = row0 + min(16 * m + c, rows - 1), i = r / p.group, h = hk * p.group + r - i * p.group;
      const T* qp = static_cast<const T*>(p.q) + s * p.sq.b + i * p.sq.l + h * p.sq.h;
#pragma unroll
      for (int j = 0; j < (int)(D * sizeof(T) / 64); j++) qf[m][j] = p.signed_query(*reinterpret_cast<const typename G::kvec*>(qp + G::key_col(q, j)));
      lim[m] = i < none ? -1 : min(keys - 1, length - p.n + i);
    }
    safe = row0 / p.group < none ? -1 : min(safe, length - p.n + row0 / p.group);

    f32x4 o[NT][D / 16];
    float mx[NT], l[NT];
#pragma unroll
    for (int m = 0; m < NT; m++) {
      mx[m] = -INFINITY, l[m] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; i++) o[m][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // ---- the wavefront's tiles: keys (step + t) * STEP + wave * KEYS ..
    const int key0 = step * STEP + wave * G::KEYS;
    const int tiles = key0 >= keys ? 0 : min(steps_here, (keys - key0 + STEP - 1) / STEP);
    struct Pages { int k, v; };
    auto lookup = [&](int t) {   // of the groups that the lane's K row and V rows are in
      const int base = key0 + min(t, tiles - 1) * STEP;
      return Pages{table[min(base + GK * (c >> 2), last_group) >> cache.shift], table[min(base + GK * q, last_group) >> cache.shift]};
    };
    struct Loaded {   // a tile's rows
      typename G::kvec k[G::KV];
      typename G::vvec v[GK];
      bool page;      // the lane's keys, tile + GK q .., have one
    };
    auto load_k = [&](Loaded& to, int t, const Pages& pg) __attribute__((always_inline)) {
      const int gk = min(key0 + t * STEP + GK * (c >> 2), last_group);
      const char* src = kp + (uint64_t)((unsigned)pg.k < (unsigned)cache.pages ? pg.k : 0) * cache.k_page + (unsigned)(gk & in_page) * cache.k_row;
#pragma unroll
      for (int j = 0; j < G::KV; j++)
        to.k[j] = load_vector<STREAM, typename G::kvec>(src + G::key_row(j) * (uint64_t)cache.k_row + G::key_col(0, j) * sizeof(T));
    };
    auto load_v = [&](Loaded& to, int t, const Pages& pg) __attribute__((always_inline)) {
      const int gv = min(key0 + t * STEP + GK * q, last_group);
      to.page = (unsigned)pg.v < (unsigned)cache.pages;
      const char* src = vp + (uint64_t)(to.page ? pg.v : 0) * cache.v_page + (unsigned)(gv & in_page) * cache.v_row;
#pragma unroll
      for (int j = 0; j < GK; j++) to.v[j] = load_vector<STREAM, typename G::vvec>(src + j * (uint64_t)cache.v_row);
    };
    // the products with tile t; `k_read` is called when those with its K have been formed
    auto compute = [&](Loaded& x, int t, auto k_read) __attribute__((always_inline)) {
      const int base = key0 + t * STEP, first = base + GK * q;   // the lane's keys
      float w[NT][GK];
#pragma unroll
      for (int m = 0; m < NT; m++) scores<D>(x.k, qf[m], w[m]);
      k_read();
      // keys that a row does not see, that no token has, that have no page: neither their scores nor their values count, whatever lies there
      if (base + G::KEYS - 1 > safe || !__all(x.page)) {
        const int most = x.page ? keys - 1 : -1;
#pragma unroll
        for (int e = 0; e < GK; e++) {
#pragma unroll
          for (int m = 0; m < NT; m++)
            if (first + e > min(lim[m], most)) w[m][e] = -INFINITY;
          if (first + e > most) x.v[e] = typename G::vvec{};
        }
      }
#pragma unroll
      for (int m = 0; m < NT; m++) {
        float top = w[m][0];
#pragma unroll
        for (int e = 1; e < GK; e++) top = fmaxf(top, w[m][e]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float now = fmaxf(mx[m], top * p.scale_log2e), ref = now == -INFINITY ? 0.f : now, alpha = ody_exp2(mx[m] - ref);
        mx[m] = now;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < GK; e++) w[m][e] = ody_exp2(fmaf(w[m][e], p.scale_log2e, -ref)), sum += w[m][e];
        l[m] = l[m] * alpha + sum;   // this lane's share of the row sum
#pragma unroll
        for (int i = 0; i < D / 16; i++) o[m][i] *= alpha;
      }
      values<D, NT>(x.v, w, o);
    };
    if (tiles > 0) {
      Pages now = lookup(0), next = lookup(1);
      Loaded x;
      load_k(x, 0, now);
      load_v(x, 0, now);
      now = next, next = lookup(2);
      for (int t = 0; t < tiles; t++) {
        compute(x, t, [&]() __attribute__((always_inline)) { if (t + 1 < tiles) load_k(x, t + 1, now); });
        if (t + 1 < tiles) {
          load_v(x, t + 1, now);
          now = next, next = lookup(t + 3);
        }
      }
    }

    // ---- the four wavefronts' results of a row: common reference, weighted sum
#pragma unroll
    for (int m = 0; m < NT; m++) {
      l[m] += __shfl_xor(l[m], 16, 64);
      l[m] += __shfl_xor(l[m], 32, 64);
      if (q == 0) sm[wave][16 * m + c] = mx[m], sl[wave][16 * m + c] = l[m];
    }
    __syncthreads();
    const bool whole = steps_here == steps;
    const int64_t slot = 2 * block + (pos > begin);   // the unit that the range begins with, or the one that it ends with
#pragma unroll
    for (int m = 0; m < NT; m++) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WAVES; w++) top = fmaxf(top, sm[w][16 * m + c]);
      const float mine = ody_exp2(mx[m] - (top == -INFINITY ? 0.f : top));
      // o[i][r] of row 4 q + r: column (4 q + r) * DV + i
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int i = 0; i < D / 16; i += 4)
          *reinterpret_cast<f32x4*>(&Os[wave][c][(4 * q + r) * G::DV + i]) = f32x4{o[m][i][r], o[m][i + 1][r], o[m][i + 2][r], o[m][i + 3][r]} * mine;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 16 * D / 4 / (64 * WAVES); e++) {
        const int idx = tid + 64 * WAVES * e, row = idx / (D / 4), d4 = idx % (D / 4), r = 16 * m + row;
        if (r >= rows) continue;
        float t = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) t = fmaxf(t, sm[w][r]);
        const float ref = t == -INFINITY ? 0.f : t;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
          sum += sl[w][r] * ody_exp2(sm[w][r] - ref);
          acc += *reinterpret_cast<const f32x4*>(&Os[w][row][4 * d4]);
        }
        if (whole) {
          const int i = (row0 + r) / p.group, h = hk * p.group + (row0 + r) - i * p.group;
          acc *= sum == 0.f ? 0.f : 1.f / sum;
          T* dst = static_cast<T*>(p.out) + s * p.so.b + i * p.so.l + h * p.so.h + 4 * d4;
          typedef T out4 __attribute__((ext_vector_type(4)));
          *reinterpret_cast<out4*>(dst) = out4{(T)acc[0], (T)acc[1], (T)acc[2], (T)acc[3]};
          if (d4 == 0) p.lse[((int64_t)s * p.Hq + h) * p.n + i] = sum == 0.f ? -INFINITY : (t + __log2f(sum)) * ODY_LN2;
        } else {
          *reinterpret_cast<f32x4*>(p.part + (slot * p.tile + r) * D + 4 * d4) = acc;
          if (d4 == 0) p.part_ml[slot * p.tile + r] = make_float2(t, sum);
        }
      }
      __syncthreads();
    }

    pos += steps_here;
    if (pos < end) at.next_unit(walk);
  }
}

// The host knows no lengths: `keys` below are the places of the table (17 tokens of one sequence behind 500 keys, 32 heads on 8: 12.6 us under a table for at most 16384
// keys, 16.2 under a wider one).
// Row tiles of 16 or 32 here (64 would not fit the registers); many rows in bf16 by the kernels for them: from 129 on, from 65 on but for few (sequence, kv head)
// pairs and few keys, where more, shorter ranges win (32 heads on 8: 17 tokens behind 500 / 2000 / 8192 / 32768 keys 13.6 / 15.1 / 25.2 / 47 us here, 17.6 / 19.6 / 26.4
// / 43 there; of 4 sequences 20 / 28 / 51 and 18 / 25 / 41), and from 33 on where there are many, which would be read from memory twice here (10 tokens each of 64
// sequences of up to 8192 keys 371 us here, 254 there, of up to 1000 63 and 54; 8 of 4000 39 and 41, one of 2000 13 and 19).
// paged_attn_wide.hip for heads of 128 where 64 units and more keep its 256 blocks busy (2000 keys, 32 heads on 8: 128 tokens, which are 16 units, 34 us, 28 in tiles of
// 128, 512 tokens, 64 units, 44 and 46; between them, and with few units of many keys, the two have not been timed against each other; 2048 tokens behind 8192 keys 312
// and 354, in pages of 16 328 and 357; 300 each of 64 sequences of up to 3000 keys, pages of 16, 637 and 774) and its tiles
// cover at most a seventh more rows than tiles of 128 would (257 rows of each of 32 heads behind 8192 keys: 91 us in two of 256, 78 in three).
struct Plan {
  int tile, row_tiles, step, blocks;
  bool joined;          // a cut may go through a unit
  bool fits;            // the steps can be counted
  size_t part_bytes, ml_bytes;
};
Plan plan(int S, int n, int group, int Hkv, int D, int page_size, int width, int dtype) {
  const int64_t most_keys = (int64_t)page_size * width;
  const int64_t rows = (int64_t)n * group;
  const double pairs = (double)S * Hkv;
  const bool chunk = dtype == ODY_BF16 && (rows > 128 || (rows > 64 ? pairs >= 16 || most_keys > 16384 : rows > 32 && pairs >= 128));
  const int64_t wide_tiles = (rows + PAGED_WIDE_ROWS - 1) / PAGED_WIDE_ROWS, chunk_tiles = (rows + PAGED_CHUNK_ROWS - 1) / PAGED_CHUNK_ROWS;
  const bool wide = chunk && D == 128 && (double)S * wide_tiles * Hkv >= 64 && 14 * wide_tiles <= 8 * chunk_tiles;
  const int tile = rows <= 16 ? 16 : wide ? PAGED_WIDE_ROWS : chunk ? PAGED_CHUNK_ROWS : 32, row_tiles = (int)((rows + tile - 1) / tile);
  const int step = chunk ? PAGED_CHUNK_KEYS : WAVES * (dtype == ODY_BF16 ? 32 : 16);
  const int64_t steps = std::max((int64_t)1, (most_keys + step - 1) / step);   // of a unit, at most
  const double all = (double)S * row_tiles * Hkv * (steps + paged_extra(tile));
  const int blocks = (int)std::min((double)(wide ? BLOCKS / 2 : BLOCKS), std::ceil(all / 8) * 8);   // a multiple of 8: paged_range
  const bool joined = steps > 1;
  const size_t parts = joined ? (size_t)blocks * 2 * tile : 0;
  return Plan{tile, row_tiles, step, blocks, joined, all < 2147483648.0, parts * D * sizeof(float), parts * sizeof(float2)};
}

template <typename T, int D, int NT>
int launch(const PagedAttnParams& p, const PagedCache& c, const Plan& pl, hipStream_t st) {
  constexpr bool LINES = D == 128;   // a tile of 16 rows is the only one
  if (NT == 1 || (LINES && pl.row_tiles == 1)) ODY_LAUNCH("paged_attn", st, (paged_attn_kernel<T, D, NT, LINES>), dim3(pl.blocks), dim3(64 * WAVES), 0, p, c);
  else ODY_LAUNCH("paged_attn", st, (paged_attn_kernel<T, D, NT, NT == 1 && LINES>), dim3(pl.blocks), dim3(64 * WAVES), 0, p, c);
  const int rc = ody_check_launch("paged_attn");
  return rc ? rc : paged_join<T, D, WAVES * Tile<T, D>::KEYS, 1>(p, c, pl.joined, pl.blocks, st);
}
template <typename T, int D>
int by_rows(const PagedAttnParams& p, const PagedCache& c, const Plan& pl, hipStream_t st) {
  if (pl.tile >= PAGED_CHUNK_ROWS) {
    const int rc = pl.tile == PAGED_WIDE_ROWS ? ody_launch_paged_wide(p, c, pl.blocks, st) : ody_launch_paged_chunk(p, D, c, pl.blocks, st);
    return rc ? rc : paged_join<bf16, D, PAGED_CHUNK_KEYS, PAGED_JOIN_ROWS>(p, c, pl.joined, pl.blocks, st);
  }
  return pl.tile == 16 ? launch<T, D, 1>(p, c, pl, st) : launch<T, D, 2>(p, c, pl, st);
}
template <typename T>
int by_head_dim(const PagedAttnParams& p, int D, const PagedCache& c, const Plan& pl, hipStream_t st) {
  return D == 64 ? by_rows<T, 64>(p, c, pl, st) : by_rows<T, 128>(p, c, pl, st);
}

}  // namespace

extern "C" size_t ody_paged_attn_workspace_bytes(int S, int n, int Hq, int Hkv, int D, int page_size, int table_width, int dtype) {
  if (S <= 0 || n <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || page_size <= 0 || table_width <= 0) return 0;   // the call refuses these
  const Plan pl = plan(S, n, Hq / Hkv, Hkv, D, page_size, table_width, dtype);
  return pl.part_bytes + pl.ml_bytes;
}

extern "C" int ody_paged_attn(const void* q, const void* k_pages, const void* v_pages, const int* page_table, const int* lengths, const int* new_tokens, void* out,
                              float* lse, int S, int n, int Hq, int Hkv, int D, int64_t sq_s, int64_t sq_n, int64_t sq_h,
                              int64_t sk_p, int64_t sk_r, int64_t sk_h, int64_t sv_p, int64_t sv_r, int64_t sv_h,
                              int64_t so_s, int64_t so_n, int64_t so_h, int pages, int page_size, int table_width, int64_t table_stride,
                              float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const PagedCache c(const_cast<void*>(k_pages), const_cast<void*>(v_pages), page_table, lengths, new_tokens, {sk_p, sk_r, sk_h}, {sv_p, sv_r, sv_h}, table_stride,
                     pages, page_size, table_width, paged_bytes(dtype));
  if (int rc = paged_check("ody_paged_attn", S, n, Hq, Hkv, D, dtype, paged_bytes(dtype), c, page_size)) return rc;
  ODY_REQUIRE(q && out && lse, ODY_ERR_NULL, "ody_paged_attn: q, out or lse is NULL");
  ODY_REQUIRE(paged_rows_aligned(q, sq_s, sq_n, sq_h, paged_bytes(dtype)) && paged_rows_aligned(out, so_s, so_n, so_h, paged_bytes(dtype)), ODY_ERR_MISALIGNED,
              "ody_paged_attn: q and out need 16-byte aligned pointers and strides");
  const Plan pl = plan(S, n, Hq / Hkv, Hkv, D, page_size, table_width, dtype);
  ODY_REQUIRE(pl.fits, ODY_ERR_BAD_SHAPE, "ody_paged_attn: 2^31 tiles of keys and more, by the table's width");
  ODY_REQUIRE(pl.part_bytes == 0 || (workspace && workspace_bytes >= pl.part_bytes + pl.ml_bytes && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0),
              ODY_ERR_WORKSPACE, "ody_paged_attn: a workspace of %zu bytes, 256-byte aligned, is needed, %zu given", pl.part_bytes + pl.ml_bytes,
              workspace_bytes);
  float* part = static_cast<float*>(workspace);
  const PagedAttnParams p{q, out, lse, {sq_s, sq_n, sq_h}, {so_s, so_n, so_h}, S, n, Hq, Hkv, Hq / Hkv,
                          scale == 0.f ? 1.f : std::fabs(scale) * ODY_LOG2E, scale == 0.f ? 0u : ~0u,
                          scale < 0.f ? (dtype == ODY_BF16 ? 0x80008000u : 0x80000000u) : 0u, pl.row_tiles, pl.tile,
                          part, reinterpret_cast<float2*>(static_cast<char*>(workspace) + pl.part_bytes)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == ODY_BF16 ? by_head_dim<bf16>(p, D, c, pl, st) : by_head_dim<float>(p, D, c, pl, st);
}
