// Attention of new tokens over a key / value cache in pages that holds its values in 8 bits.
//
// The products and their operands are those of paged_attn.hip, and so is the division of the work: nothing but registers lies between memory and the matrix
// cores, and a wavefront takes a tile of keys for all rows of a row tile.  A value is converted where it becomes an operand, to the queries' type and with its
// block's power of two: exactly (paged_q8.h: but for the ends of the type).  Half the bytes make a tile of twice the keys, two sub-tiles of which each is the contraction of one product with V, so that as many bytes
// are under way:
//
//      S^T = K Q^T          A: K rows, 16 columns a lane in 16 bytes, which are the lane's of two products (bf16) or sixteen (fp32); Q^T is read in the same order
//      O^T += V^T P^T       A: V^T, GK rows of DV columns a lane, transposed in its registers   B: P^T = accumulator layout of S^T
//
// A group of GK keys lies within a block, so that a lane needs one scale for its K row and one for its V rows of a sub-tile.
//
// Bound by memory where there is enough: single tokens of 64 sequences of up to 8192 keys, 32 heads on 8 of 128, 96.7 us with the join, 5.6 TB/s (in 16 bits 171 to 196).  One sequence of 8192 11.5 us (13.5), five
// tokens each of eight of up to 5000, 16 heads on 4 of 64, 14.0 (16.7): latencies of the two launches, lengths, table, keys, LDS.
#include <algorithm>
#include <cmath>
#include "paged_join.h"
#include "paged_q8.h"

namespace {

constexpr int WAVES = 4, BLOCKS = 512;
// Sub-tiles of a tile: two, but for 32 rows of heads of 128, where two do not fit the registers.
__host__ __device__ constexpr int subs(int row_tile, int D) { return row_tile == 32 && D == 128 ? 1 : 2; }

template <typename T, int D> struct Sub;   // a sub-tile
template <int D> struct Sub<bf16, D> {
  static constexpr int KEYS = 32, GK = 8, KR = 2;   // keys; keys of a group; K rows a lane
  typedef bf16x8 qvec;
};
template <int D> struct Sub<float, D> {
  static constexpr int KEYS = 16, GK = 4, KR = 1;
  typedef f32x4 qvec;
};
// vector j of the lane's columns of a query: 64 (j / PER) + 16 q + N (j % PER) ..
template <typename T> constexpr int QN = 16 / (int)sizeof(T);
template <typename T> __device__ constexpr int query_col(int q, int j) { return 64 * (j / (16 / QN<T>)) + 16 * q + QN<T> * (j % (16 / QN<T>)); }

// scores of the lane's keys against column c's query row, for all NT
template <int D, int NT>
__device__ __forceinline__ void scores(const u32x4 (&k)[2][D / 64], float scale, const bf16x8 (&qf)[NT][D / 32], float (&x)[NT][8]) {
#pragma unroll
  for (int st = 0; st < 2; st++) {
    f32x4 s[NT];
#pragma unroll
    for (int m = 0; m < NT; m++) s[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < D / 64; j++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const bf16x8 kf = q8_operand(k[st][j][2 * h], k[st][j][2 * h + 1], scale);
#pragma unroll
        for (int m = 0; m < NT; m++) s[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[m][2 * j + h], s[m], 0, 0, 0);
      }
#pragma unroll
    for (int m = 0; m < NT; m++)
#pragma unroll
      for (int r = 0; r < 4; r++) x[m][4 * st + r] = s[m][r];
  }
}
template <int D, int NT>
__device__ __forceinline__ void scores(const u32x4 (&k)[1][D / 64], float scale, const f32x4 (&qf)[NT][D / 16], float (&x)[NT][4]) {
  f32x4 s[NT];
#pragma unroll
  for (int m = 0; m < NT; m++) s[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < D / 64; j++)
#pragma unroll
    for (int w = 0; w < 4; w++) {
      float kf[4];
      q8_values(k[0][j][w], scale, kf);
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int m = 0; m < NT; m++) s[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[m][4 * j + w][e], s[m], 0, 0, 0);
    }
#pragma unroll
  for (int m = 0; m < NT; m++)
#pragma unroll
    for (int r = 0; r < 4; r++) x[m][r] = s[m][r];
}

// o[i], row c: column c * DV + i of the result
template <int D, int NT>
__device__ __forceinline__ void values(const unsigned (&rows)[8][D / 64], float scale, const float (&w)[NT][8], f32x4 (&o)[NT][D / 16]) {
  bf16x8 pb[NT];
#pragma unroll
  for (int m = 0; m < NT; m++)
#pragma unroll
    for (int e = 0; e < 8; e++) pb[m][e] = (bf16)w[m][e];
  unsigned v[8][D / 32];
#pragma unroll
  for (int j = 0; j < 8; j++)
#pragma unroll
    for (int i = 0; i < D / 64; i++) {
      v[j][2 * i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(rows[j][i], scale, false));
      v[j][2 * i + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(rows[j][i], scale, true));
    }
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
__device__ __forceinline__ void values(const unsigned (&rows)[4][D / 64], float scale, const float (&w)[NT][4], f32x4 (&o)[NT][D / 16]) {
#pragma unroll
  for (int r = 0; r < 4; r++)
#pragma unroll
    for (int i = 0; i < D / 64; i++) {
      float vf[4];
      q8_values(rows[r][i], scale, vf);
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int m = 0; m < NT; m++) o[m][4 * i + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[e], w[m][r], o[m][4 * i + e], 0, 0, 0);
    }
}

template <bool STREAM, int WORDS>
__device__ __forceinline__ void load_words(unsigned* to, const uint8_t* from) {
  typedef unsigned raw __attribute__((ext_vector_type(WORDS)));
  raw x;
  if constexpr (STREAM) x = __builtin_nontemporal_load(reinterpret_cast<const raw*>(from));
  else x = *reinterpret_cast<const raw*>(from);
  __builtin_memcpy(to, &x, sizeof(x));
}

// STREAM: keys that one row tile reads take no cache room.
template <typename T, int D, int NT, bool STREAM>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_attn_q8_kernel(const PagedAttnParams p, const PagedCache cache, const PagedScales z) {
  typedef Sub<T, D> G;
  constexpr int SUBS = subs(16 * NT, D), KEYS = SUBS * G::KEYS, STEP = WAVES * KEYS, GK = G::GK, DV = D / 16, QV = D / QN<T> / 4, OP = D + 4;
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
  const unsigned of_lane_k = (c & 3) * cache.k_row + 16 * q, of_lane_v = c * DV;
  PagedPlace<STEP> at(walk, pos, each);

  while (pos < end) {
    const int s = at.s, rt = at.rt, hk = at.hk, length = at.length, step = at.step, steps = at.steps, row0 = rt * p.tile;
    const int rows = min(p.tile, p.n * p.group - row0);
    const int none = p.n - at.fresh;   // the first tokens, which are none
    const int keys = paged_keys(p, cache, length, at.fresh, rt), steps_here = min(steps - step, end - pos);
    const uint8_t* kp = static_cast<const uint8_t*>(cache.k) + hk * cache.sk.h + of_lane_k;
    const uint8_t* vp = static_cast<const uint8_t*>(cache.v) + hk * cache.sv.h + of_lane_v;
    const uint8_t *kz = z.k + hk * z.sk.h, *vz = z.v + hk * z.sv.h;
    const int* table = cache.table + s * cache.table_stride;
    const int in_page = (1 << cache.shift) - 1, last_group = max(keys - 1, 0) & -GK;

    // ---- row 16 m + c: token (row0 + ..) / group, query head hk * group + (row0 + ..) % group
    typename G::qvec qf[NT][QV];
    int lim[NT];   // last key the row sees
    int safe = keys - 1;
#pragma unroll
    for (int m = 0; m < NT; m++) {
      const int r = row0 + min(16 * m + c, rows - 1), i = r / p.group, h = hk * p.group + r - i * p.group;
      const T* qp = static_cast<const T*>(p.q) + s * p.sq.b + i * p.sq.l + h * p.sq.h;
#pragma unroll
      for (int j = 0; j < QV; j++) qf[m][j] = p.signed_query(*reinterpret_cast<const typename G::qvec*>(qp + query_col<T>(q, j)));
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
    const int key0 = step * STEP + wave * KEYS;
    const int tiles = key0 >= keys ? 0 : min(steps_here, (keys - key0 + STEP - 1) / STEP);
    struct Pages { int k[SUBS], v[SUBS]; };
    auto lookup = [&](int t) __attribute__((always_inline)) {   // of the groups that the lane's K rows and V rows are in
      Pages g;
#pragma unroll
      for (int u = 0; u < SUBS; u++) {
        const int base = key0 + min(t, tiles - 1) * STEP + u * G::KEYS;
        g.k[u] = table[min(base + GK * (c >> 2), last_group) >> cache.shift], g.v[u] = table[min(base + GK * q, last_group) >> cache.shift];
      }
      return g;
    };
    struct Loaded {   // a tile's rows
      u32x4 k[SUBS][G::KR][D / 64];
      unsigned v[SUBS][GK][D / 64];
      uint8_t kz[SUBS], vz[SUBS];
      bool page[SUBS];   // the lane's keys, sub-tile + GK q .., have one
    };
    auto load_k = [&](Loaded& to, int t, const Pages& pg) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < SUBS; u++) {
        const int row = min(key0 + t * STEP + u * G::KEYS + GK * (c >> 2), last_group) & in_page, page = (unsigned)pg.k[u] < (unsigned)cache.pages ? pg.k[u] : 0;
        const uint8_t* src = kp + (uint64_t)page * cache.k_page + (unsigned)row * cache.k_row;
        to.kz[u] = kz[page * z.sk.p + (row >> z.shift) * z.sk.r];
#pragma unroll
        for (int j = 0; j < G::KR; j++)
#pragma unroll
          for (int e = 0; e < D / 64; e++) load_words<STREAM, 4>(reinterpret_cast<unsigned*>(&to.k[u][j][e]), src + 4 * j * (uint64_t)cache.k_row + 64 * e);
      }
    };
    auto load_v = [&](Loaded& to, int t, const Pages& pg) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < SUBS; u++) {
        const int row = min(key0 + t * STEP + u * G::KEYS + GK * q, last_group) & in_page;
        to.page[u] = (unsigned)pg.v[u] < (unsigned)cache.pages;
        const int page = to.page[u] ? pg.v[u] : 0;
        const uint8_t* src = vp + (uint64_t)page * cache.v_page + (unsigned)row * cache.v_row;
        to.vz[u] = vz[page * z.sv.p + (row >> z.shift) * z.sv.r];
#pragma unroll
        for (int j = 0; j < GK; j++) load_words<STREAM, D / 64>(to.v[u][j], src + j * (uint64_t)cache.v_row);
      }
    };
    // the products with tile t; `k_read` is called when those with its K have been formed
    auto compute = [&](Loaded& x, int t, auto k_read) __attribute__((always_inline)) {
      const int base = key0 + t * STEP;
      float w[SUBS][NT][GK];
#pragma unroll
      for (int u = 0; u < SUBS; u++) scores<D, NT>(x.k[u], q8_scale(x.kz[u]), qf, w[u]);
      k_read();
      // keys that a row does not see, that no token has, that have no page: neither their scores nor their values count, whatever lies there
      bool all = true;
#pragma unroll
      for (int u = 0; u < SUBS; u++) all = all && x.page[u];
      if (base + KEYS - 1 > safe || !__all(all)) {
#pragma unroll
        for (int u = 0; u < SUBS; u++) {
          const int first = base + u * G::KEYS + GK * q, most = x.page[u] ? keys - 1 : -1;
#pragma unroll
          for (int e = 0; e < GK; e++) {
#pragma unroll
            for (int m = 0; m < NT; m++)
              if (first + e > min(lim[m], most)) w[u][m][e] = -INFINITY;
            if (first + e > most)
#pragma unroll
              for (int i = 0; i < D / 64; i++) x.v[u][e][i] = 0;
          }
          if (first > most) x.vz[u] = 127;   // 0 times what lies in the place of a scale may be no number
        }
      }
#pragma unroll
      for (int m = 0; m < NT; m++) {
        float top = w[0][m][0];
#pragma unroll
        for (int u = 0; u < SUBS; u++)
#pragma unroll
          for (int e = 0; e < GK; e++) top = fmaxf(top, w[u][m][e]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float now = fmaxf(mx[m], top * p.scale_log2e), ref = now == -INFINITY ? 0.f : now, alpha = ody_exp2(mx[m] - ref);
        mx[m] = now;
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < SUBS; u++)
#pragma unroll
          for (int e = 0; e < GK; e++) w[u][m][e] = ody_exp2(fmaf(w[u][m][e], p.scale_log2e, -ref)), sum += w[u][m][e];
        l[m] = l[m] * alpha + sum;   // this lane's share of the row sum
#pragma unroll
        for (int i = 0; i < D / 16; i++) o[m][i] *= alpha;
      }
#pragma unroll
      for (int u = 0; u < SUBS; u++) values<D, NT>(x.v[u], q8_scale(x.vz[u]), w[u], o);
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
          *reinterpret_cast<f32x4*>(&Os[wave][c][(4 * q + r) * DV + i]) = f32x4{o[m][i][r], o[m][i + 1][r], o[m][i + 2][r], o[m][i + 3][r]} * mine;
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

// The host knows no lengths.  Row tiles of 16 or 32 here, the kernels for many rows in bf16 where there is work for them: more than 64 rows, and 2048 in all (32 heads on 8 of 128, us
// here / in tiles of 128: 17 tokens behind 500 keys 12.3 / 18.7, behind 32768 37.8 / 43.4; of 4 sequences, 2176 rows, behind 2000 24.5 / 24.1, behind 8192 41.0 / 41.3; 33 tokens
// behind 2000 16.9 / 22.6; 128 tokens, 4096 rows, behind 2000 31.5 / 25.4, behind 8192 48.8 / 43.4; 10 tokens each of 64 sequences, which are read twice here, of up to 8192 keys
// 209 / 198, of up to 1000 51 / 55).
// Tiles of 256 for heads of 128 by the rule of paged_attn.hip, where 64 of them keep the chip busy and cover few rows more than tiles of 128 (us in tiles of 128 / 256: 128 tokens, which are
// 16 units, behind 2000 keys 25.4 / 29.6; 512 tokens, 64 units, 45.7 / 42.0; 512 behind 32768 337 / 290, 2048 behind 8192 384 / 342, 300 each of 64 sequences of up to 3000
// keys 1424 / 1109; 257 rows of each of 32 heads behind 8192 keys, which are two tiles of 256, 81 / 91).
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
  const bool chunk = dtype == ODY_BF16 && rows > 64 && rows * pairs >= 2048;
  const int64_t wide_tiles = (rows + PAGED_WIDE_ROWS - 1) / PAGED_WIDE_ROWS, chunk_tiles = (rows + PAGED_CHUNK_ROWS - 1) / PAGED_CHUNK_ROWS;
  const bool wide = chunk && D == 128 && pairs * wide_tiles >= 64 && 14 * wide_tiles <= 8 * chunk_tiles;
  const int tile = rows <= 16 ? 16 : wide ? PAGED_WIDE_ROWS : chunk ? PAGED_CHUNK_ROWS : 32, row_tiles = (int)((rows + tile - 1) / tile);
  const int step = chunk ? PAGED_CHUNK_KEYS : WAVES * subs(tile, D) * (dtype == ODY_BF16 ? 32 : 16);
  const int64_t steps = std::max((int64_t)1, (most_keys + step - 1) / step);   // of a unit, at most
  const double all = (double)S * row_tiles * Hkv * (steps + paged_extra(tile));
  const int blocks = (int)std::min((double)(wide ? BLOCKS / 2 : BLOCKS), std::ceil(all / 8) * 8);   // a multiple of 8: paged_range
  const bool joined = steps > 1;
  const size_t parts = joined ? (size_t)blocks * 2 * tile : 0;
  return Plan{tile, row_tiles, step, blocks, joined, all < 2147483648.0, parts * D * sizeof(float), parts * sizeof(float2)};
}

template <typename T, int D, int NT>
int launch(const PagedAttnParams& p, const PagedCache& c, const PagedScales& z, const Plan& pl, hipStream_t st) {
  constexpr bool LINES = D == 128;   // a tile of 16 rows is the only one
  if (NT == 1 || (LINES && pl.row_tiles == 1)) ODY_LAUNCH("paged_attn_q8", st, (paged_attn_q8_kernel<T, D, NT, LINES>), dim3(pl.blocks), dim3(64 * WAVES), 0, p, c, z);
  else ODY_LAUNCH("paged_attn_q8", st, (paged_attn_q8_kernel<T, D, NT, NT == 1 && LINES>), dim3(pl.blocks), dim3(64 * WAVES), 0, p, c, z);
  const int rc = ody_check_launch("paged_attn_q8");
  return rc ? rc : paged_join<T, D, WAVES * subs(16 * NT, D) * Sub<T, D>::KEYS, 1>(p, c, pl.joined, pl.blocks, st);
}
int many_rows(const PagedAttnParams& p, int D, const PagedCache& c, const PagedScales& z, const Plan& pl, hipStream_t st) {
  const int rc = pl.tile == PAGED_WIDE_ROWS ? ody_launch_paged_wide_q8(p, c, z, pl.blocks, st) : ody_launch_paged_chunk_q8(p, D, c, z, pl.blocks, st);
  if (rc) return rc;
  return D == 64 ? paged_join<bf16, 64, PAGED_CHUNK_KEYS, PAGED_JOIN_ROWS>(p, c, pl.joined, pl.blocks, st)
                 : paged_join<bf16, 128, PAGED_CHUNK_KEYS, PAGED_JOIN_ROWS>(p, c, pl.joined, pl.blocks, st);
}
template <typename T>
int by_head_dim(const PagedAttnParams& p, int D, const PagedCache& c, const PagedScales& z, const Plan& pl, hipStream_t st) {
  if (D == 64) return pl.tile == 16 ? launch<T, 64, 1>(p, c, z, pl, st) : launch<T, 64, 2>(p, c, z, pl, st);
  return pl.tile == 16 ? launch<T, 128, 1>(p, c, z, pl, st) : launch<T, 128, 2>(p, c, z, pl, st);
}

}  // namespace

extern "C" size_t ody_paged_attn_q8_workspace_bytes(int S, int n, int Hq, int Hkv, int D, int page_size, int table_width, int dtype) {
  if (S <= 0 || n <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || page_size <= 0 || table_width <= 0) return 0;   // the call refuses these
  const Plan pl = plan(S, n, Hq / Hkv, Hkv, D, page_size, table_width, dtype);
  return pl.part_bytes + pl.ml_bytes;
}

extern "C" int ody_paged_attn_q8(const void* q, const void* k_pages, const void* v_pages, const uint8_t* k_scales, const uint8_t* v_scales, const int* page_table,
                                 const int* lengths, const int* new_tokens, void* out, float* lse, int S, int n, int Hq, int Hkv, int D,
                                 int64_t sq_s, int64_t sq_n, int64_t sq_h, int64_t sk_p, int64_t sk_r, int64_t sk_h, int64_t sv_p, int64_t sv_r, int64_t sv_h,
                                 int64_t skz_p, int64_t skz_b, int64_t skz_h, int64_t svz_p, int64_t svz_b, int64_t svz_h,
                                 int64_t so_s, int64_t so_n, int64_t so_h, int pages, int page_size, int block, int table_width, int64_t table_stride,
                                 float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const PagedCache c(const_cast<void*>(k_pages), const_cast<void*>(v_pages), page_table, lengths, new_tokens, {sk_p, sk_r, sk_h}, {sv_p, sv_r, sv_h}, table_stride,
                     pages, page_size, table_width, 1);
  const PagedScales z{const_cast<uint8_t*>(k_scales), const_cast<uint8_t*>(v_scales), {skz_p, skz_b, skz_h}, {svz_p, svz_b, svz_h}, paged_q8_shift(block)};
  if (int rc = paged_check("ody_paged_attn_q8", S, n, Hq, Hkv, D, dtype, 1, c, page_size)) return rc;
  if (int rc = paged_q8_check("ody_paged_attn_q8", z, page_size, block)) return rc;
  ODY_REQUIRE(q && out && lse, ODY_ERR_NULL, "ody_paged_attn_q8: q, out or lse is NULL");
  const int bytes = paged_bytes(dtype);
  ODY_REQUIRE(paged_rows_aligned(q, sq_s, sq_n, sq_h, bytes) && paged_rows_aligned(out, so_s, so_n, so_h, bytes), ODY_ERR_MISALIGNED,
              "ody_paged_attn_q8: q and out need 16-byte aligned pointers and strides");
  const Plan pl = plan(S, n, Hq / Hkv, Hkv, D, page_size, table_width, dtype);
  ODY_REQUIRE(pl.fits, ODY_ERR_BAD_SHAPE, "ody_paged_attn_q8: 2^31 tiles of keys and more, by the table's width");
  ODY_REQUIRE(pl.part_bytes == 0 || (workspace && workspace_bytes >= pl.part_bytes + pl.ml_bytes && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0),
              ODY_ERR_WORKSPACE, "ody_paged_attn_q8: a workspace of %zu bytes, 256-byte aligned, is needed, %zu given", pl.part_bytes + pl.ml_bytes,
              workspace_bytes);
  float* part = static_cast<float*>(workspace);
  const PagedAttnParams p{q, out, lse, {sq_s, sq_n, sq_h}, {so_s, so_n, so_h}, S, n, Hq, Hkv, Hq / Hkv,
                          scale == 0.f ? 1.f : std::fabs(scale) * ODY_LOG2E, scale == 0.f ? 0u : ~0u,
                          scale < 0.f ? (dtype == ODY_BF16 ? 0x80008000u : 0x80000000u) : 0u, pl.row_tiles, pl.tile,
                          part, reinterpret_cast<float2*>(static_cast<char*>(workspace) + pl.part_bytes)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (pl.tile >= PAGED_CHUNK_ROWS) return many_rows(p, D, c, z, pl, st);
  return dtype == ODY_BF16 ? by_head_dim<bf16>(p, D, c, z, pl, st) : by_head_dim<float>(p, D, c, z, pl, st);
}
