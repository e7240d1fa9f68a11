// Attention of many new tokens over a key / value cache in pages, bf16: a chunk of a prompt, more than 64 rows of a kv head (its query heads
// times the tokens).
//
// Bound by the matrix cores and, as much, by the vector work of the softmax between the two products.  A block of four wavefronts takes 128 rows of one
// (sequence, kv head), 32 a wavefront, and streams the keys in tiles of 64 through LDS, two buffers, the loads a tile ahead and the page numbers
// two.  Both products are computed transposed, so that a row's maximum, sum and rescaling belong to one lane (and the one 32 lanes away):
//
//      S^T (keys x rows) = K Q^T        A: K rows from LDS      B: this lane's query row, in registers
//      O^T (D x rows) += V^T P^T        B: P^T as the accumulators of S^T hold it      A: V^T by transposing LDS reads
//
// on v_mfma_f32_32x32x16_bf16 (lane = 32 g + i: A row i / B column i, k = 8 g .. 8 g + 7; accumulator column i, rows 8 (r / 4) + 4 g + r % 4).
#include <cmath>
#include "paged.h"

namespace {

constexpr int KEYS = PAGED_CHUNK_KEYS, ROWS = PAGED_CHUNK_ROWS;

template <int D>
__global__ __launch_bounds__(256, 2) void paged_chunk_kernel(const PagedAttnParams p, const PagedCache cache) {
  constexpr int KP = D + 8;     // pitches: 16-byte reads of 16 rows, and transposing reads of 4 rows x 32 columns, hit every bank alike
  constexpr int VP = D + 32;
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int CPR = D / 8, RPL = 256 / CPR, LOADS = KEYS / RPL;   // 16-byte chunks of a row, rows of one load of the block
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
  bf16* Ks = reinterpret_cast<bf16*>(smem_raw);            // [2][KEYS][KP]
  bf16* Vs = Ks + 2 * KEYS * KP;                           // [2][KEYS][VP]
  __shared__ __attribute__((aligned(8))) unsigned char paged[2][KEYS / 8];   // the tile's groups of 8 keys that have a page

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 5, i = lane & 31;
  PagedWalk<KEYS> walk(p, cache, lane);
  const PagedCuts cuts(walk.total() * p.Hkv, gridDim.x);
  const int block = blockIdx.x;
  if (block >= cuts.blocks) return;
  const int begin = cuts.at(block), end = cuts.at(block + 1);
  int pos = begin, hk, step, steps, entry = walk.find(pos, hk, step, steps);

  while (pos < end) {
    const int s = p.row_tiles == 1 ? entry : entry / p.row_tiles, rt = entry - s * p.row_tiles, row0 = rt * ROWS;
    const int rows = min(ROWS, p.n * p.group - row0), length = paged_length(cache, s);
    const int keys = paged_keys(p, cache, length, rt), steps_here = min(steps - step, end - pos);
    const bf16* kp = static_cast<const bf16*>(cache.k) + hk * cache.sk.h;
    const bf16* vp = static_cast<const bf16*>(cache.v) + hk * cache.sv.h;
    const int* table = cache.table + s * cache.table_stride;

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
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int e = 0; e < 16; e++) o[dt][e] = 0.f;

    // ---- loads: row tid / CPR + RPL j of a tile, 16 bytes at column 8 (tid % CPR)
    const int lr = tid / CPR, lc = tid % CPR * 8;
    int pg[LOADS];
    bf16x8 kr[LOADS], vr[LOADS];
    unsigned has;   // bit j: row j's page is one
    auto lookup = [&](int t) {
#pragma unroll
      for (int j = 0; j < LOADS; j++) pg[j] = table[max(0, min((step + t) * KEYS + lr + RPL * j, keys - 1)) >> cache.shift];
    };
    auto load = [&](int t) {
      has = 0;
#pragma unroll
      for (int j = 0; j < LOADS; j++) {
        const int key = (step + t) * KEYS + lr + RPL * j, row = key & ((1 << cache.shift) - 1);
        const bool ok = (unsigned)pg[j] < (unsigned)cache.pages;
        has |= (unsigned)ok << j;
        if (ok && key < keys) {
          kr[j] = *reinterpret_cast<const bf16x8*>(kp + pg[j] * cache.sk.p + row * cache.sk.r + lc);
          vr[j] = *reinterpret_cast<const bf16x8*>(vp + pg[j] * cache.sv.p + row * cache.sv.r + lc);
        } else {
          kr[j] = vr[j] = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
        }
      }
    };
    auto store = [&](int buf) {
#pragma unroll
      for (int j = 0; j < LOADS; j++) {
        *reinterpret_cast<bf16x8*>(Ks + (buf * KEYS + lr + RPL * j) * KP + lc) = kr[j];
        *reinterpret_cast<bf16x8*>(Vs + (buf * KEYS + lr + RPL * j) * VP + lc) = vr[j];
        if (lc == 0 && (lr + RPL * j) % 8 == 0) paged[buf][(lr + RPL * j) / 8] = has >> j & 1;
      }
    };
    const int tiles = keys > 0 ? steps_here : 0;
    if (tiles > 0) {
      lookup(0);
      load(0);
      lookup(1);
      store(0);
    }
    __syncthreads();

    const int tr_row = (i & 15) >> 2, tr_col = 16 * (i >> 4) + 4 * (i & 3);   // of a transposing read, within 16 lanes
    for (int t = 0; t < tiles; t++) {
      const int buf = t & 1, n0 = (step + t) * KEYS;
      if (t + 1 < tiles) {
        load(t + 1);
        lookup(t + 2);
      }
      if (n0 <= seen) {
        const bf16* Kb = Ks + buf * KEYS * KP;
        const bf16* Vb = Vs + buf * KEYS * VP;
        f32x16 x[2];
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
#pragma unroll
          for (int e = 0; e < 16; e++) x[kt][e] = 0.f;
#pragma unroll
          for (int ks = 0; ks < KS; ks++) x[kt] = mfma32(*reinterpret_cast<const bf16x8*>(Kb + (32 * kt + i) * KP + 16 * ks + 8 * g), qf[ks], x[kt]);
        }
        const uint64_t have = *reinterpret_cast<const uint64_t*>(paged[buf]);
        if (n0 + KEYS - 1 > safe || !__all(have == 0x0101010101010101ull)) {
#pragma unroll
          for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
              const int group = 4 * kt + (e >> 2);
              if (n0 + 8 * group + 4 * g + (e & 3) > lim || (have >> (8 * group) & 1) == 0) x[kt][e] = -INFINITY;
            }
        }
        float top = x[0][0];
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
          for (int e = 0; e < 16; e++) top = fmaxf(top, x[kt][e]);
        top = fmaxf(top, xor32(top)) * p.scale_log2e;
        const float now = fmaxf(m, top), ref = now == -INFINITY ? 0.f : now;
        if (!__all(now == m)) {   // somebody's maximum has grown
          const float alpha = ody_exp2(m - ref);
          l *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[dt][e] *= alpha;
        }
        m = now;
        bf16x8 pb[2][2];
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
          for (int e = 0; e < 16; e++) {
            const float w = ody_exp2(fmaf(x[kt][e], p.scale_log2e, -ref));
            l += w;
            pb[kt][e / 8][e % 8] = (bf16)w;
          }
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
          for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int ss = 0; ss < 2; ss++) {
              const bf16* va = Vb + (32 * kt + 16 * ss + 4 * g + tr_row) * VP + 32 * dt + tr_col;
              o[dt] = mfma32(concat4(lds_read_tr16(va), lds_read_tr16(va + 8 * VP)), pb[kt][ss], o[dt]);
            }
      }
      if (t + 1 < tiles) store(buf ^ 1);
      __syncthreads();
    }

    // ---- o[dt][4 a + e] of this lane's row: column 32 dt + 8 a + 4 g + e
    const float sum = l + xor32(l);
    const bool whole = steps_here == steps;
    if (32 * wave + i < rows) {
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        bf16* dst = static_cast<bf16*>(p.out) + s * p.so.b + ri * p.so.l + h * p.so.h + 4 * g;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
          for (int a = 0; a < 4; a++) {
            bf16x4 w;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = (bf16)(o[dt][4 * a + e] * inv);
            *reinterpret_cast<bf16x4*>(dst + 32 * dt + 8 * a) = w;
          }
        if (g == 0) p.lse[((int64_t)s * p.Hq + h) * p.n + ri] = sum == 0.f ? -INFINITY : (m + __log2f(sum)) * ODY_LN2;
      } else {
        const int64_t at = (int64_t)(2 * block + (pos > begin)) * ROWS + 32 * wave + i;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
          for (int a = 0; a < 4; a++)
            *reinterpret_cast<f32x4*>(p.part + at * D + 32 * dt + 8 * a + 4 * g) = f32x4{o[dt][4 * a], o[dt][4 * a + 1], o[dt][4 * a + 2], o[dt][4 * a + 3]};
        if (g == 0) p.part_ml[at] = make_float2(m, sum);
      }
    }
    pos += steps_here;
    step = 0;
    if (++hk == p.Hkv && pos < end) hk = 0, steps = paged_steps<KEYS>(p, cache, ++entry);
  }
}

template <int D>
int launch(const PagedAttnParams& p, const PagedCache& c, int blocks, hipStream_t st) {
  constexpr size_t smem = (size_t)2 * KEYS * ((D + 8) + (D + 32)) * sizeof(bf16);
  if (int rc = ody_allow_dynamic_lds(reinterpret_cast<const void*>(&paged_chunk_kernel<D>), smem, "ody_paged_attn")) return rc;
  ODY_LAUNCH("paged_chunk", st, (paged_chunk_kernel<D>), dim3(blocks), dim3(256), smem, p, c);
  return ody_check_launch("paged_chunk");
}

}  // namespace

int ody_launch_paged_chunk(const PagedAttnParams& p, int D, const PagedCache& c, int blocks, hipStream_t st) {
  return D == 64 ? launch<64>(p, c, blocks, st) : launch<128>(p, c, blocks, st);
}
