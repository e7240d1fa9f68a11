// New tokens into a key / value cache in pages that holds its values in 8 bits, and what such a cache holds back out of it.
#include <algorithm>
#include <cmath>
#include "paged_q8.h"

namespace {

struct AppendParams {
  const void* x;        // (S, n, Hq + 2 Hkv, D): the packed projection
  void* q;              // (S, n, Hq, D), or null: nothing is rotated, and the queries stay where they are
  const int64_t* pos;   // (S, n), or null: the tokens' places in their sequences
  const float* inv_freq;
  AttnStrides sx, sq;
  int S, n, Hq, Hkv;
  int blocks;           // of a sequence that n tokens may reach
};

template <bool PAST, typename V> __device__ __forceinline__ V load(const void* from) {   // 16 bytes; PAST the caches
  typedef unsigned raw __attribute__((ext_vector_type(4)));
  if constexpr (PAST) return __builtin_bit_cast(V, __builtin_nontemporal_load(static_cast<const raw*>(from)));
  else return *static_cast<const V*>(from);
}
template <typename T> __device__ __forceinline__ float rounded(float x) { return (float)(T)x; }

// x1 c - x2 s and x2 c + x1 s, rounded once to 32 bits: the products of bf16 are exact there, those of fp32 in 64.
__device__ __forceinline__ void rotate(bf16 x1, bf16 x2, float c, float s, float& a, float& b) {
  a = (float)x1 * c - (float)x2 * s;
  b = (float)x2 * c + (float)x1 * s;
}
__device__ __forceinline__ void rotate(float x1, float x2, float c, float s, float& a, float& b) {
  a = (float)((double)x1 * c - (double)x2 * s);
  b = (float)((double)x2 * c + (double)x1 * s);
}

// The least e from -126 on with top <= 448 * 2^e = 1.75 * 2^(8 + e), for a finite top: from its bits.
__device__ __forceinline__ int exponent_of(float top) {
  const unsigned bits = __builtin_bit_cast(unsigned, top);
  return max(-126, (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000));
}
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}
// Eight values to e4m3, to the nearest, half way to the even one; what is not finite becomes its one NaN.
__device__ __forceinline__ unsigned four(const float* x, int e) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(x[0], -e), ldexpf(x[1], -e), 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(x[2], -e), ldexpf(x[3], -e), lo, true);
}
__device__ __forceinline__ unsigned rescaled(unsigned word, int down) {   // times 2^-down
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(word, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
  const float x[4] = {a[0], a[1], b[0], b[1]};
  return four(x, down);
}

// A block of threads takes the new tokens of one block of one sequence (blockIdx.x) and a share of their heads (blockIdx.y): it evaluates the tokens' angles, which go to
// LDS, and its wavefronts take heads in turn, keys and values first.  ROWS rows of a head lie in a wavefront at once, LANES lanes on a row, of which each has
// x[j] together with x[j + D / 2].  A unit -- the keys or the values of a head -- is read once into registers, its largest value found, its scale set, its rows written; where the block
// holds earlier tokens and the scale rises, their rows are rounded to the new one (by powers of two: only values that fall below 2^-6 of the scale change).
// ONE token a sequence: ROWS heads in a wavefront at once, each LANES lanes with a scale of their own.
//
// Bound by memory: four prompts of 2500 to 4096 tokens, 32 heads on 32 of 128, 137 us for 580 MB, 4.2 TB/s (a copy 5.1; with one row of queries a thread under way 10 more).  Angles, which each share of the heads
// evaluates for itself, do not show (a shorter evaluation left the time as it was).  Few tokens by latencies: 64 single ones, 32 heads on 8, 4.6 us.
template <typename T, int D, int BLOCK, bool ROTATE, bool ONE, bool PAST>
__global__ __launch_bounds__(256) void paged_append_q8_kernel(const AppendParams p, const PagedCache cache, const PagedScales z) {
  constexpr int N = Vec16B<T>::N, HALF = D / 2, LANES = HALF / N, ROWS = 64 / LANES, TURNS = ONE ? 1 : (BLOCK + ROWS - 1) / ROWS;
  constexpr int TOKENS = ONE ? 1 : BLOCK;
  typedef typename Vec16B<T>::type vec;
  typedef unsigned raw __attribute__((ext_vector_type(4)));
  __shared__ __attribute__((aligned(16))) float cs[TOKENS][HALF], sn[TOKENS][HALF];
  const int s = blockIdx.x / p.blocks, tid = threadIdx.x, lane = tid & 63, sub = lane / LANES, col = lane % LANES * N;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) + 4 * blockIdx.y, waves = 4 * gridDim.y;
  const int length = paged_length(cache, s), fresh = paged_fresh(cache, s, p.n);
  const int first = length - p.n;                                                       // place of token 0, which may be negative
  const int start = ((first >> z.shift) + (int)(blockIdx.x - s * p.blocks)) << z.shift;   // the block's first place
  const int i0 = max(0, start - first), tokens = min(p.n, start + BLOCK - first) - i0;
  if (tokens <= 0) return;
  // tokens i0 .. i0 + tokens; from token `real` on they are tokens
  const int real = max(p.n - fresh, -first) - i0, since = max(length - min(fresh, length), max(start, 0));   // first new place of the block
  const T* x = static_cast<const T*>(p.x) + s * p.sx.b + i0 * p.sx.l + col;

  if (ROTATE) {
    for (int k = tid; k < tokens * HALF; k += 256) {
      const int t = k / HALF, j = k % HALF;
      const float at = p.pos ? (float)p.pos[(int64_t)s * p.n + i0 + t] : (float)(first + i0 + t), th = at * p.inv_freq[j];
      // rounded to the values' type before use, as ody_rope has them; from 64 bits, for a key on a border of its eight bits would show which way a cosine went
      double sine, cosine;
      sincos((double)th, &sine, &cosine);
      float c = (float)cosine, si = (float)sine;
      asm("" : "+v"(c), "+v"(si));   // of 32 bits first: the compiler makes one rounding of the two, which differs at ties
      cs[t][j] = rounded<T>(c), sn[t][j] = rounded<T>(si);
    }
  }

  // ---- keys and values
  int page = -1;
  if (start >= 0 && start >> cache.shift < cache.width) page = cache.table[s * cache.table_stride + (start >> cache.shift)];
  const int row0 = start & ((1 << cache.shift) - 1);   // of the block in its page
  const bool there = (unsigned)page < (unsigned)cache.pages && real < tokens;
  __syncthreads();
  const int units = 2 * p.Hkv, turn = ONE ? ROWS : 1;
  for (int first_unit = wave * turn; there && first_unit < units; first_unit += waves * turn) {
    const int unit = ONE ? first_unit + sub : first_unit;
    const bool mine = unit < units, key = unit < p.Hkv;
    const int head = key ? unit : unit - p.Hkv;
    uint8_t* byte = (key ? z.k : z.v) + page * (key ? z.sk : z.sv).p + (row0 >> z.shift) * (key ? z.sk : z.sv).r + head * (key ? z.sk : z.sv).h;
    const int before = mine && since > start ? (int)*byte - 127 : -128;
    vec a[TURNS], b[TURNS];
    float top = 0.f;
    auto turned = [&](int k, int t, float (&u)[N], float (&v)[N]) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < N; e++) {
        u[e] = (float)a[k][e], v[e] = (float)b[k][e];
        if (ROTATE && key) rotate(a[k][e], b[k][e], cs[t][col + e], sn[t][col + e], u[e], v[e]);
      }
    };
#pragma unroll
    for (int k = 0; k < TURNS; k++) {
      const int t = ONE ? 0 : k * ROWS + sub;
      a[k] = b[k] = vec{};
      if (mine && t >= real && t < tokens) {
        const T* src = x + t * p.sx.l + (p.Hq + unit) * p.sx.h;
        a[k] = load<PAST, vec>(src), b[k] = load<PAST, vec>(src + HALF);
      }
    }
#pragma unroll
    for (int k = 0; k < TURNS; k++) {
      const int t = ONE ? 0 : k * ROWS + sub;
      if (mine && t >= real && t < tokens) {
        float u[N], v[N];
        turned(k, t, u, v);
#pragma unroll
        for (int e = 0; e < N; e++) top = fmaxf(top, fmaxf(finite_abs(u[e]), finite_abs(v[e])));
      }
    }
#pragma unroll
    for (int d = 1; d < (ONE ? LANES : 64); d *= 2) top = fmaxf(top, __shfl_xor(top, d, 64));
    const int e = max(before, exponent_of(top));
    uint8_t* rows = static_cast<uint8_t*>(key ? cache.k : cache.v) + page * (key ? cache.sk : cache.sv).p + head * (key ? cache.sk : cache.sv).h;
    const int64_t pitch = (key ? cache.sk : cache.sv).r;
    if (mine) {
#pragma unroll
      for (int k = 0; k < TURNS; k++) {
        const int t = ONE ? 0 : k * ROWS + sub;
        if (t < real || t >= tokens) continue;
        float u[N], v[N];
        turned(k, t, u, v);
        uint8_t* dst = rows + (row0 + first + i0 + t - start) * pitch + col;
        if constexpr (N == 8) {
          *reinterpret_cast<u32x2*>(dst) = u32x2{four(u, e), four(u + 4, e)};
          *reinterpret_cast<u32x2*>(dst + HALF) = u32x2{four(v, e), four(v + 4, e)};
        } else {
          *reinterpret_cast<unsigned*>(dst) = four(u, e);
          *reinterpret_cast<unsigned*>(dst + HALF) = four(v, e);
        }
      }
      if (since > start && e > before) {
        typedef unsigned piece __attribute__((ext_vector_type(D / LANES / 4)));
        for (int r = ONE ? 0 : sub; r < since - start; r += ONE ? 1 : ROWS) {
          piece* at = reinterpret_cast<piece*>(rows + (row0 + r) * pitch) + lane % LANES;
          piece w = *at;
#pragma unroll
          for (int i = 0; i < D / LANES / 4; i++) w[i] = rescaled(w[i], e - before);
          *at = w;
        }
      }
      if (ONE ? lane % LANES == 0 : lane == 0) *byte = (uint8_t)(e + 127);
    }
  }

  // ---- queries: rows (token, head), heads in a row
  if (!ROTATE) return;
  constexpr int AHEAD = ONE ? 1 : 4;   // rows of a thread under way
  const int rows = tokens * p.Hq;
  for (int r0 = wave * ROWS + sub; r0 < rows; r0 += AHEAD * waves * ROWS) {
    vec a[AHEAD], b[AHEAD];
    int t[AHEAD], h[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; k++) {
      const int r = r0 + k * waves * ROWS;
      t[k] = ONE ? 0 : r / p.Hq, h[k] = r - t[k] * p.Hq;
      a[k] = b[k] = vec{};
      if (r < rows && t[k] >= real) {
        const T* src = x + t[k] * p.sx.l + h[k] * p.sx.h;
        a[k] = load<PAST, vec>(src), b[k] = load<PAST, vec>(src + HALF);
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; k++) {
      if (r0 + k * waves * ROWS >= rows) break;
      T* dst = static_cast<T*>(p.q) + s * p.sq.b + (i0 + t[k]) * p.sq.l + h[k] * p.sq.h + col;
      vec a1{}, b1{};
      if (t[k] >= real) {
#pragma unroll
        for (int e = 0; e < N; e++) {
          const float c = cs[t[k]][col + e], sine = sn[t[k]][col + e], x1 = (float)a[k][e], x2 = (float)b[k][e];
          a1[e] = (T)(x1 * c - x2 * sine);
          b1[e] = (T)(x2 * c + x1 * sine);
        }
      }
      __builtin_nontemporal_store(__builtin_bit_cast(raw, a1), reinterpret_cast<raw*>(dst));
      __builtin_nontemporal_store(__builtin_bit_cast(raw, b1), reinterpret_cast<raw*>(dst + HALF));
    }
  }
}

template <typename T, int D, int BLOCK>
int launch(const AppendParams& p, const PagedCache& c, const PagedScales& z, hipStream_t st) {
  // shares of the heads: enough blocks for the chip, and something to do for each of their wavefronts
  constexpr int LANES = D / 2 / Vec16B<T>::N, ROWS = 64 / LANES;
  const int64_t groups = (int64_t)p.S * p.blocks, tokens = std::min(p.n, BLOCK);
  const int64_t turns = (p.q ? (tokens * p.Hq + ROWS - 1) / ROWS : 0) + (p.n == 1 ? (2 * p.Hkv + ROWS - 1) / ROWS : 2 * p.Hkv);
  const unsigned shares = (unsigned)std::max((int64_t)1, std::min({(turns + 3) / 4, (2048 + groups - 1) / groups, (int64_t)65535}));
  const dim3 grid((unsigned)groups, shares);
  // A projection that the last-level cache (256 MB) does not hold along with what else a layer touches is read past the caches, which keep the new rows for who reads them next; a smaller
  // one lies there (1324 tokens of 8 MB 11.6 -> 12.7 us so).  Behind the product that writes it, through / past the caches: 402 MB 150.9 / 130.4, 201 MB 76.4 / 73.5, 132 MB 52.0 / 51.7.  Not where half a row,
  // which a load of several rows takes, is half a line (heads of 64 in bf16, 201 MB: 73.2 / 95.4, each line comes twice).  What is not rotated is read by attention next: past the caches only where they
  // have none of it then (with reading it once more, 201 MB 123.9 / 129.5, 255 MB 154.3 / 161.6, 294 MB 205.7 / 206.9, 402 MB 287.7 / 282.6).
  constexpr bool LINES = D / 2 * sizeof(T) >= 128;
  const bool past = LINES && (double)p.S * p.n * (p.Hq + 2 * p.Hkv) * D * sizeof(T) >= (p.q ? 128e6 : 268e6);
#define LAUNCH(R, O, P) ODY_LAUNCH("paged_append_q8", st, (paged_append_q8_kernel<T, D, BLOCK, R, O, P>), grid, dim3(256), 0, p, c, z)
  if (p.n == 1) {
    if (p.q) LAUNCH(true, true, false);
    else LAUNCH(false, true, false);
  } else if (past) {
    if (p.q) LAUNCH(true, false, LINES);
    else LAUNCH(false, false, LINES);
  } else {
    if (p.q) LAUNCH(true, false, false);
    else LAUNCH(false, false, false);
  }
#undef LAUNCH
  return ody_check_launch("paged_append_q8");
}
template <typename T, int D>
int by_block(const AppendParams& p, const PagedCache& c, const PagedScales& z, hipStream_t st) {
  switch (z.shift) {
    case 3: return launch<T, D, 8>(p, c, z, st);
    case 4: return launch<T, D, 16>(p, c, z, st);
    case 5: return launch<T, D, 32>(p, c, z, st);
    default: return launch<T, D, 64>(p, c, z, st);
  }
}

// ---- what the cache holds: a thread takes the keys and the values that make 16 bytes, so that a wavefront writes whole lines; consecutive threads the columns of a head, heads, places.  Memory is all of it:
// 16 sequences of up to 4001 tokens, 16 heads of 64, 45 us for 335 MB, 7.4 TB/s, of which 262 written past the caches (62 through them); in fp32 89 (eight values a
// thread, of which either half of a line is a store: 244, and 139 through the caches); one of 8191, 8 heads of 128, 7.3 us, in fp32 13
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_read_q8_kernel(T* k, T* v, const PagedCache cache, const PagedScales z, int places, int Hkv, int S) {
  constexpr int N = 16 / (int)sizeof(T), LANES = D / N;
  typedef unsigned piece __attribute__((ext_vector_type(N / 4)));
  const int64_t per_sequence = (int64_t)places * Hkv * LANES;
  const int s = blockIdx.y;
  const int length = paged_length(cache, s);
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < per_sequence; at += (int64_t)gridDim.x * 256) {
    const int row = (int)(at / LANES), col = (int)(at % LANES) * N, place = row / Hkv, h = row - place * Hkv;
    int page = -1;
    if (place < length && place >> cache.shift < cache.width) page = cache.table[s * cache.table_stride + (place >> cache.shift)];
    T a[N] = {}, b[N] = {};
    if ((unsigned)page < (unsigned)cache.pages) {
      const int r = place & ((1 << cache.shift) - 1);
      const piece kw = *reinterpret_cast<const piece*>(static_cast<const uint8_t*>(cache.k) + page * cache.sk.p + r * cache.sk.r + h * cache.sk.h + col);
      const piece vw = *reinterpret_cast<const piece*>(static_cast<const uint8_t*>(cache.v) + page * cache.sv.p + r * cache.sv.r + h * cache.sv.h + col);
      const float ks = q8_scale(z.k[page * z.sk.p + (r >> z.shift) * z.sk.r + h * z.sk.h]), vs = q8_scale(z.v[page * z.sv.p + (r >> z.shift) * z.sv.r + h * z.sv.h]);
#pragma unroll
      for (int e = 0; e < N / 4; e++) q8_values(kw[e], ks, a + 4 * e), q8_values(vw[e], vs, b + 4 * e);
    }
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, a), reinterpret_cast<u32x4*>(k) + s * per_sequence + at);
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, b), reinterpret_cast<u32x4*>(v) + s * per_sequence + at);
  }
}

template <typename T, int D>
int launch_read(void* k, void* v, const PagedCache& c, const PagedScales& z, int S, int places, int Hkv, hipStream_t st) {
  const int64_t blocks = ((int64_t)places * Hkv * (D * sizeof(T) / 16) + 255) / 256;
  const dim3 grid((unsigned)std::min(blocks, (int64_t)1 << 16), (unsigned)S);
  ODY_LAUNCH("paged_read_q8", st, (paged_read_q8_kernel<T, D>), grid, dim3(256), 0, static_cast<T*>(k), static_cast<T*>(v), c, z, places, Hkv, S);
  return ody_check_launch("paged_read_q8");
}

}  // namespace

int paged_q8_check(const char* who, const PagedScales& z, int page_size, int block) {
  ODY_REQUIRE(z.k && z.v, ODY_ERR_NULL, "%s: k_scales or v_scales is NULL", who);
  ODY_REQUIRE(block >= 8 && block <= 64 && (block & (block - 1)) == 0 && block <= page_size, ODY_ERR_UNSUPPORTED,
              "%s: a scale for each %d tokens: a power of two from 8 to 64, at most a page", who, block);
  return ODY_OK;
}

extern "C" int ody_paged_append_q8(const void* qkv, void* q, void* k_pages, void* v_pages, uint8_t* k_scales, uint8_t* v_scales, const int* page_table, const int* lengths,
                                   const int* new_tokens, const int64_t* position_ids, const float* inv_freq, int S, int n, int Hq, int Hkv, int D,
                                   int64_t sx_s, int64_t sx_n, int64_t sx_h, int64_t sq_s, int64_t sq_n, int64_t sq_h,
                                   int64_t sk_p, int64_t sk_r, int64_t sk_h, int64_t sv_p, int64_t sv_r, int64_t sv_h,
                                   int64_t skz_p, int64_t skz_b, int64_t skz_h, int64_t svz_p, int64_t svz_b, int64_t svz_h,
                                   int pages, int page_size, int block, int table_width, int64_t table_stride, int dtype, void* stream) {
  const char* who = "ody_paged_append_q8";
  const PagedCache c(k_pages, v_pages, page_table, lengths, new_tokens, {sk_p, sk_r, sk_h}, {sv_p, sv_r, sv_h}, table_stride, pages, page_size, table_width, 1);
  const PagedScales z{k_scales, v_scales, {skz_p, skz_b, skz_h}, {svz_p, svz_b, svz_h}, paged_q8_shift(block)};
  if (int rc = paged_check(who, S, n, Hq, Hkv, D, dtype, 1, c, page_size)) return rc;
  if (int rc = paged_q8_check(who, z, page_size, block)) return rc;
  ODY_REQUIRE((int64_t)S * n < (int64_t)1 << 24, ODY_ERR_BAD_SHAPE, "%s: 2^24 new tokens and more", who);
  const int64_t blocks = ((int64_t)n - 1 + block - 1) / block + 1;   // that n tokens may reach
  ODY_REQUIRE(S * blocks < (int64_t)1 << 23, ODY_ERR_BAD_SHAPE, "%s: 2^23 blocks of new tokens and more", who);
  ODY_REQUIRE(qkv && (q == nullptr || inv_freq), ODY_ERR_NULL, "%s: qkv, or inv_freq of a rotation, is NULL", who);
  const int bytes = paged_bytes(dtype);
  ODY_REQUIRE(paged_rows_aligned(qkv, sx_s, sx_n, sx_h, bytes) && (q == nullptr || paged_rows_aligned(q, sq_s, sq_n, sq_h, bytes)), ODY_ERR_MISALIGNED,
              "%s: qkv and q need 16-byte aligned pointers and strides", who);
  const AppendParams p{qkv, q, position_ids, inv_freq, {sx_s, sx_n, sx_h}, {sq_s, sq_n, sq_h}, S, n, Hq, Hkv, (int)blocks};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == ODY_BF16) return D == 64 ? by_block<bf16, 64>(p, c, z, st) : by_block<bf16, 128>(p, c, z, st);
  return D == 64 ? by_block<float, 64>(p, c, z, st) : by_block<float, 128>(p, c, z, st);
}

extern "C" int ody_paged_read_q8(const void* k_pages, const void* v_pages, const uint8_t* k_scales, const uint8_t* v_scales, const int* page_table, const int* lengths,
                                 void* k, void* v, int S, int places, int Hkv, int D, int64_t sk_p, int64_t sk_r, int64_t sk_h, int64_t sv_p, int64_t sv_r, int64_t sv_h,
                                 int64_t skz_p, int64_t skz_b, int64_t skz_h, int64_t svz_p, int64_t svz_b, int64_t svz_h,
                                 int pages, int page_size, int block, int table_width, int64_t table_stride, int dtype, void* stream) {
  const char* who = "ody_paged_read_q8";
  const PagedCache c(const_cast<void*>(k_pages), const_cast<void*>(v_pages), page_table, lengths, nullptr, {sk_p, sk_r, sk_h}, {sv_p, sv_r, sv_h}, table_stride, pages,
                     page_size, table_width, 1);
  const PagedScales z{const_cast<uint8_t*>(k_scales), const_cast<uint8_t*>(v_scales), {skz_p, skz_b, skz_h}, {svz_p, svz_b, svz_h}, paged_q8_shift(block)};
  if (int rc = paged_check(who, S, 1, Hkv, Hkv, D, dtype, 1, c, page_size)) return rc;
  if (int rc = paged_q8_check(who, z, page_size, block)) return rc;
  ODY_REQUIRE(places > 0 && (int64_t)places * Hkv < (int64_t)1 << 31, ODY_ERR_BAD_SHAPE, "%s: %d places of %d heads", who, places, Hkv);
  ODY_REQUIRE(S < 65536, ODY_ERR_BAD_SHAPE, "%s: %d sequences, 65535 at most", who, S);
  ODY_REQUIRE(k && v, ODY_ERR_NULL, "%s: k or v is NULL", who);
  ODY_REQUIRE(ody_aligned16(k) && ody_aligned16(v), ODY_ERR_MISALIGNED, "%s: k and v need 16-byte aligned pointers", who);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == ODY_BF16) return D == 64 ? launch_read<bf16, 64>(k, v, c, z, S, places, Hkv, st) : launch_read<bf16, 128>(k, v, c, z, S, places, Hkv, st);
  return D == 64 ? launch_read<float, 64>(k, v, c, z, S, places, Hkv, st) : launch_read<float, 128>(k, v, c, z, S, places, Hkv, st);
}
