// New tokens into a key / value cache in pages, their queries and keys rotated on the way.
#include <algorithm>
#include <cmath>
#include "paged.h"

namespace {

struct AppendParams {
  const void* x;        // (S, n, Hq + 2 Hkv, D): the packed projection
  void* q;              // (S, n, Hq, D), or null: nothing is rotated, and the queries stay where they are
  const int64_t* pos;   // (S, n), or null: the tokens' places in their sequences
  const float* inv_freq;
  AttnStrides sx, sq;
  int S, n, Hq, Hkv;
};

template <typename T> __device__ __forceinline__ float rounded(float x) { return (float)(T)x; }

// A block takes a token: consecutive threads take consecutive vectors of a head, x[j] together with x[j + D / 2].  Bound by memory, or for few tokens by
// latencies: a thread's first vectors are under way while the block evaluates the token's angles, which go to LDS (64 tokens of 48 heads 3.8 -> 3.2 us,
// launch included).  Results leave without taking cache room (3001 tokens of 48 heads 15.5 -> 12.7 us), and operands that the last-level cache cannot hold
// beside them are read past it (STREAM; 4 x 4096 tokens of 96 heads 141 -> 135 us, 5.0 TB/s; 3001 of 48 12.7 -> 14.3).  A token that is none: its
// queries become 0, nothing else is written.
template <typename T, int D, bool ROTATE, bool STREAM>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendParams p, const PagedCache cache) {
  constexpr int N = Vec16B<T>::N, HALF = D / 2, VECS = HALF / N;
  typedef typename Vec16B<T>::type vec;
  typedef unsigned raw __attribute__((ext_vector_type(4)));
  __shared__ __attribute__((aligned(16))) float cs[HALF], sn[HALF];
  const int token = blockIdx.x, s = token / p.n, i = token - s * p.n, tid = threadIdx.x;
  const int h0 = ROTATE ? 0 : p.Hq, items = (p.Hq + 2 * p.Hkv - h0) * VECS;   // pairs of vectors
  const T* x = static_cast<const T*>(p.x) + s * p.sx.b + i * p.sx.l + h0 * p.sx.h;
  auto load = [&](int v, vec& a, vec& b) {
    const T* src = x + v / VECS * p.sx.h + v % VECS * N;
    if (STREAM) {
      a = __builtin_bit_cast(vec, __builtin_nontemporal_load(reinterpret_cast<const raw*>(src)));
      b = __builtin_bit_cast(vec, __builtin_nontemporal_load(reinterpret_cast<const raw*>(src + HALF)));
    } else {
      a = *reinterpret_cast<const vec*>(src);
      b = *reinterpret_cast<const vec*>(src + HALF);
    }
  };
  vec a, b;
  if (tid < items) load(tid, a, b);
  const int place = i < p.n - paged_fresh(cache, s, p.n) ? -1 : max(cache.lengths[s], 0) - p.n + i;
  // where the token's keys and values go
  int page = -1;
  if (place >= 0 && place >> cache.shift < cache.width) page = cache.table[s * cache.table_stride + (place >> cache.shift)];
  const bool paged = (unsigned)page < (unsigned)cache.pages;
  const int row = place & ((1 << cache.shift) - 1);
  if (ROTATE) {
    if (tid < HALF) {
      const float pos = p.pos ? (float)p.pos[token] : (float)place, th = pos * p.inv_freq[tid];
      cs[tid] = rounded<T>(cosf(th));   // rounded to the values' type before use, as ody_rope has them
      sn[tid] = rounded<T>(sinf(th));
    }
    __syncthreads();
  }
  for (int v = tid; v < items; v += 256) {
    const int j = v % VECS * N, h = h0 + v / VECS;
    if (v != tid) load(v, a, b);
    T* dst;
    if (h < p.Hq) {
      dst = static_cast<T*>(p.q) + s * p.sq.b + i * p.sq.l + h * p.sq.h + j;
      if (place < 0) a = b = vec{};
    } else {
      if (!paged) continue;
      const bool key = h < p.Hq + p.Hkv;
      const PageStrides& st = key ? cache.sk : cache.sv;
      dst = static_cast<T*>(key ? cache.k : cache.v) + page * st.p + row * st.r + (h - p.Hq - (key ? 0 : p.Hkv)) * st.h + j;
    }
    if (ROTATE && h < p.Hq + p.Hkv) {
      vec a1, b1;
#pragma unroll
      for (int e = 0; e < N; e++) {
        const float c = cs[j + e], sine = sn[j + e], x1 = (float)a[e], x2 = (float)b[e];
        a1[e] = (T)(x1 * c - x2 * sine);
        b1[e] = (T)(x2 * c + x1 * sine);
      }
      a = a1, b = b1;
    }
    __builtin_nontemporal_store(__builtin_bit_cast(raw, a), reinterpret_cast<raw*>(dst));
    __builtin_nontemporal_store(__builtin_bit_cast(raw, b), reinterpret_cast<raw*>(dst + HALF));
  }
}

template <typename T, int D>
int launch(const AppendParams& p, const PagedCache& cache, hipStream_t st) {
  const dim3 grid((unsigned)(p.S * p.n));
  const bool stream = (double)2 * p.S * p.n * (p.Hq + 2 * p.Hkv) * D * sizeof(T) > (double)((size_t)192 << 20);
#define LAUNCH(R, ST) ODY_LAUNCH("paged_append", st, (paged_append_kernel<T, D, R, ST>), grid, dim3(256), 0, p, cache)
  if (p.q) {
    if (stream) LAUNCH(true, true);
    else LAUNCH(true, false);
  } else {
    if (stream) LAUNCH(false, true);
    else LAUNCH(false, false);
  }
#undef LAUNCH
  return ody_check_launch("paged_append");
}

}  // namespace

PagedCache::PagedCache(void* k_, void* v_, const int* table_, const int* lengths_, const int* fresh_, PageStrides sk_, PageStrides sv_, int64_t table_stride_, int pages_,
                       int page_size, int width_, int value_bytes)
    : k(k_), v(v_), table(table_), lengths(lengths_), fresh(fresh_), sk(sk_), sv(sv_), table_stride(table_stride_), pages(pages_), shift(paged_shift(page_size)),
      width(width_) {
  const int64_t bytes = value_bytes;
  k_page = (unsigned)(bytes * sk.p), k_row = (unsigned)(bytes * sk.r), v_page = (unsigned)(bytes * sv.p), v_row = (unsigned)(bytes * sv.r);
}

int paged_check(const char* who, int S, int n, int Hq, int Hkv, int D, int dtype, int value_bytes, const PagedCache& c, int page_size) {
  ODY_REQUIRE(c.k && c.v && c.table && c.lengths, ODY_ERR_NULL, "%s: k_pages, v_pages, page_table or lengths is NULL", who);
  ODY_REQUIRE(S > 0 && n > 0 && Hq > 0 && Hkv > 0 && c.pages > 0 && c.width > 0, ODY_ERR_BAD_SHAPE,
              "%s: sizes must be positive (S=%d n=%d Hq=%d Hkv=%d pages=%d table_width=%d)", who, S, n, Hq, Hkv, c.pages, c.width);
  ODY_REQUIRE(Hq % Hkv == 0, ODY_ERR_BAD_SHAPE, "%s: Hq=%d is not a multiple of Hkv=%d", who, Hq, Hkv);
  ODY_REQUIRE(D == 64 || D == 128, ODY_ERR_UNSUPPORTED, "%s: head_dim %d not built (64, 128)", who, D);
  ODY_REQUIRE(dtype == ODY_BF16 || dtype == ODY_F32, ODY_ERR_UNSUPPORTED, "%s: dtype %d unknown", who, dtype);
  ODY_REQUIRE(page_size >= 8 && (page_size & (page_size - 1)) == 0, ODY_ERR_UNSUPPORTED, "%s: page_size %d: a power of two from 8 on", who, page_size);
  ODY_REQUIRE((int64_t)c.width * page_size <= ((int64_t)1 << 31) - PAGED_AHEAD, ODY_ERR_BAD_SHAPE, "%s: a table of more than 2^31 - %d places (%d columns, pages of %d)",
              who, PAGED_AHEAD, c.width, page_size);
  // rows are counted in 32 bits, up to the end of the last row tile, and vectors of a token up to the end of a block's turn; the product itself may be beyond 64
  const int64_t heads = Hq + 2 * (int64_t)Hkv;
  ODY_REQUIRE(heads < ((int64_t)1 << 31) / 16 - 256 && (double)S * n * heads < (double)(((int64_t)1 << 31) - PAGED_WIDE_ROWS), ODY_ERR_BAD_SHAPE,
              "%s: %lld heads of a token, or heads of all new tokens together, are too many", who, (long long)heads);
  const int64_t bytes = value_bytes, most = (int64_t)1 << 32;
  for (const PageStrides& s : {c.sk, c.sv})
    ODY_REQUIRE(s.p >= 0 && s.r >= 0 && s.p < most / bytes && s.r < most / bytes / page_size, ODY_ERR_UNSUPPORTED,
                "%s: pages, or the rows of a page, lie 4 GiB and more apart", who);
  ODY_REQUIRE(c.table_stride >= c.width || S == 1, ODY_ERR_BAD_SHAPE, "%s: rows of the page table overlap", who);
  ODY_REQUIRE(paged_rows_aligned(c.k, c.sk.p, c.sk.r, c.sk.h, value_bytes) && paged_rows_aligned(c.v, c.sv.p, c.sv.r, c.sv.h, value_bytes), ODY_ERR_MISALIGNED,
              "%s: k_pages and v_pages need 16-byte aligned pointers and strides", who);
  return ODY_OK;
}

extern "C" int ody_paged_append(const void* qkv, void* q, void* k_pages, void* v_pages, const int* page_table, const int* lengths,
                                const int* new_tokens, const int64_t* position_ids, const float* inv_freq, int S, int n, int Hq, int Hkv, int D,
                                int64_t sx_s, int64_t sx_n, int64_t sx_h, int64_t sq_s, int64_t sq_n, int64_t sq_h,
                                int64_t sk_p, int64_t sk_r, int64_t sk_h, int64_t sv_p, int64_t sv_r, int64_t sv_h,
                                int pages, int page_size, int table_width, int64_t table_stride, int dtype, void* stream) {
  const PagedCache c(k_pages, v_pages, page_table, lengths, new_tokens, {sk_p, sk_r, sk_h}, {sv_p, sv_r, sv_h}, table_stride, pages, page_size, table_width, paged_bytes(dtype));
  if (int rc = paged_check("ody_paged_append", S, n, Hq, Hkv, D, dtype, paged_bytes(dtype), c, page_size)) return rc;
  ODY_REQUIRE((int64_t)S * n < (int64_t)1 << 24, ODY_ERR_BAD_SHAPE, "ody_paged_append: 2^24 new tokens and more (a block of 256 threads each)");
  ODY_REQUIRE(qkv && (q == nullptr || inv_freq), ODY_ERR_NULL, "ody_paged_append: qkv, or inv_freq of a rotation, is NULL");
  ODY_REQUIRE(paged_rows_aligned(qkv, sx_s, sx_n, sx_h, paged_bytes(dtype)) && (q == nullptr || paged_rows_aligned(q, sq_s, sq_n, sq_h, paged_bytes(dtype))), ODY_ERR_MISALIGNED,
              "ody_paged_append: qkv and q need 16-byte aligned pointers and strides");
  const AppendParams p{qkv, q, position_ids, inv_freq, {sx_s, sx_n, sx_h}, {sq_s, sq_n, sq_h}, S, n, Hq, Hkv};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == ODY_BF16) return D == 64 ? launch<bf16, 64>(p, c, st) : launch<bf16, 128>(p, c, st);
  return D == 64 ? launch<float, 64>(p, c, st) : launch<float, 128>(p, c, st);
}
