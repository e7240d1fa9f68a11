// A key / value cache in pages, as the kernels that fill and read it see it.
#pragma once
#include "attn_params.h"

struct PageStrides {
  int64_t p, r, h;  // page, row of a page, head: elements; head_dim stride is 1
};

struct PagedCache {
  void* k;              // (pages, page size, Hkv, D)
  void* v;
  const int* table;     // (S, width): page of rows [c << shift, (c + 1) << shift) of a sequence; outside [0, pages): none
  const int* lengths;   // (S): tokens of the sequence, the new ones included
  PageStrides sk, sv;
  int64_t table_stride;
  int pages, shift, width;
};

#ifdef __HIPCC__
// Tokens of sequence s that can have a page: a length of less than nothing is nothing, what lies behind the table's last column has
// no page (the host checks width << shift < 2^31).
__device__ __forceinline__ int paged_length(const PagedCache& c, int s) { return max(0, min(c.lengths[s], c.width << c.shift)); }
#endif

// Host side: the checks that both entry points share.
int paged_check(const char* who, int S, int n, int Hq, int Hkv, int D, int dtype, const PagedCache& c, int page_size);
static inline bool paged_rows_aligned(const void* ptr, int64_t a, int64_t b, int64_t c, int dtype) {
  const int q = dtype == ODY_BF16 ? 8 : 4;
  return ody_aligned16(ptr) && a % q == 0 && b % q == 0 && c % q == 0;
}
static inline int paged_shift(int page_size) { return page_size > 0 ? __builtin_ctz((unsigned)page_size) : 0; }
