// Attention of new tokens over a key / value cache in pages.
#include <cmath>
#include "paged.h"

namespace {

struct PagedAttnParams {
  const void* q;   // (S, n, Hq, D)
  void* out;       // (S, n, Hq, D)
  float* lse;      // (S, Hq, n)
  AttnStrides sq, so;
  int S, n, Hq, Hkv, group;
  float scale_log2e;
};

// One wavefront per (sequence, token, query head), a key after the other.
template <typename T, int D>
__global__ __launch_bounds__(64) void paged_attn_kernel(const PagedAttnParams p, const PagedCache cache) {
  constexpr int N = D / 64;
  const int lane = threadIdx.x, h = blockIdx.x % p.Hq, i = blockIdx.x / p.Hq % p.n, s = blockIdx.x / (p.Hq * p.n), hk = h / p.group;
  float q[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < N; e++) {
    q[e] = (float)static_cast<const T*>(p.q)[s * p.sq.b + i * p.sq.l + h * p.sq.h + lane * N + e] * p.scale_log2e;
    o[e] = 0.f;
  }
  const int keys = min(paged_length(cache, s), max(cache.lengths[s], 0) - p.n + i + 1);
  for (int k = 0; k < keys; k++) {
    const int page = cache.table[s * cache.table_stride + (k >> cache.shift)], row = k & ((1 << cache.shift) - 1);
    if (page < 0 || page >= cache.pages) continue;
    const T* kp = static_cast<const T*>(cache.k) + page * cache.sk.p + row * cache.sk.r + hk * cache.sk.h + lane * N;
    const T* vp = static_cast<const T*>(cache.v) + page * cache.sv.p + row * cache.sv.r + hk * cache.sv.h + lane * N;
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < N; e++) x = fmaf(q[e], (float)kp[e], x);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d, 64);
    const float top = fmaxf(m, x), ref = top == -INFINITY ? 0.f : top, alpha = ody_exp2(m - ref), w = ody_exp2(x - ref);
    m = top, l = l * alpha + w;
#pragma unroll
    for (int e = 0; e < N; e++) o[e] = fmaf(w, (float)vp[e], o[e] * alpha);
  }
#pragma unroll
  for (int e = 0; e < N; e++)
    static_cast<T*>(p.out)[s * p.so.b + i * p.so.l + h * p.so.h + lane * N + e] = (T)(l == 0.f ? 0.f : o[e] / l);
  if (lane == 0) p.lse[((int64_t)s * p.Hq + h) * p.n + i] = l == 0.f ? -INFINITY : (m + log2f(l)) * ODY_LN2;
}

template <typename T>
int by_head_dim(const PagedAttnParams& p, int D, const PagedCache& c, hipStream_t st) {
  const dim3 grid((unsigned)(p.S * p.n * p.Hq));
  if (D == 64) ODY_LAUNCH("paged_attn", st, (paged_attn_kernel<T, 64>), grid, dim3(64), 0, p, c);
  else ODY_LAUNCH("paged_attn", st, (paged_attn_kernel<T, 128>), grid, dim3(64), 0, p, c);
  return ody_check_launch("paged_attn");
}

}  // namespace

extern "C" size_t ody_paged_attn_workspace_bytes(int S, int n, int Hq, int Hkv, int D, int page_size, int table_width, int dtype) { return 0; }

extern "C" int ody_paged_attn(const void* q, const void* k_pages, const void* v_pages, const int* page_table, const int* lengths, void* out,
                              float* lse, int S, int n, int Hq, int Hkv, int D, int64_t sq_s, int64_t sq_n, int64_t sq_h,
                              int64_t sk_p, int64_t sk_r, int64_t sk_h, int64_t sv_p, int64_t sv_r, int64_t sv_h,
                              int64_t so_s, int64_t so_n, int64_t so_h, int pages, int page_size, int table_width, int64_t table_stride,
                              float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const PagedCache c{const_cast<void*>(k_pages), const_cast<void*>(v_pages), page_table, lengths, {sk_p, sk_r, sk_h}, {sv_p, sv_r, sv_h},
                     table_stride, pages, paged_shift(page_size), table_width};
  if (int rc = paged_check("ody_paged_attn", S, n, Hq, Hkv, D, dtype, c, page_size)) return rc;
  ODY_REQUIRE(q && out && lse, ODY_ERR_NULL, "ody_paged_attn: q, out or lse is NULL");
  ODY_REQUIRE(paged_rows_aligned(q, sq_s, sq_n, sq_h, dtype) && paged_rows_aligned(out, so_s, so_n, so_h, dtype), ODY_ERR_MISALIGNED,
              "ody_paged_attn: q and out need 16-byte aligned pointers and strides");
  const PagedAttnParams p{q, out, lse, {sq_s, sq_n, sq_h}, {so_s, so_n, so_h}, S, n, Hq, Hkv, Hq / Hkv, scale * ODY_LOG2E};
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == ODY_BF16 ? by_head_dim<bf16>(p, D, c, st) : by_head_dim<float>(p, D, c, st);
}
