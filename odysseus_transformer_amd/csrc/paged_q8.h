// A key / value cache in pages that holds its values in 8 bits: e4m3 with a power of two (e8m0) for each block of tokens and head.
#pragma once
#include "paged.h"

struct PagedScales {
  uint8_t *k, *v;       // (pages, page size >> shift, Hkv): 2^(byte - 127); 0 and 255 are never written
  PageStrides sk, sv;   // page, block of a page, head
  int shift;            // a block has 1 << shift tokens: 8 to 64, at most a page
};

#ifdef __HIPCC__
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float q8_scale(unsigned byte) { return __builtin_bit_cast(float, byte << 23); }
// Four values, exactly but at the ends of the type: an e4m3 value has four bits, a power of two moves its exponent.  Below bf16's smallest number (scales of 2^-126 and 2^-125) the nearest one,
// from 2^128 on infinite.
__device__ __forceinline__ void q8_values(unsigned word, float scale, bf16* to) {
  *reinterpret_cast<bf16x2*>(to) = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, false);
  *reinterpret_cast<bf16x2*>(to + 2) = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, true);
}
__device__ __forceinline__ void q8_values(unsigned word, float scale, float* to) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(word, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
  to[0] = a[0] * scale, to[1] = a[1] * scale, to[2] = b[0] * scale, to[3] = b[1] * scale;
}
__device__ __forceinline__ bf16x8 q8_operand(unsigned lo, unsigned hi, float scale) {
  bf16x8 r;
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  r[0] = a[0], r[1] = a[1], r[2] = b[0], r[3] = b[1], r[4] = c[0], r[5] = c[1], r[6] = d[0], r[7] = d[1];
  return r;
}
#endif

// The kernels of many rows (paged_q8_chunk.hip, paged_q8_wide.hip), by p.tile.
int ody_launch_paged_chunk_q8(const PagedAttnParams& p, int D, const PagedCache& c, const PagedScales& z, int blocks, hipStream_t st);
int ody_launch_paged_wide_q8(const PagedAttnParams& p, const PagedCache& c, const PagedScales& z, int blocks, hipStream_t st);

// Host side: what the entry points of such a cache check, behind paged_check.
int paged_q8_check(const char* who, const PagedScales& z, int page_size, int block);
static inline int paged_q8_shift(int block) { return block > 0 ? __builtin_ctz((unsigned)block) : 0; }
