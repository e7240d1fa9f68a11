// A token of each row of logits, by temperature, top-k, top-p and min-p, from a given random number.
//
// The order of a row's tokens is by falling logits, the lower index first among equals.  Each cut leaves a prefix of that order, and the token is where the sums of the
// weights exp((x - max) / T) along it pass the random number's share of what is kept: all of it asks for one thing, the first token at which a sum along the order (of
// tokens, or of weights) reaches a target.  No row is sorted for that.  Sums by buckets of x, 2048 of them, say which bucket the place is in; the bucket's tokens, a few as a
// rule, are gathered and sorted; a bucket of too many tokens is divided anew, by the bits of x, until it has few or one value.
//
// Weights are whole numbers of 2^-FRAC (FRAC = 62 - log2 of the row's length, 45 for a vocabulary of 128000), evaluated in 64 bits: sums in any order, by atomics too, are the same, and
// as exact as sums of so many weights in 64-bit floating point.  2^y = 2^-(n / 64) 2^-r, |r| <= 1 / 128: a table of 64 entries and a polynomial of the fifth degree, off by
// 2^-50 of themselves.
#include <algorithm>
#include <cmath>
#include "ody_common.h"

namespace {

typedef unsigned long long u64;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int THREADS = 1024, WAVES = THREADS / 64, BUCKETS = 2048, LIST = 4096;
constexpr int MOST = (1 << 21) - 4;   // tokens of a row: nth_of() counts the matches of 16 wavefronts a turn in 2 * LIST numbers, at most 512 turns of 4 * THREADS tokens

struct SampleParams {
  const void* logits;
  int64_t row_stride;
  const float *u, *temperature, *top_p, *min_p;   // of each row; but for u null: the numbers below for all
  const int* top_k;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int64_t* tokens;
  float* logprobs;
  int vocab, frac;
};

// 2^(-j / 64)
struct Table { double x[64]; };
constexpr Table powers() {
  Table t{};
  double root[6] = {};   // 2^(-1/2), 2^(-1/4) .. 2^(-1/64): by Newton's iteration
  double of = 0.5;
  for (int k = 0; k < 6; k++) {
    double y = of;
    for (int i = 0; i < 60; i++) y = 0.5 * (y + of / y);
    root[k] = of = y;
  }
  for (int j = 0; j < 64; j++) {
    t.x[j] = 1.0;
    for (int k = 0; k < 6; k++)
      if (j >> (5 - k) & 1) t.x[j] *= root[k];
  }
  return t;
}
__device__ const Table POWERS = powers();

// x as a number whose order is that of the logits: -0 as 0, NaN as the lowest
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __builtin_bit_cast(unsigned, x);
  return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned k) { return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// a thread's share of a row
template <typename T> struct Reader {
  static constexpr int N = 16 / (int)sizeof(T);
  const T* base;      // 16-byte aligned, at most N - 1 values before the row
  int head, vocab, vectors;
  bool infinite;      // the largest logit is +inf: those count, as equals
  __device__ __forceinline__ Reader(const T* row, int vocab_) : vocab(vocab_), infinite(false) {
    head = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    base = row - head;
    vectors = (head + vocab + N - 1) / N;
  }
  __device__ __forceinline__ float value(float x) const {
    x = x == x ? x + 0.f : -INFINITY;
    return infinite ? (x == INFINITY ? 0.f : -INFINITY) : x;
  }
  // f(x, index) of the vectors v0, v0 + step .. in rising order
  template <typename F> __device__ __forceinline__ void vector(int v, F f) const {
    const u32x4 raw = *(const u32x4 __attribute__((address_space(1)))*)(base + (int64_t)v * N);
    const int first = v * N - head;
#pragma unroll
    for (int e = 0; e < N; e++) {
      const unsigned word = sizeof(T) == 2 ? raw[e / 2] : raw[e], bits = sizeof(T) == 4 ? word : e & 1 ? word & 0xffff0000u : word << 16;
      if ((unsigned)(first + e) < (unsigned)vocab) f(value(__builtin_bit_cast(float, bits)), first + e);
    }
  }
  template <typename F> __device__ __forceinline__ void all(F f) const {
#pragma unroll 2
    for (int v = threadIdx.x; v < vectors; v += THREADS) vector(v, f);
  }
};

struct Weights {
  double c, top, magic;   // 64 log2(e) / T; the largest logit; 2^(52 - FRAC)
  const double* table;
  // 64 log2 of max weight over weight, at most what no weight is left of
  __device__ __forceinline__ double steps(float x) const { return fmin((top - (double)x) * c, 64.0 * 60.0); }
  __device__ __forceinline__ int nearest(double t, double& r) const {
    const double k = t + 6755399441055744.0;   // 1.5 * 2^52
    r = t - (k - 6755399441055744.0);
    return (int)(unsigned)__builtin_bit_cast(u64, k);
  }
  __device__ __forceinline__ u64 of(double t, int& bucket) const {
    double r;
    const int n = nearest(t, r);
    bucket = (int)min((unsigned)n, (unsigned)BUCKETS - 1);
    constexpr double L = -0.010830424696249145;   // -ln 2 / 64
    double p = L * L * L * L * L / 120;
    p = fma(p, r, L * L * L * L / 24);
    p = fma(p, r, L * L * L / 6);
    p = fma(p, r, L * L / 2);
    p = fma(p, r, L);
    p = fma(p, r, 1.0);
    const double e = __builtin_bit_cast(double, __builtin_bit_cast(u64, table[n & 63]) - ((u64)(n >> 6) << 52));
    return __builtin_bit_cast(u64, fma(e, p, magic)) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 of(float x) const {
    int b;
    return of(steps(x), b);
  }
};

__device__ __forceinline__ u64 shfl_up64(u64 x, int d) {
  return (u64)__shfl_up((unsigned)(x >> 32), d, 64) << 32 | __shfl_up((unsigned)x, d, 64);
}
__device__ __forceinline__ u64 wave_scan(u64 x, int lane) {   // inclusive
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u64 y = shfl_up64(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

struct Shared {
  double table[64];
  u64 mass[BUCKETS];
  unsigned count[BUCKETS];
  u64 list[LIST];
  u64 wave[WAVES];
  u64 found[4];
  unsigned words[4];
};

// Exclusive sum over the block; `all`: of all threads
__device__ __forceinline__ u64 block_scan(Shared& s, u64 x, u64& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 upto = wave_scan(x, lane);
  __syncthreads();
  if (lane == 63) s.wave[wave] = upto;
  __syncthreads();
  u64 before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) {
    if (w < wave) before += s.wave[w];
    all += s.wave[w];
  }
  return before + upto - x;
}

// A place in the order: the tokens and weights before it, and what it is among -- the keys lo .. hi
struct Place {
  unsigned lo, hi;
  u64 count, mass;
};

template <typename T>
struct Sampler {
  Shared& s;
  Reader<T> row;
  Weights w;

  // Ascending, of n entries; the rest of the power of two is filled with the highest.
  __device__ void sort(int n) {
    int size = 64;
    while (size < n) size *= 2;
    __syncthreads();
    for (int i = threadIdx.x; i < size; i += THREADS)
      if (i >= n) s.list[i] = ~0ull;
    for (int k = 2; k <= size; k *= 2)
      for (int j = k / 2; j > 0; j /= 2) {
        __syncthreads();
        for (int i = threadIdx.x; i < size / 2; i += THREADS) {
          const int a = 2 * i - (i & (j - 1)), b = a + j;
          const u64 x = s.list[a], y = s.list[b];
          if ((x > y) == ((a & k) == 0)) s.list[a] = y, s.list[b] = x;
        }
      }
    __syncthreads();
  }

  // Tokens for which keep(x) holds into the list, (falling key, index); how many there are, which may be more than fit.
  template <typename F> __device__ int gather(F keep) {
    __syncthreads();
    if (threadIdx.x == 0) s.words[0] = 0;
    __syncthreads();
    row.all([&](float x, int i) {
      if (keep(x)) {
        const unsigned at = atomicAdd(&s.words[0], 1u);
        if (at < LIST) s.list[at] = (u64)~key_of(x) << 32 | (unsigned)i;
      }
    });
    __syncthreads();
    return (int)s.words[0];
  }

  // The first of the sorted list's n entries at which the sum (of tokens, or of weights) behind `before` reaches the target: its entry, and the sums up to and with it.
  __device__ void reach(int n, bool by_count, u64 target, u64 count, u64 mass, u64& entry, u64& mass_upto) {
    constexpr int PER = LIST / THREADS;
    u64 mine[PER], sum = 0;
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int i = threadIdx.x * PER + k;
      if (i < n) sum += w.of(of_key(~(unsigned)(s.list[i] >> 32)));
      mine[k] = sum;
    }
    u64 all;
    const u64 before = mass + block_scan(s, sum, all);
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int i = threadIdx.x * PER + k;
      const u64 now = before + mine[k], was = k ? before + mine[k - 1] : before;
      if (i < n && (by_count ? count + i + 1 == target : was < target && now >= target)) s.found[0] = s.list[i], s.found[1] = now;
    }
    __syncthreads();
    entry = s.found[0], mass_upto = s.found[1];
    __syncthreads();
  }

  // The bucket in which the sum reaches the target, and the sums before it.
  __device__ int bucket_of(bool by_count, u64 target, u64& count, u64& mass) {
    constexpr int PER = BUCKETS / THREADS;
    const int b0 = threadIdx.x * PER;
    u64 sum = 0, tokens = 0, all;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; k++) sum += s.mass[b0 + k], tokens += s.count[b0 + k];
    u64 m = mass + block_scan(s, sum, all), c = count + block_scan(s, tokens, all);
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const u64 m1 = m + s.mass[b0 + k], c1 = c + s.count[b0 + k];
      if (by_count ? c < target && c1 >= target : m < target && m1 >= target) s.words[1] = b0 + k, s.found[0] = c, s.found[1] = m;
      m = m1, c = c1;
    }
    __syncthreads();
    count = s.found[0], mass = s.found[1];
    const int b = s.words[1];
    __syncthreads();
    return b;
  }
  __device__ void clear() {
    __syncthreads();
    for (int b = threadIdx.x; b < BUCKETS; b += THREADS) s.mass[b] = 0, s.count[b] = 0;
    __syncthreads();
  }

  // The `nth` (from 1) token with this key, by its index.
  __device__ int nth_of(unsigned key, unsigned nth) {
    unsigned* counts = reinterpret_cast<unsigned*>(s.list);   // [turn][wavefront]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, turns = (row.vectors + THREADS - 1) / THREADS;
    __syncthreads();
    auto matches = [&](int turn, unsigned& mask) {
      mask = 0;
      const int v = turn * THREADS + threadIdx.x;
      if (v < row.vectors) row.vector(v, [&](float x, int i) { if (key_of(x) == key) mask |= 1u << (i + row.head - v * row.N); });
    };
    for (int turn = 0; turn < turns; turn++) {
      unsigned mask;
      matches(turn, mask);
      const u64 upto = wave_scan(__popc(mask), lane);
      if (lane == 63) counts[turn * WAVES + wave] = (unsigned)upto;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned left = nth;
      int at = 0;
      while (at < turns * WAVES - 1 && counts[at] < left) left -= counts[at++];
      s.words[2] = at, s.words[3] = left;
    }
    __syncthreads();
    const int turn = s.words[2] / WAVES;
    if (wave == (int)s.words[2] % WAVES) {
      unsigned mask;
      matches(turn, mask);
      const unsigned mine = __popc(mask), upto = (unsigned)wave_scan(mine, lane);
      unsigned left = s.words[3];
      if (upto - mine < left && upto >= left) {
        left -= upto - mine;
        while (--left) mask &= mask - 1;
        s.words[1] = (turn * THREADS + threadIdx.x) * row.N - row.head + __ffs(mask) - 1;
      }
    }
    __syncthreads();
    const int index = s.words[1];
    __syncthreads();
    return index;
  }

  // Where the sum reaches the target, among the tokens for which in(x) holds, `count` and `mass` before them: the entry (falling key, index), and the weights up to and with it.
  template <typename F> __device__ void resolve(F in, bool by_count, u64 target, u64 count, u64 mass, bool want_index, u64& entry, u64& mass_upto) {
    int n = gather(in);
    if (n <= LIST) {
      sort(n);
      reach(n, by_count, target, count, mass, entry, mass_upto);
      return;
    }
    // many: the keys that they lie between, and from there on by those
    if (threadIdx.x == 0) s.words[2] = ~0u, s.words[3] = 0;
    __syncthreads();
    unsigned lo = ~0u, hi = 0;
    row.all([&](float x, int) {
      if (in(x)) lo = min(lo, key_of(x)), hi = max(hi, key_of(x));
    });
    atomicMin(&s.words[2], lo);
    atomicMax(&s.words[3], hi);
    __syncthreads();
    lo = s.words[2], hi = s.words[3];
    for (;;) {
      if (lo == hi) {   // equals
        const u64 each = w.of(of_key(lo)), nth = by_count ? target - count : (target - mass + each - 1) / each;
        mass_upto = mass + nth * each;
        entry = (u64)~lo << 32 | (unsigned)(want_index ? nth_of(lo, (unsigned)nth) : 0);
        return;
      }
      const int shift = max(0, 32 - __clz(hi - lo) - 11);
      clear();
      row.all([&](float x, int) {
        const unsigned k = key_of(x);
        if (k >= lo && k <= hi) {
          atomicAdd(&s.mass[(hi - k) >> shift], w.of(x));
          atomicAdd(&s.count[(hi - k) >> shift], 1u);
        }
      });
      const int b = bucket_of(by_count, target, count, mass);
      hi -= (unsigned)b << shift;
      if (hi - lo >= 1u << shift) lo = hi - ((1u << shift) - 1);
      n = gather([&](float x) { return key_of(x) >= lo && key_of(x) <= hi; });
      if (n <= LIST) {
        sort(n);
        reach(n, by_count, target, count, mass, entry, mass_upto);
        return;
      }
    }
  }
};

template <typename T>
__global__ __launch_bounds__(THREADS) void sample_kernel(const SampleParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float temperature = p.temperature ? p.temperature[r] : p.temperature_all, top_p = p.top_p ? p.top_p[r] : p.top_p_all,
              min_p = p.min_p ? p.min_p[r] : p.min_p_all, u = p.u[r];
  const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  Sampler<T> a{s, Reader<T>(static_cast<const T*>(p.logits) + r * p.row_stride, p.vocab), {}};
  if (tid < 64) s.table[tid] = POWERS.x[tid];

  // ---- the first of the order
  float best = -INFINITY;
  int at = 0x7fffffff;
  a.row.all([&](float x, int i) {
    if (x > best) best = x, at = i;
  });
  u64 first = (u64)~key_of(best) << 32 | (unsigned)at;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u64 y = (u64)__shfl_xor((unsigned)(first >> 32), d, 64) << 32 | __shfl_xor((unsigned)first, d, 64);
    first = min(first, y);
  }
  if (lane == 0) s.wave[wave] = first;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < WAVES; k++) first = min(first, s.wave[k]);
  const float largest = of_key(~(unsigned)(first >> 32));
  if (largest == -INFINITY || !(temperature > 0.f)) {   // nothing to choose from, or nothing but the first
    if (tid == 0) {
      p.tokens[r] = largest == -INFINITY ? -1 : (int64_t)(unsigned)first;
      p.logprobs[r] = largest == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  a.row.infinite = largest == INFINITY;
  a.w = Weights{64.0 * 1.4426950408889634 / (double)temperature, a.row.infinite ? 0.0 : (double)largest, __builtin_bit_cast(double, (u64)(1023 + 52 - p.frac) << 52), s.table};
  const u64 one = 1ull << p.frac;
  const bool cut_k = top_k > 0 && top_k < p.vocab, cut_p = top_p < 1.f, cut_m = min_p > 0.f;
  const u64 least = cut_m ? (u64)fmin(ceil((double)min_p * (double)one), 9e18) : 0;

  // ---- sums of the buckets
  a.clear();
  u64 over = 0;   // of weights that are not less than min_p
  a.row.all([&](float x, int) {
    int b;
    const u64 wt = a.w.of(a.w.steps(x), b);
    atomicAdd(&s.mass[b], wt);
    if (cut_k) atomicAdd(&s.count[b], 1u);
    if (cut_m && wt >= least) over += wt;
  });
  u64 total;
  {
    u64 sum = 0;
    __syncthreads();
    for (int b = tid; b < BUCKETS; b += THREADS) sum += s.mass[b];
    block_scan(s, sum, total);
  }
  if (cut_m) {
    u64 all;
    block_scan(s, over, all);
    over = max(all, one);   // the first one at any rate
  }
  // the tokens of a bucket
  auto in_bucket = [&](int b) {
    return [&a, b](float x) {
      double rest;
      return (int)min((unsigned)a.w.nearest(a.w.steps(x), rest), (unsigned)BUCKETS - 1) == b;
    };
  };
  u64 entry, kept = total;
  // resolve() may use the buckets for others
  auto again = [&]() {
    a.clear();
    a.row.all([&](float x, int) {
      int b;
      const u64 wt = a.w.of(a.w.steps(x), b);
      atomicAdd(&s.mass[b], wt);
    });
  };
  if (cut_k) {
    u64 count = 0, mass = 0;
    const int b = a.bucket_of(true, top_k, count, mass);
    a.resolve(in_bucket(b), true, top_k, count, mass, false, entry, kept);
    again();
  }
  if (cut_p) {
    const u64 target = max((u64)1, (u64)ceil(fmax((double)top_p, 0.0) * (double)kept));
    u64 count = 0, mass = 0, upto;
    const int b = a.bucket_of(false, target, count, mass);
    a.resolve(in_bucket(b), false, target, count, mass, false, entry, upto);
    kept = min(kept, upto);
    again();
  }
  if (cut_m) kept = min(kept, over);
  const double share = (double)u * (double)kept;
  const u64 target = share > 0.0 ? min((u64)fmin(share, 9e18) + 1, kept) : 1;
  u64 count = 0, mass = 0, upto;
  const int b = a.bucket_of(false, target, count, mass);
  a.resolve(in_bucket(b), false, target, count, mass, true, entry, upto);
  if (tid == 0) {
    p.tokens[r] = (int64_t)(unsigned)entry;
    const double log2w = -a.w.steps(of_key(~(unsigned)(entry >> 32))) / 64.0;
    p.logprobs[r] = (float)((log2w + p.frac) * 0.6931471805599453 - log((double)kept));
  }
}

template <typename T>
int launch(const SampleParams& p, int rows, hipStream_t st) {
  if (int rc = ody_allow_dynamic_lds(reinterpret_cast<const void*>(&sample_kernel<T>), sizeof(Shared), "ody_sample")) return rc;
  ODY_LAUNCH("sample", st, (sample_kernel<T>), dim3((unsigned)rows), dim3(THREADS), sizeof(Shared), p);
  return ody_check_launch("sample");
}

}  // namespace

extern "C" int ody_sample(const void* logits, const float* u, const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                          float temperature_all, int top_k_all, float top_p_all, float min_p_all, int64_t* tokens, float* logprobs, int rows, int vocab,
                          int64_t row_stride, int dtype, void* stream) {
  ODY_REQUIRE(logits && u && tokens && logprobs, ODY_ERR_NULL, "ody_sample: logits, u, tokens or logprobs is NULL");
  ODY_REQUIRE(rows > 0 && vocab > 0 && rows < 1 << 22 && vocab <= MOST, ODY_ERR_BAD_SHAPE, "ody_sample: %d rows of %d logits (fewer than 2^22 of at most %d)", rows, vocab, MOST);
  ODY_REQUIRE(row_stride >= vocab || rows == 1, ODY_ERR_BAD_SHAPE, "ody_sample: rows overlap (stride %lld)", (long long)row_stride);
  ODY_REQUIRE(dtype == ODY_BF16 || dtype == ODY_F32, ODY_ERR_UNSUPPORTED, "ody_sample: dtype %d unknown", dtype);
  ODY_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (dtype == ODY_BF16 ? 1 : 3)) == 0, ODY_ERR_MISALIGNED, "ody_sample: logits are not aligned to their size");
  int bits = 0;
  while (1 << bits < vocab) bits++;
  const SampleParams p{logits, row_stride, u, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all, top_k_all, tokens, logprobs, vocab,
                       std::min(50, 62 - bits)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == ODY_BF16 ? launch<bf16>(p, rows, st) : launch<float>(p, rows, st);
}
