// A token of each row of logits, by temperature, top-k, top-p and min-p, from a given random number.
//
// The order of a row's tokens is by falling logits, the lower index first among equals.  Each cut leaves a prefix of that order, and the token is where the sums of the
// weights exp((x - max) / T) along it pass the random number's share of what is kept: all of it asks for one thing, the first token at which a sum along the order (of
// tokens, or of weights) reaches a target.  No row is sorted for that.  Sums by buckets of x, 2048 of them, say which bucket the place is in; the bucket's tokens, a few as a
// rule, are gathered and ordered; a bucket of too many tokens is divided anew, by the bits of x, until it has few or one value.  Where top_k is small, the buckets count tokens, what may be
// among the first is gathered, and nothing else has a weight formed.
//
// Weights are whole numbers of 2^-FRAC (FRAC = 62 - log2 of the row's length, 45 for a vocabulary of 128000): sums in any order, by atomics too, are the same.  They are formed in 64 bits, whose
// vector rate is that of 32 here, as 2^-(n / 1024) 2^(-r / 1024), |r| <= 1 / 2, from a table and a polynomial of the second degree: off by 2^-37 of themselves, so that a place is
// missed where a random number is as near to a border of its share as that.
//
// A block has a row, which stays in its registers where it fits (1024 threads of 16 vectors) and is read again for each pass where not.
#include <algorithm>
#include <cmath>
#include "ody_common.h"

namespace {

typedef unsigned long long u64;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef const u32x4 __attribute__((address_space(1)))* vector_ptr;

constexpr int THREADS = 1024, WAVES = THREADS / 64, BUCKETS = 2048, LIST = 4096, OCTAVE = 1024;
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

// 2^(-j / 32) and 2^(-j / 1024)
struct Table { double x[2][32]; };
constexpr Table powers() {
  Table t{};
  double root[10] = {}, of = 0.5;   // 2^(-1/2), 2^(-1/4) ..: by Newton's iteration
  for (int k = 0; k < 10; k++) {
    double y = of;
    for (int i = 0; i < 60; i++) y = 0.5 * (y + of / y);
    root[k] = of = y;
  }
  for (int half = 0; half < 2; half++)
    for (int j = 0; j < 32; j++) {
      t.x[half][j] = 1.0;
      for (int k = 0; k < 5; k++)
        if (j >> (4 - k) & 1) t.x[half][j] *= root[5 * half + k];
    }
  return t;
}
__device__ const Table POWERS = powers();

// x as a number whose order is that of the logits: -0 as 0, NaN as the lowest
__device__ __forceinline__ unsigned key_of(float x) {
  x = x == x ? x + 0.f : -INFINITY;
  const unsigned b = __builtin_bit_cast(unsigned, x);
  return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned k) { return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// A row, in vectors of 16 bytes that hold at least one value of it.  What is not the row's counts as -inf, which has no weight and so is never a result.
template <typename T, int NV>
struct Row {
  static constexpr int N = 16 / (int)sizeof(T);
  const T* base;      // 16-byte aligned, at most N - 1 values before the row
  int head, vocab, vectors;
  bool infinite;      // the largest logit is +inf: those count as 0, all others as -inf
  u32x4 held[NV > 0 ? NV : 1];

  __device__ __forceinline__ Row(const T* row, int vocab_) : vocab(vocab_), infinite(false) {
    head = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    base = row - head;
    vectors = (head + vocab + N - 1) / N;
    if constexpr (NV > 0) {
#pragma unroll
      for (int v = 0; v < NV; v++) {
        const int at = v * THREADS + (int)threadIdx.x;
        held[v] = at < vectors ? ((vector_ptr)base)[at] : u32x4{LOWEST, LOWEST, LOWEST, LOWEST};
      }
#pragma unroll
      for (int v = 0; v < NV; v++) {
        const int at = v * THREADS + (int)threadIdx.x;
        if (at * N < head || (at + 1) * N > head + vocab) held[v] = without(held[v], at);
      }
    }
  }
  static constexpr unsigned LOWEST = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;   // -inf
  __device__ __forceinline__ u32x4 without(u32x4 raw, int at) const {
    const int first = at * N - head;
#pragma unroll
    for (int e = 0; e < N; e++)
      if ((unsigned)(first + e) >= (unsigned)vocab) {
        if (sizeof(T) == 4) raw[e] = LOWEST;
        else raw[e / 2] = e & 1 ? (raw[e / 2] & 0xffffu) | (LOWEST & 0xffff0000u) : (raw[e / 2] & 0xffff0000u) | (LOWEST & 0xffffu);
      }
    return raw;
  }
  __device__ __forceinline__ static float element(const u32x4& raw, int e) {
    const unsigned word = sizeof(T) == 2 ? raw[e / 2] : raw[e], bits = sizeof(T) == 4 ? word : e & 1 ? word & 0xffff0000u : word << 16;
    return __builtin_bit_cast(float, bits);
  }
  __device__ __forceinline__ int index(int v, int e) const { return (v * THREADS + (int)threadIdx.x) * N - head + e; }
  __device__ __forceinline__ static u32x4 infinite_only(u32x4 raw) {
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const unsigned x = raw[w];
      if (sizeof(T) == 4) raw[w] = x == 0x7f800000u ? 0u : LOWEST;
      else raw[w] = ((x & 0xffffu) == 0x7f80u ? 0u : LOWEST & 0xffffu) | ((x & 0xffff0000u) == 0x7f800000u ? 0u : LOWEST & 0xffff0000u);
    }
    return raw;
  }
  // the thread's vector of a turn, from memory
  __device__ __forceinline__ u32x4 read(int v) const {
    const int at = v * THREADS + (int)threadIdx.x;
    u32x4 raw = {LOWEST, LOWEST, LOWEST, LOWEST};
    if (at < vectors) {
      raw = ((vector_ptr)base)[at];
      if (at * N < head || (at + 1) * N > head + vocab) raw = without(raw, at);
      if (infinite) raw = infinite_only(raw);
    }
    return raw;
  }
  // +inf is the largest: from now on
  __device__ void only_infinite() {
    infinite = true;
#pragma unroll
    for (int v = 0; v < NV; v++) held[v] = infinite_only(held[v]);
  }
  // Element e, which no constant is.
  __device__ __forceinline__ static float any_element(const u32x4& raw, int e) {
    const int at = sizeof(T) == 2 ? e >> 1 : e;
    const unsigned word = at == 0 ? raw[0] : at == 1 ? raw[1] : at == 2 ? raw[2] : raw[3], bits = sizeof(T) == 4 ? word : e & 1 ? word & 0xffff0000u : word << 16;
    return __builtin_bit_cast(float, bits);
  }
  // f(x, index) for every x for which keep(x) holds, which are few
  template <typename K, typename F> __device__ __forceinline__ void matches(K keep, F f) {
    auto vector = [&](const u32x4& raw, int v) __attribute__((always_inline)) {
      unsigned mask = 0;
#pragma unroll
      for (int e = 0; e < N; e++) mask |= keep(element(raw, e)) ? 1u << e : 0u;
      while (mask) {
        const int e = __ffs(mask) - 1;
        mask &= mask - 1;
        int t = threadIdx.x;
        asm volatile("" : "+v"(t));   // the index here, and not of all elements in front of it
        f(any_element(raw, e), (v * THREADS + t) * N - head + e);
      }
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int v = 0; v < NV; v++) {
        asm volatile("" : "+v"(held[v]));
        vector(held[v], v);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      for (int v = 0; v * THREADS < vectors; v++) vector(read(v), v);
    }
  }
  // f(x, turn, element): index(turn, element) is the token's
  template <typename F> __device__ __forceinline__ void turn(int v, F f) const {
    const u32x4 raw = read(v);
#pragma unroll
    for (int e = 0; e < N; e++) f(element(raw, e), v, e);
  }
  template <typename F> __device__ __forceinline__ void again(F f) const {   // for the seldom passes, whose code would be as long as the row
    for (int v = 0; v * THREADS < vectors; v++) turn(v, f);
  }
  template <typename F> __device__ __forceinline__ void all(F f) {
    if constexpr (NV > 0) {
#pragma unroll
      for (int v = 0; v < NV; v++) {
        asm volatile("" : "+v"(held[v]));   // what one pass makes of a value is not kept for the next one: there are no registers for that
#pragma unroll
        for (int e = 0; e < N; e++) f(element(held[v], e), v, e);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      again(f);
    }
  }
};

struct Weights {
  double c, top, magic;   // OCTAVE log2(e) / T; the largest logit; 2^(52 - FRAC)
  float topf;
  const double* table;    // 2^(-j / OCTAVE)
  // OCTAVE log2 of max weight over weight, at most what no weight is left of, which NaN is too
  __device__ __forceinline__ double steps(float x) const { return fmin((top - (double)x) * c, 60.0 * OCTAVE); }
  __device__ __forceinline__ static unsigned nearest(double t, double& r) {
    const double k = t + 6755399441055744.0;   // 1.5 * 2^52
    r = t - (k - 6755399441055744.0);
    return (unsigned)__builtin_bit_cast(u64, k);
  }
  __device__ __forceinline__ static unsigned bucket_of(unsigned n) { return min(n / (OCTAVE / 64), (unsigned)BUCKETS - 1); }
  __device__ __forceinline__ unsigned bucket(float x) const {
    double r;
    return bucket_of(nearest(steps(x), r));
  }
  // of a bucket by the value alone: 64 of them for 1
  __device__ __forceinline__ unsigned plain_bucket(float x) const { return (unsigned)fminf((topf - x) * 64.f, (float)(BUCKETS - 1)); }
  __device__ __forceinline__ u64 of(float x, unsigned& bucket) const {
    double r;
    const unsigned n = nearest(steps(x), r);
    bucket = bucket_of(n);
    constexpr double L = -0.6931471805599453 / OCTAVE;
    const double p = fma(fma(L * L / 2, r, L), r, 1.0);
    u64 e = __builtin_bit_cast(u64, table[n % OCTAVE]);
    e = (u64)((unsigned)(e >> 32) - (n / OCTAVE << 20)) << 32 | (unsigned)e;
    return __builtin_bit_cast(u64, fma(__builtin_bit_cast(double, e), p, magic)) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 of(float x) const {
    unsigned b;
    return of(x, b);
  }
};

// Inclusive sums over the lanes of a wavefront, or over each 16 of them.
template <int CTRL, int ROWS> __device__ __forceinline__ u64 dpp_add(u64 x) {
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (unsigned)x, CTRL, ROWS, 0xf, true), hi = __builtin_amdgcn_update_dpp(0, (unsigned)(x >> 32), CTRL, ROWS, 0xf, true);
  return x + ((u64)hi << 32 | lo);
}
__device__ __forceinline__ u64 row_scan(u64 x) { return dpp_add<0x118, 0xf>(dpp_add<0x114, 0xf>(dpp_add<0x112, 0xf>(dpp_add<0x111, 0xf>(x)))); }   // row_shr:1, 2, 4, 8
__device__ __forceinline__ u64 wave_scan(u64 x) { return dpp_add<0x143, 0xc>(dpp_add<0x142, 0xa>(row_scan(x))); }   // row_bcast:15, row_bcast:31
__device__ __forceinline__ u64 read_lane(u64 x, int lane) {
  return (u64)(unsigned)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 | (unsigned)__builtin_amdgcn_readlane((int)x, lane);
}

struct Shared {
  double table[OCTAVE];
  u64 mass[BUCKETS], finer[BUCKETS];        // of the first division, and of further ones
  unsigned count[BUCKETS], finer_count[BUCKETS];
  u64 list[LIST], ordered[LIST];
  unsigned rank[256];
  u64 wave[2][WAVES];
  float wave_max[WAVES];
  u64 found[2], least;
  unsigned words[4];
};
static_assert(WAVES == 16, "a row of 16 lanes sums up the wavefronts");

// Exclusive sum over the block; `all`: of all threads.  Calls take turns with `k`.
__device__ __forceinline__ u64 block_scan(Shared& s, int k, u64 x, u64& all) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const u64 upto = wave_scan(x);
  if (lane == 63) s.wave[k][wave] = upto;
  __syncthreads();
  const u64 waves = row_scan(s.wave[k][lane & 15]);
  all = read_lane(waves, 15);
  const u64 before = wave ? read_lane(waves, wave - 1) : 0;
  return before + upto - x;
}

template <typename T, int NV>
struct Sampler {
  Shared& s;
  Row<T, NV>& row;
  Weights w;

  // s.list's n entries in rising order to s.ordered.
  __device__ void order(int n) {
    const int tid = threadIdx.x;
    if (n <= 256) {   // by the number of smaller ones, which 1024 / 64, 1024 / 128 or 1024 / 256 threads count for each
      const int size = n <= 64 ? 64 : n <= 128 ? 128 : 256, i = tid & (size - 1), parts = THREADS / size, part = tid / size, each = (n + parts - 1) / parts;
      if (tid < size) s.rank[tid] = 0;
      __syncthreads();
      if (i < n) {
        const u64 mine = s.list[i];
        unsigned smaller = 0;
        for (int j = part * each; j < min(n, (part + 1) * each); j++) smaller += s.list[j] < mine;
        atomicAdd(&s.rank[i], smaller);
      }
      __syncthreads();
      if (tid < n) s.ordered[s.rank[tid]] = s.list[tid];
      __syncthreads();
      return;
    }
    int size = 512;
    while (size < n) size *= 2;
    for (int i = tid; i < size; i += THREADS) s.ordered[i] = i < n ? s.list[i] : ~0ull;
    for (int k = 2; k <= size; k *= 2)
      for (int j = k / 2; j > 0; j /= 2) {
        __syncthreads();
        for (int i = tid; i < size / 2; i += THREADS) {
          const int a = 2 * i - (i & (j - 1)), b = a + j;
          const u64 x = s.ordered[a], y = s.ordered[b];
          if ((x > y) == ((a & k) == 0)) s.ordered[a] = y, s.ordered[b] = x;
        }
      }
    __syncthreads();
  }

  // Tokens for which keep(x) holds into s.list, as (falling key, index); how many there are, which may be more than fit.
  template <bool AGAIN, typename F> __device__ __forceinline__ int gather(F keep) {
    __syncthreads();
    if (threadIdx.x == 0) s.words[0] = 0;
    __syncthreads();
    auto take = [&](float x, int i) __attribute__((always_inline)) {
      const unsigned at = atomicAdd(&s.words[0], 1u);
      if (at < LIST) s.list[at] = (u64)~key_of(x) << 32 | (unsigned)i;
    };
    if constexpr (AGAIN) row.again([&](float x, int v, int e) { if (keep(x)) take(x, row.index(v, e)); });
    else row.matches(keep, take);
    __syncthreads();
    return (int)s.words[0];
  }

  static constexpr int PER = LIST / THREADS;   // entries of the ordered list a thread
  // Sums of the weights up to and with each entry of a thread, `mass` before all of them; without an entry that of the one before.
  __device__ u64 sums(int n, u64 mass, u64 (&upto)[PER], u64 (&was)[PER]) {
    u64 mine[PER], sum = 0, all;
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int i = threadIdx.x * PER + k;
      if (i < n) sum += w.of(of_key(~(unsigned)(s.ordered[i] >> 32)));
      mine[k] = sum;
    }
    const u64 before = mass + block_scan(s, 0, sum, all);
#pragma unroll
    for (int k = 0; k < PER; k++) upto[k] = before + mine[k], was[k] = k ? upto[k - 1] : before;
    return mass + all;
  }
  // The first of the n ordered entries at which the sum (of tokens, or of weights) behind `before` reaches the target: its entry, and the sum of weights up to and with it.
  __device__ void reach(int n, bool by_count, u64 target, u64 count, u64 mass, u64& entry, u64& mass_upto) {
    u64 upto[PER], was[PER];
    sums(n, mass, upto, was);
    find(n, by_count, target, count, upto, was, entry, mass_upto);
  }
  __device__ void find(int n, bool by_count, u64 target, u64 count, const u64 (&upto)[PER], const u64 (&was)[PER], u64& entry, u64& mass_upto) {
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int i = threadIdx.x * PER + k;
      if (i < n && (by_count ? count + i + 1 == target : was[k] < target && upto[k] >= target)) s.found[0] = s.ordered[i], s.found[1] = upto[k];
    }
    __syncthreads();
    entry = s.found[0], mass_upto = s.found[1];
  }

  // The bucket in which the sum reaches the target; the sums before it are added to `count` and `mass`.
  __device__ int bucket_of(const u64* masses, const unsigned* counts, bool by_count, bool both, u64 target, u64& count, u64& mass) {
    constexpr int EACH = BUCKETS / THREADS;
    const int b0 = threadIdx.x * EACH;
    u64 sum = 0, tokens = 0, all, c = count;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EACH; k++) sum += masses[b0 + k], tokens += counts[b0 + k];
    u64 m = mass + block_scan(s, 0, sum, all);
    if (both) c += block_scan(s, 1, tokens, all);
#pragma unroll
    for (int k = 0; k < EACH; k++) {
      const u64 m1 = m + masses[b0 + k], c1 = c + counts[b0 + k];
      if (by_count ? c < target && c1 >= target : m < target && m1 >= target) s.words[1] = b0 + k, s.found[0] = c, s.found[1] = m;
      m = m1, c = c1;
    }
    __syncthreads();
    count = s.found[0], mass = s.found[1];
    return s.words[1];
  }

  // The `nth` (from 1) token with this key, by its index.
  __device__ int nth_of(unsigned key, unsigned nth) {
    unsigned* counts = reinterpret_cast<unsigned*>(s.list);   // [turn][wavefront]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, turns = (row.vectors + THREADS - 1) / THREADS;
    __syncthreads();
    auto matches = [&](int turn, unsigned& mask) {
      mask = 0;
      row.turn(turn, [&](float x, int, int e) { if (key_of(x) == key) mask |= 1u << e; });
    };
    for (int turn = 0; turn < turns; turn++) {
      unsigned mask;
      matches(turn, mask);
      const unsigned upto = (unsigned)wave_scan(__popc(mask));
      if (lane == 63) counts[turn * WAVES + wave] = upto;
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
      const unsigned mine = __popc(mask), upto = (unsigned)wave_scan(mine);
      unsigned left = s.words[3];
      if (upto - mine < left && upto >= left) {
        left -= upto - mine;
        while (--left) mask &= mask - 1;
        s.words[1] = row.index(turn, __ffs(mask) - 1);
      }
    }
    __syncthreads();
    return s.words[1];
  }

  // Sum of the weights that are not less than `least`.
  __device__ u64 heavy(u64 least) {
    u64 sum = 0, all;
    row.again([&](float x, int, int) {
      const u64 wt = w.of(x);
      if (wt >= least) sum += wt;
    });
    block_scan(s, 1, sum, all);
    return all;
  }

  // Where the sum reaches the target, among the tokens of a bucket, `count` and `mass` before them: the entry (falling key, index), and the weights up to and with it.
  __device__ void resolve(unsigned bucket, bool by_count, u64 target, u64 count, u64 mass, bool want_index, u64& entry, u64& mass_upto) {
    const auto in = [&](float x) __attribute__((always_inline)) { return w.bucket(x) == bucket; };
    int n = gather<false>(in);
    if (n <= LIST) {
      order(n);
      reach(n, by_count, target, count, mass, entry, mass_upto);
      return;
    }
    // many: the keys that they lie between, and from there on by those
    if (threadIdx.x == 0) s.words[2] = ~0u, s.words[3] = 0;
    __syncthreads();
    unsigned lo = ~0u, hi = 0;
    row.again([&](float x, int, int) {
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
      __syncthreads();
      for (int b = threadIdx.x; b < BUCKETS; b += THREADS) s.finer[b] = 0, s.finer_count[b] = 0;
      __syncthreads();
      row.again([&](float x, int, int) {
        const unsigned k = key_of(x);
        if (k >= lo && k <= hi) {
          atomicAdd(&s.finer[(hi - k) >> shift], w.of(x));
          atomicAdd(&s.finer_count[(hi - k) >> shift], 1u);
        }
      });
      const int b = bucket_of(s.finer, s.finer_count, by_count, true, target, count, mass);
      hi -= (unsigned)b << shift;
      if (hi - lo >= 1u << shift) lo = hi - ((1u << shift) - 1);
      n = gather<true>([&](float x) { return key_of(x) >= lo && key_of(x) <= hi; });
      if (n <= LIST) {
        order(n);
        reach(n, by_count, target, count, mass, entry, mass_upto);
        return;
      }
    }
  }
};

template <typename T, int NV>
__global__ __launch_bounds__(THREADS) void sample_kernel(const SampleParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Row<T, NV> row(static_cast<const T*>(p.logits) + r * p.row_stride, p.vocab);
  const float temperature = p.temperature ? p.temperature[r] : p.temperature_all, top_p = p.top_p ? p.top_p[r] : p.top_p_all,
              min_p = p.min_p ? p.min_p[r] : p.min_p_all, u = p.u[r];
  const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  s.table[tid] = POWERS.x[0][tid >> 5] * POWERS.x[1][tid & 31];
  for (int b = tid; b < BUCKETS; b += THREADS) s.mass[b] = 0, s.count[b] = 0;
  static_assert(OCTAVE == THREADS, "a thread for each entry");

  float largest = -INFINITY;
  row.all([&](float x, int, int) { largest = fmaxf(largest, x); });   // of a NaN and a number the number
#pragma unroll
  for (int d = 1; d < 64; d *= 2) largest = fmaxf(largest, __shfl_xor(largest, d, 64));
  if (lane == 0) s.wave_max[wave] = largest;
  if (tid == 0) s.words[1] = 0x7fffffff, s.least = ~0ull;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < WAVES; k++) largest = fmaxf(largest, s.wave_max[k]);
  if (largest == -INFINITY || !(temperature > 0.f)) {   // nothing to choose from, or nothing but the first
    if (largest != -INFINITY) {
      int at = 0x7fffffff;
      row.again([&](float x, int v, int e) { if (x == largest) at = min(at, row.index(v, e)); });
      if (at != 0x7fffffff) atomicMin(&s.words[1], (unsigned)at);
      __syncthreads();
    }
    if (tid == 0) {
      p.tokens[r] = largest == -INFINITY ? -1 : (int64_t)s.words[1];
      p.logprobs[r] = largest == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  if (largest == INFINITY) {
    row.only_infinite();
    largest = 0.f;
  }
  Sampler<T, NV> a{s, row, Weights{OCTAVE * 1.4426950408889634 / (double)temperature, (double)largest, __builtin_bit_cast(double, (u64)(1023 + 52 - p.frac) << 52), largest, s.table}};
  const u64 one = 1ull << p.frac;
  const bool cut_k = top_k > 0 && top_k < p.vocab, cut_p = top_p < 1.f, cut_m = min_p > 0.f;
  const u64 least = cut_m ? (u64)fmin(ceil((double)min_p * (double)one), 9e18) : 0;
  auto target_p = [&](u64 kept) { return max((u64)1, (u64)ceil(fmax((double)top_p, 0.0) * (double)kept)); };
  auto target_u = [&](u64 kept) {
    const double share = (double)u * (double)kept;
    return share > 0.0 ? min((u64)fmin(share, 9e18) + 1, kept) : (u64)1;
  };
  u64 entry = 0, kept = 0;

  // ---- few: all that may be among the first top_k into the list
  bool few = cut_k && top_k <= LIST / 2;
  if (few) {
    row.all([&](float x, int, int) { atomicAdd(&s.count[a.w.plain_bucket(x)], 1u); });
    u64 count = 0, mass = 0;
    const unsigned last = a.bucket_of(s.mass, s.count, true, true, top_k, count, mass);
    const int n = a.template gather<false>([&](float x) { return a.w.plain_bucket(x) <= last; });
    few = n <= LIST;
    if (few) {
      a.order(n);
      const int k = min(n, top_k);
      u64 upto[a.PER], was[a.PER], upto_p;
      kept = a.sums(k, 0, upto, was);
      if (cut_p) {
        a.find(k, false, target_p(kept), 0, upto, was, entry, upto_p);
        kept = min(kept, upto_p);
      }
      if (cut_m) {   // up to the last one that is heavy enough
        u64 over = one;
#pragma unroll
        for (int j = 0; j < a.PER; j++)
          if (tid * a.PER + j < k && upto[j] - was[j] >= least) over = max(over, upto[j]);
        __syncthreads();
        if (tid == 0) s.least = 0;
        __syncthreads();
        atomicMax(&s.least, over);
        __syncthreads();
        kept = min(kept, s.least);
      }
      __syncthreads();
      a.find(k, false, target_u(kept), 0, upto, was, entry, upto_p);
    } else {
      __syncthreads();
      for (int b = tid; b < BUCKETS; b += THREADS) s.count[b] = 0;
    }
  }

  // ---- sums of the weights by buckets of all
  if (!few) {
    __syncthreads();
    row.all([&](float x, int, int) {
      unsigned b;
      const u64 wt = a.w.of(x, b);
      atomicAdd(&s.mass[b], wt);
    });
    if (cut_k) row.again([&](float x, int, int) { atomicAdd(&s.count[a.w.bucket(x)], 1u); });
    __syncthreads();
    u64 sum = 0, over = 0;
    for (int b = tid; b < BUCKETS; b += THREADS) sum += s.mass[b];
    block_scan(s, 0, sum, kept);
    if (cut_m) over = max(one, a.heavy(least));   // the first one at any rate
    for (int step = cut_k ? 0 : cut_p ? 1 : 2; step < 3; step++) {
      if (step == 1 && !cut_p) continue;
      if (step == 2 && cut_m) kept = min(kept, over);
      const u64 target = step == 0 ? (u64)top_k : step == 1 ? target_p(kept) : target_u(kept);
      u64 count = 0, mass = 0, upto;
      __syncthreads();
      const unsigned b = a.bucket_of(s.mass, s.count, step == 0, step == 0, target, count, mass);
      a.resolve(b, step == 0, target, count, mass, step == 2, entry, upto);
      if (step < 2) kept = min(kept, upto);
    }
  }
  if (tid == 0) {
    p.tokens[r] = (int64_t)(unsigned)entry;
    const double log2w = -a.w.steps(of_key(~(unsigned)(entry >> 32))) / OCTAVE;
    p.logprobs[r] = (float)((log2w + p.frac) * 0.6931471805599453 - log((double)kept));
  }
}

template <typename T, int NV>
int launch(const SampleParams& p, int rows, hipStream_t st) {
  if (int rc = ody_allow_dynamic_lds(reinterpret_cast<const void*>(&sample_kernel<T, NV>), sizeof(Shared), "ody_sample")) return rc;
  ODY_LAUNCH("sample", st, (sample_kernel<T, NV>), dim3((unsigned)rows), dim3(THREADS), sizeof(Shared), p);
  return ody_check_launch("sample");
}
template <typename T>
int by_length(const SampleParams& p, int rows, hipStream_t st) {
  constexpr int N = 16 / (int)sizeof(T);
  const int turns = (p.vocab + 2 * N - 2 + THREADS * N - 1) / (THREADS * N);   // however rows are aligned
  if (turns <= 4) return launch<T, 4>(p, rows, st);
  if (turns <= 8) return launch<T, 8>(p, rows, st);
  if (turns <= 16) return launch<T, 16>(p, rows, st);
  return launch<T, 0>(p, rows, st);
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
  return dtype == ODY_BF16 ? by_length<bf16>(p, rows, st) : by_length<float>(p, rows, st);
}
