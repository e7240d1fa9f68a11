// A token of each row of logits, by temperature, top-k, top-p and min-p, from a given random number.
//
// The order of a row's tokens is by falling logits, the lower index first among equals.  Each cut leaves a prefix of that order, and the token is where the sums of the
// weights exp((x - max) / T) along it pass the random number's share of what is kept: all of it asks for one thing, the first token at which a sum along the order (of
// tokens, or of weights) reaches a target.  No row is sorted for that:
//
//   bf16   There are few values.  Tokens are counted by value -- 8192 of them, 32 octaves of either sign, from the largest that can have a weight down; the few tokens nearer to 0
//          keep weights of their own -- and a weight is formed for each value and not for each token.
//   fp32   Sums of the weights by buckets of x, 2048 of them, say which bucket the place is in; the bucket's tokens, a few as a rule, are gathered and ordered.  Where top_k is small the
//          buckets count tokens, what may be among the first is gathered, and nothing else has a weight formed.
//
// What is gathered and too many to be ordered is divided by the bits of x, until it is few or has one value.
//
// Weights are whole numbers of 2^-FRAC: sums in any order, by atomics too, are the same.  FRAC is 50, or, for rows beyond 16382, what is left of 64 bits for a sum of all weights, of at most 1, and one more:
// 47 for a vocabulary of 128000, 43 for the longest rows.  They are formed in 64 bits, whose vector rate is that of 32 here, as 2^-(n / 1024) 2^(-r / 1024), |r| <= 1 / 2, from a table and a polynomial of the
// second degree (bf16: of the third, for what a value's weight is times a factor for each of up to fifteen steps): off by 2^-37 of themselves at most and by half of 2^-FRAC.  Both can have one direction in all of a tail of equals, so that a sum is off by 2^-37 of itself and vocab 2^-(FRAC + 1), 2^-31 for
// 128000 and 2^-23 for the longest rows, where the largest weight is 1: as near to a border of its share a random number may give the token on its other side.
//
// A block has a row.  bf16: counting is one pass, finding the tokens of the value that the place is in another; up to 32 754 tokens the row stays in registers between them, a longer one is read again
// from its end, of which the caches have more.  fp32: the largest, then sums (or counts), then what is gathered, each a pass.
//
// Bound by latencies for few rows, a chain of some thirty barriers and LDS reads behind a load: one of 32000 in bf16 13.0 us, of which counting takes 1.8.  For many by LDS atomics and the second
// reading: 256 of 128000, 37.4 us, of which counting takes 11 (8 atomics a vector, 5.5 of their lanes a cycle and compute unit, as they meet in banks; the bytes take 12.9 at a copy's rate) and the
// second pass 9.  fp32 by the instructions of the weights, 30 for each: 64 rows of 32001, a third of them without top_k, 23.4 us, of which weights take some 6.  A block has
// 145 KB of LDS, so that a compute unit has one: of more rows than there are the others wait for whole chains (512 rows of 32000 in bf16 28 us, 490 of 11166 in fp32 27).  Lists of more than 256 are sorted with a
// barrier for each of 45 steps and more (two fp32 rows of 81959, top_k 351 32 us, 1000 37; top_k 200 24.7); an fp32 row with a top_k above 2048 is one block's (250000 logits 148 us).  The blocks of 1024 threads leave 128
// registers: 18 go to memory.
//
// Few long rows would leave most compute units idle: they go in slices, a block each, with what the slices have to know of one another between launches (sums are of whole numbers, so a row's result
// is the same to the bit).  bf16 in two: counts; then every block adds up the slices' counts, finds the value and whose slice has its token.  fp32 in four: the largest; sums by buckets; what is in the
// buckets that matter, into a list; the token.  Tried: the list's last writer going on by itself, for the fourth launch; the fences that this takes write back and empty whole caches (64 rows of 128000 83 us, 41 so).
#include <algorithm>
#include <cmath>
#include "ody_common.h"

namespace {

typedef unsigned long long u64;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef const u32x4 __attribute__((address_space(1)))* vector_ptr;

constexpr int BUCKETS = 2048, LIST = 4096, OCTAVE = 1024, VALUES = 8192;
// Threads of a block.  fp32 rows are read and weighed by all that a compute unit has (256 rows of 128000 78 us, 84 by 512; 64 of 32001 23.4 and 25.6).  bf16 by 512, in whose registers short rows stay (512 rows of
// 32000 30 us, 45 by 1024; 256 of 128000 37.5 and 35.4).
struct ShortRow {   // fp32, of a short row
  float x;
};
template <typename T> constexpr int THREADS_OF = 512;
template <> constexpr int THREADS_OF<float> = 1024;
constexpr int MOST = (1 << 21) - 4;   // tokens of a row: nth_of() counts the matches in each 64 vectors, of 4 values or 8, in 2 * LIST numbers

// What finding the token among listed ones takes: top_p's weights, those before its bucket, before the random number's; of the list those before top_p's bucket
struct Ends {
  u64 target, mass, mass_u, in_front;
};
struct RowEnds {
  Ends q;
  u64 kept, most;   // all weights; what min_p keeps of them
};
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
  // a row in `slices` of `slice` tokens: results of the slices, [row][slice][BUCKETS]; of bf16 rows [row][slice][VALUES]
  int slices, slice;
  u64 *mass, *over;        // sums of the weights by buckets, or (counts) of the tokens; what min_p keeps of a slice
  unsigned* counts;
  int2* ends;              // bf16: the least and the largest bits
  float* largest;
  unsigned* listed;        // [row]: entries of its list
  RowEnds* ends_of_rows;
  u64* lists;              // [row][LIST]
};

// x as a number whose order is that of the logits: -0 as 0, NaN as the lowest
__device__ __forceinline__ unsigned key_of(float x) {
  x = x == x ? x + 0.f : -INFINITY;
  const unsigned b = __builtin_bit_cast(unsigned, x);
  return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned k) { return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// A row, in vectors of 16 bytes that hold at least one value of it.  What is not the row's counts as -inf, which has no weight and so is never a result.
template <typename T, int NV = 0>
struct Row {
  static constexpr int THREADS = THREADS_OF<T>, N = 16 / (int)sizeof(T), AHEAD = 4;   // values of a vector; vectors under way, where they are read for each pass
  static constexpr unsigned LOWEST = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;   // -inf
  const T* base;      // 16-byte aligned, at most N - 1 values before the row
  int head, vocab, vectors;
  u32x4 held[NV > 0 ? NV : 1];   // NV: the thread's vectors, all of them, read once

  __device__ __forceinline__ Row(const T* row, int vocab_) : vocab(vocab_) {
    head = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    base = row - head;
    vectors = (head + vocab + N - 1) / N;
    if constexpr (NV > 0) {
      const int tid = threadIdx.x;
#pragma unroll
      for (int k = 0; k < NV; k++) held[k] = ((vector_ptr)base)[min(k * THREADS + tid, vectors - 1)];
      if (tid == 0) held[0] = without(held[0], 0);
      const u32x4 last = without(((vector_ptr)base)[vectors - 1], vectors - 1), none = {LOWEST, LOWEST, LOWEST, LOWEST};
#pragma unroll
      for (int k = 0; k < NV; k++) {
        const int at = k * THREADS + tid;
        if ((k + 1) * THREADS >= vectors) held[k] = at < vectors - 1 ? held[k] : at == vectors - 1 ? last : none;
      }
    }
  }
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
  __device__ __forceinline__ int index(int at, int e) const { return at * N - head + e; }
  // What vector `at`, which was read, holds of the row.
  __device__ __forceinline__ u32x4 of_row(u32x4 raw, int at) const {
    if (at * N < head || (at + 1) * N > head + vocab) raw = without(raw, at);   // the first and the last one, and those behind
    return raw;
  }
  __device__ __forceinline__ u32x4 read(int at) const { return of_row(((vector_ptr)base)[min(at, vectors - 1)], at); }
  // f(vector, turn) for each of a thread's vectors, which are THREADS apart
  template <typename F> __device__ __forceinline__ void each(F f) {
    if constexpr (NV > 0) {
#pragma unroll
      for (int k = 0; k < NV; k++) {
        asm volatile("" : "+v"(held[k]));   // what one pass makes of a vector is not kept for the next one
        f(held[k], k);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      again([&](const u32x4& raw, int at) __attribute__((always_inline)) { f(raw, at / THREADS); });
    }
  }
  // ... from memory, by its number, AHEAD of them under way; code of one length for all rows.  Threads without one in the last turn have what is nowhere in the row.
  template <bool BACK = false, typename F> __device__ __forceinline__ void again(F f) const {
    again<BACK>(f, [](int) {});
  }
  // behind(turns): now and then, and at the end.  BACK: from the row's end, which is what a cache has of a long row that was read before.
  template <bool BACK = false, typename F, typename G> __device__ __forceinline__ void again(F f, G behind) const {
    const int tid = threadIdx.x, turns = (vectors + THREADS - 1) / THREADS, last = min(tid, vectors - 1 - (turns - 1) * THREADS);
    auto load = [&](int turn) __attribute__((always_inline)) {
      turn = BACK ? max(turns - 1 - turn, 0) : min(turn, turns - 1);
      return ((vector_ptr)base + turn * THREADS)[turn < turns - 1 ? tid : last];
    };
    u32x4 next[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; k++) next[k] = load(k);
    for (int turn = 0; turn < turns; turn += AHEAD) {
#pragma unroll
      for (int k = 0; k < AHEAD; k++) {
        if (turn + k >= turns) break;
        u32x4 raw = next[k];
        next[k] = load(turn + k + AHEAD);
        const int at = (BACK ? turns - 1 - (turn + k) : turn + k) * THREADS + tid;
        if (turn + k == 0 || turn + k == turns - 1) raw = of_row(raw, at);
        f(raw, at);
      }
      behind(min(turn + AHEAD, turns));
    }
  }
  // f(x, vector, element) for each value
  template <typename F> __device__ __forceinline__ void all(F f) const {
    again([&](const u32x4& raw, int at) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < N; e++) f(element(raw, e), at, e);
    });
  }
  // f(mask, turn): of TURNS turns of a thread's vectors, from `turn` on, a bit for each x for which keep(x) holds, which are few: a wavefront goes as often over them as its busiest thread has.
  template <typename K, typename F> __device__ __forceinline__ void masks(K keep, F f) const {
    constexpr int TURNS = 64 / N;
    static_assert(TURNS % AHEAD == 0, "the bits of whole turns");
    u64 mask = 0;
    again(
        [&](const u32x4& raw, int at) __attribute__((always_inline)) {
          unsigned those = 0;
#pragma unroll
          for (int e = 0; e < N; e++) those |= keep(element(raw, e)) ? 1u << e : 0u;
          mask |= (u64)those << at / THREADS % TURNS * N;
        },
        [&](int turns) __attribute__((always_inline)) {
          if (turns % TURNS && turns * THREADS < vectors) return;
          f(mask, (turns - 1) / TURNS * TURNS);
          mask = 0;
        });
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (sizeof(T) == 4) return ((const float __attribute__((address_space(1)))*)base)[head + i];
    else return (float)((const T __attribute__((address_space(1)))*)base)[head + i];
  }
  // f(x, index) for every x of the row for which keep(x) holds, which are few
  template <typename K, typename F> __device__ __forceinline__ void matches(K keep, F f) const {
    masks(keep, [&](u64 mask, int turn) __attribute__((always_inline)) {
      while (mask) {
        const int bit = __ffsll(mask) - 1, i = index((turn + bit / N) * THREADS + (int)threadIdx.x, bit % N);
        mask &= mask - 1;
        if ((unsigned)i < (unsigned)vocab) f(value(i), i);
      }
    });
  }
  // ---- bf16
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ u16x2 lower(u16x2 a, u16x2 b) { return __builtin_elementwise_min(a, b); }
  // count[] by value, VALUES / 2 - 1 - d or VALUES / 2 + d for the bits base + d of the positive or the negative value.  Others, NaN among them, are not counted: bits below the base, of which
  // `least` tells, positive ones beyond, of which `most` tells, and negative ones beyond.
  __device__ __forceinline__ void count_values(unsigned* count, unsigned base, unsigned& least, int& most) {
    const u16x2 from = {(unsigned short)base, (unsigned short)base};
    u16x2 l = {0xffff, 0xffff};
    i16x2 g = {-0x8000, -0x8000};
    each([&](const u32x4& raw, int) __attribute__((always_inline)) {
#pragma unroll
      for (int w = 0; w < 4; w++) {
        const unsigned word = raw[w];
        const i16x2 both = __builtin_bit_cast(i16x2, word);
        const u16x2 size = __builtin_bit_cast(u16x2, word & 0x7fff7fffu), sign = __builtin_bit_cast(u16x2, both >> 15);
        const u16x2 d = size - from, place = (u16x2){VALUES / 2 - 1, VALUES / 2 - 1} - (d ^ sign);
        l = lower(l, size), g = __builtin_elementwise_max(g, both);
        if (d[0] < VALUES / 2) atomicAdd(&count[place[0]], 1u);
        if (d[1] < VALUES / 2) atomicAdd(&count[place[1]], 1u);
      }
    });
    least = min(l[0], l[1]), most = max(g[0], g[1]);
  }
  // f(x, index) of every x with these bits, of which there are few: a bit for each in what four vectors leave clear of 32
  template <typename F> __device__ __forceinline__ void equals(unsigned bits, F f) {
    static_assert(AHEAD == 4 && NV % 4 == 0, "vectors of a mask");
    const unsigned both = bits << 16 | bits;
    auto others = [&](const u32x4& raw) __attribute__((always_inline)) {   // bits w and 16 + w: elements 2 w and 2 w + 1 are others
      unsigned mask = 0;
#pragma unroll
      for (int w = 0; w < 4; w++) mask |= __builtin_bit_cast(unsigned, lower(__builtin_bit_cast(u16x2, raw[w] ^ both), (u16x2){1, 1})) << w;
      return mask;
    };
    auto take = [&](unsigned mask, auto turn) __attribute__((always_inline)) {
      while (mask) {
        const int bit = __ffs(mask) - 1;
        mask &= mask - 1;
        f(__builtin_bit_cast(float, bits << 16), index(turn(bit >> 2 & 3) * THREADS + (int)threadIdx.x, 2 * (bit & 3) + (bit >> 4)));
      }
    };
    if constexpr (NV > 0) {
      unsigned mask[NV / 4] = {};
      each([&](const u32x4& raw, int k) __attribute__((always_inline)) { mask[k / 4] |= others(raw) << 4 * (k % 4); });
#pragma unroll
      for (int i = 0; i < NV / 4; i++) take(~mask[i], [&](int k) __attribute__((always_inline)) { return 4 * i + k; });
    } else {
      const int turns = (vectors + THREADS - 1) / THREADS;
      unsigned mask = ~0u;
      int k = 0;
      again<true>([&](const u32x4& raw, int) __attribute__((always_inline)) { mask ^= (others(raw) ^ 0xf000fu) << 4 * (k++ & 3); },
                  [&](int behind) __attribute__((always_inline)) {
                    if (mask != ~0u) take(~mask, [&](int j) __attribute__((always_inline)) { return turns - 1 - ((behind - 1) / 4 * 4 + j); });
                    mask = ~0u;
                  });
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
  __device__ __forceinline__ float plain(float x) const { return (topf - x) * 64.f; }
  __device__ __forceinline__ unsigned plain_bucket(float x) const { return (unsigned)fminf(plain(x), (float)(BUCKETS - 1)); }
  // 2^(-t / OCTAVE), 0 <= t; n: t to the nearest.  TERMS of the series: two leave 2^-37, three 2^-48
  template <int TERMS = 2> __device__ __forceinline__ double power(double t, unsigned& n) const {
    double r;
    n = nearest(t, r);
    constexpr double L = -0.6931471805599453 / OCTAVE;
    const double p = fma(fma(TERMS == 3 ? fma(L * L * L / 6, r, L * L / 2) : L * L / 2, r, L), r, 1.0);
    u64 e = __builtin_bit_cast(u64, table[n % OCTAVE]);
    e = (u64)((unsigned)(e >> 32) - (n / OCTAVE << 20)) << 32 | (unsigned)e;
    return __builtin_bit_cast(double, e) * p;
  }
  __device__ __forceinline__ u64 whole(double weight) const {
#pragma clang fp contract(off)   // the same bits wherever it is formed
    return __builtin_bit_cast(u64, weight + magic) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 of(float x, unsigned& bucket) const {
    unsigned n;
    const double weight = power(steps(x), n);
    bucket = bucket_of(n);
    return whole(weight);
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
  unsigned count[VALUES], finer_count[BUCKETS];
  u64 list[LIST], ordered[LIST];
  unsigned rank[256];
  u64 wave[16];
  float wave_max[16];
  u64 found[3], small[2];
  unsigned words[4], small_tokens;
};

// Exclusive sum over the block; `all`: of all threads.
template <typename T> __device__ __forceinline__ u64 block_scan(Shared& s, u64 x, u64& all) {
  constexpr int WAVES = THREADS_OF<T> / 64;
  static_assert(WAVES <= 16, "a row of 16 lanes sums up the wavefronts");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const u64 upto = wave_scan(x);
  __syncthreads();   // a sum before this one has been read
  if (lane == 63) s.wave[wave] = upto;
  __syncthreads();
  const u64 waves = row_scan(s.wave[lane & (WAVES - 1)]);
  all = read_lane(waves, WAVES - 1);
  const u64 before = wave ? read_lane(waves, wave - 1) : 0;
  return before + upto - x;
}

template <typename T, int NV = 0>
struct Sampler {
  static constexpr int THREADS = THREADS_OF<T>, WAVES = THREADS / 64;
  Shared& s;
  Row<T, NV>& row;
  Weights w;

  // s.list's n entries in rising order to s.ordered.
  __device__ __forceinline__ void order(int n) {
    const int tid = threadIdx.x;
    if (n <= 256) {   // by the number of smaller ones, which THREADS / 64, / 128 or / 256 threads count for each
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
  template <typename F> __device__ __forceinline__ int gather(F keep) {
    return listed([&](auto take) __attribute__((always_inline)) { row.matches(keep, take); });
  }
  // ... for which beyond(x) is not above 0, which it is for -inf
  template <typename F> __device__ __forceinline__ int gather_within(F beyond) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid == 0) s.words[0] = 0;
    __syncthreads();
    row.masks([&](float x) __attribute__((always_inline)) { return beyond(x) <= 0.f; }, [&](u64 mask, int turn) __attribute__((always_inline)) {
      if (mask == 0) return;
      unsigned to = atomicAdd(&s.words[0], (unsigned)__popcll(mask));
      for (; mask && to < LIST; to++) {
        const int bit = __ffsll(mask) - 1;
        mask &= mask - 1;
        s.list[to] = (u64)row.index((turn + bit / row.N) * THREADS + tid, bit % row.N);
      }
    });
    __syncthreads();
    const int n = (int)s.words[0];
    if (n > LIST) return n;
    for (int k = tid; k < n; k += THREADS) {   // their values at once
      const unsigned i = (unsigned)s.list[k];
      s.list[k] = (u64)~key_of(row.value(i)) << 32 | i;
    }
    __syncthreads();
    return n;
  }
  template <typename F> __device__ __forceinline__ int listed(F walk) {
    __syncthreads();
    if (threadIdx.x == 0) s.words[0] = 0;
    __syncthreads();
    walk([&](float x, int i) __attribute__((always_inline)) {
      const unsigned at = atomicAdd(&s.words[0], 1u);
      if (at < LIST) s.list[at] = (u64)~key_of(x) << 32 | (unsigned)i;
    });
    __syncthreads();
    return (int)s.words[0];
  }

  static constexpr int PER = LIST / THREADS;   // entries of the ordered list a thread
  // Sums of the weights up to and with each entry of a thread, `mass` before all of them; without an entry that of the one before.
  __device__ __forceinline__ u64 sums(int n, u64 mass, u64 (&upto)[PER], u64 (&was)[PER]) {
    u64 mine[PER], sum = 0, all;
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int i = threadIdx.x * PER + k;
      if (i < n) sum += w.of(of_key(~(unsigned)(s.ordered[i] >> 32)));
      mine[k] = sum;
    }
    const u64 before = mass + block_scan<T>(s, sum, all);
#pragma unroll
    for (int k = 0; k < PER; k++) upto[k] = before + mine[k], was[k] = k ? upto[k - 1] : before;
    return mass + all;
  }
  // The first of the n ordered entries at which the sum (of tokens, or of weights) behind `before` reaches the target: its entry, and the sum of weights up to and with it.
  __device__ __forceinline__ void reach(int n, bool by_count, u64 target, u64 count, u64 mass, u64& entry, u64& mass_upto) {
    u64 upto[PER], was[PER];
    sums(n, mass, upto, was);
    find(n, by_count, target, count, upto, was, entry, mass_upto);
  }
  __device__ __forceinline__ void find(int n, bool by_count, u64 target, u64 count, const u64 (&upto)[PER], const u64 (&was)[PER], u64& entry, u64& mass_upto) {
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int i = threadIdx.x * PER + k;
      if (i < n && (by_count ? count + i + 1 == target : was[k] < target && upto[k] >= target)) s.found[0] = s.ordered[i], s.found[1] = upto[k];
    }
    __syncthreads();
    entry = s.found[0], mass_upto = s.found[1];
  }

  // Where the sum reaches the target among a thread's SLOTS of tokens and weights, `c` and `m` before them: the slot's number, first + k, to all, with the sums before it.
  template <int SLOTS> __device__ __forceinline__ int slot_of(bool by_count, u64 target, int first, u64 c, u64 m, const unsigned (&tokens)[SLOTS], const u64 (&weights)[SLOTS], u64& count,
                                                              u64& mass) {
    __syncthreads();
    u64 weights_here = 0;
    unsigned tokens_here = 0;
#pragma unroll
    for (int k = 0; k < SLOTS; k++) weights_here += weights[k], tokens_here += tokens[k];
    if (by_count ? c < target && c + tokens_here >= target : m < target && m + weights_here >= target) {
#pragma unroll
      for (int k = 0; k < SLOTS; k++) {
        const u64 m1 = m + weights[k], c1 = c + tokens[k];
        if (by_count ? c < target && c1 >= target : m < target && m1 >= target) s.words[1] = first + k, s.found[0] = c, s.found[1] = m;
        m = m1, c = c1;
      }
    }
    __syncthreads();
    count = s.found[0], mass = s.found[1];
    return s.words[1];
  }
  // ... among buckets, `count` and `mass` before them all
  __device__ __forceinline__ int bucket_of(const u64* masses, const unsigned* counts, bool by_count, u64 target, u64& count, u64& mass) {
    constexpr int EACH = BUCKETS / THREADS;
    u64 weights[EACH], sum = 0, tokens = 0, all;
    unsigned numbers[EACH];
#pragma unroll
    for (int k = 0; k < EACH; k++) {
      const int b = threadIdx.x * EACH + k;
      weights[k] = masses ? masses[b] : 0, numbers[k] = counts[b];
      sum += weights[k], tokens += numbers[k];
    }
    const u64 m = masses ? mass + block_scan<T>(s, sum, all) : 0, c = count + block_scan<T>(s, tokens, all);
    if (by_count && count + all < target) return BUCKETS;   // fewer than that are counted
    return slot_of<EACH>(by_count, target, threadIdx.x * EACH, c, m, numbers, weights, count, mass);
  }

  // ---- fp32
  // Tokens by buckets of their values alone
  __device__ __forceinline__ void count_buckets() {
    row.all([&](float x, int, int) {
      const unsigned b = w.plain_bucket(x);
      if (b < BUCKETS - 1) atomicAdd(&s.count[b], 1u);
    });
  }
  // Sums of the weights by buckets; what a thread has of weights that are not less than `least`, where that is asked for.
  // (Many can be in the last bucket, which is everything below 2^-32: it is summed up by each thread.)
  __device__ __forceinline__ u64 add_weights(bool cut_m, u64 least) {
    u64 over = 0, tail = 0;
    const auto put = [&](u64 wt, unsigned b) __attribute__((always_inline)) {
      if (b == BUCKETS - 1) tail += wt;
      else atomicAdd(&s.mass[b], wt);
    };
    if (cut_m)
      row.all([&](float x, int, int) {
        unsigned b;
        const u64 wt = w.of(x, b);
        put(wt, b);
        over += wt >= least ? wt : 0;
      });
    else
      row.all([&](float x, int, int) {
        unsigned b;
        const u64 wt = w.of(x, b);
        put(wt, b);
      });
    tail = wave_scan(tail);
    if ((threadIdx.x & 63) == 63) atomicAdd(&s.mass[BUCKETS - 1], tail);
    return over;
  }
  // The few that may be among the first top_k, s.count by buckets: into the list.  More than LIST: not so few.
  __device__ __forceinline__ int gather_first(int top_k) {
    u64 count = 0, mass = 0;
    const int last = bucket_of(nullptr, s.count, true, top_k, count, mass);
    if (last >= BUCKETS) return LIST + 1;
    const float end = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, (float)(last + 1)) - 1);   // up to the number below it, of buckets
    return gather_within([&](float x) __attribute__((always_inline)) { return w.plain(x) - end; });
  }
  // ... of which there are n: the token's entry
  template <typename S> __device__ __forceinline__ u64 among_first(int n, const S& set, u64& kept) {
    order(n);
    const int k = min(n, set.top_k);
    u64 upto[PER], was[PER], upto_p, entry;
    kept = sums(k, 0, upto, was);
    if (set.cut_p) {
      find(k, false, set.target_p(kept), 0, upto, was, entry, upto_p);
      kept = min(kept, upto_p);
    }
    if (set.cut_m) {
      u64 over = 0, heavy;
#pragma unroll
      for (int j = 0; j < PER; j++) over += upto[j] - was[j] >= set.least && (int)threadIdx.x * PER + j < k ? upto[j] - was[j] : 0;
      block_scan<T>(s, over, heavy);
      kept = min(kept, max(set.one, heavy));   // the first one at any rate
    }
    __syncthreads();
    find(k, false, set.target_u(kept), 0, upto, was, entry, upto_p);
    return entry;
  }
  // top_p and the token in one go: whichever token of its bucket top_p ends with, the random number's is in one or two buckets, which are gathered with it.  
  static constexpr int EACH = BUCKETS / THREADS;
  // Into the list, by a thread's buckets with `m` in front of them, `kept` in all, of which min_p keeps `most`; more than LIST: too many.
  template <typename S> __device__ __forceinline__ int gather_ends(const S& set, u64 m, const u64 (&weights)[EACH], u64 kept, u64 most, Ends& q) {
    const unsigned none[EACH] = {};
    u64 count = 0, mass_v = 0;
    const auto bucket_with = [&](u64 sum, u64& before) __attribute__((always_inline)) {
      return (unsigned)slot_of<EACH>(false, sum, (int)threadIdx.x * EACH, 0, m, none, weights, count, before);
    };
    float lo, hi, lo_u, hi_u, nothing;
    q = Ends{};
    if (!set.cut_p) {
      range_of(bucket_with(set.target_u(min(kept, most)), q.mass_u), lo, hi);
      return gather_within([&](float x) __attribute__((always_inline)) { return outside(x, lo, hi); });
    }
    q.target = set.target_p(kept);
    const unsigned b = bucket_with(q.target, q.mass), u = bucket_with(set.target_u(min(most, q.mass + 1)), q.mass_u), v = bucket_with(set.target_u(min(most, q.mass + s.mass[b])), mass_v);
    q.in_front = (v == b ? q.mass : mass_v + s.mass[v]) - q.mass_u;
    range_of(b, lo, hi), range_of(u, lo_u, hi_u);
    if (v != u) range_of(v, lo_u, nothing);
    return gather_within([&](float x) __attribute__((always_inline)) { return fminf(outside(x, lo, hi), outside(x, lo_u, hi_u)); });
  }
  // The token's entry among the n of the list.
  template <typename S> __device__ __forceinline__ u64 among_ends(int n, const S& set, u64 most, const Ends& q, u64& kept) {
    u64 upto[PER], was[PER], upto_p, entry;
    order(n);
    sums(n, 0, upto, was);
    if (set.cut_p) {
      find(n, false, q.target - q.mass + q.in_front, 0, upto, was, entry, upto_p);
      kept = min(kept, q.mass + (upto_p - q.in_front));
      __syncthreads();
    }
    kept = min(kept, most);
    find(n, false, set.target_u(kept) - q.mass_u, 0, upto, was, entry, upto_p);
    return entry;
  }

  // The `nth` (from 1) token with this key, by its index.
  __device__ __forceinline__ int nth_of(unsigned key, unsigned nth) {
    unsigned* counts = reinterpret_cast<unsigned*>(s.list);   // of each 64 vectors
    const int lane = threadIdx.x & 63, groups = (row.vectors + 63) / 64;
    __syncthreads();
    auto matches = [&](int group) {
      unsigned mask = 0;
      const int at = group * 64 + lane;
      const u32x4 raw = row.read(at);
#pragma unroll
      for (int e = 0; e < row.N; e++) mask |= key_of(row.element(raw, e)) == key && at < row.vectors ? 1u << e : 0u;
      return mask;
    };
    for (int group = threadIdx.x / 64; group < groups; group += WAVES) {
      const unsigned upto = (unsigned)wave_scan(__popc(matches(group)));
      if (lane == 63) counts[group] = upto;
    }
    __syncthreads();
    if (threadIdx.x < 64) {   // the first wavefront: the group, and the token in it
      unsigned left = nth;
      int group = 0;
      for (int g = 0; g < groups; g += 64) {
        const unsigned mine = g + lane < groups ? counts[g + lane] : 0, upto = (unsigned)wave_scan(mine);
        const u64 behind = __ballot(upto >= left);
        if (behind) {
          const int k = __ffsll(behind) - 1;
          group = g + k, left -= __builtin_amdgcn_readlane(upto - mine, k);
          break;
        }
        left -= __builtin_amdgcn_readlane(upto, 63);
      }
      unsigned mask = matches(group);
      const unsigned mine = __popc(mask), upto = (unsigned)wave_scan(mine);
      if (upto - mine < left && upto >= left) {
        left -= upto - mine;
        while (--left) mask &= mask - 1;
        s.words[1] = row.index(group * 64 + lane, __ffs(mask) - 1);
      }
    }
    __syncthreads();
    return s.words[1];
  }

  // The `nth` (from 1) token with logit x: its entry.
  __device__ __forceinline__ u64 pick(float x, unsigned nth) {
    int n;
    const unsigned bits = __builtin_bit_cast(unsigned, x);
    if (sizeof(T) == 2 && x != 0.f) n = listed([&](auto take) __attribute__((always_inline)) { row.equals(bits >> 16, take); });
    else n = gather([&](float y) __attribute__((always_inline)) { return y == x; });
    return nth_listed(n, x, nth);
  }
  // ... where the list has the n tokens with it, if they are not too many
  __device__ __forceinline__ u64 nth_listed(int n, float x, unsigned nth) {
    if (n <= LIST) {
      order(n);
      return s.ordered[nth - 1];
    }
    const unsigned key = key_of(x);
    return (u64)~key << 32 | (unsigned)nth_of(key, nth);
  }

  // The least key for which holds(key), which holds for all from there up to `most`, for it too: 64 of them at once.
  template <typename F> __device__ __forceinline__ static unsigned least_key(F holds, unsigned least, unsigned most, unsigned guess) {
    const unsigned lane = threadIdx.x & 63;
    if (guess > least && guess < most && guess - least > 31 && most - guess > 31) {   // 64 around what it should be
      const u64 those = __ballot(holds(guess - 32 + lane));
      if (those >> 63 && !(those & 1)) return guess - 33 + __ffsll(those);
    }
    while (most > least) {
      const unsigned step = (most - least) / 64 + 1, at = least + lane * step;
      const u64 those = __ballot(at >= most || at < least || holds(at));   // at < least: beyond 32 bits
      const int k = those ? __ffsll(those) - 1 : 64;
      if (k < 64) most = min(most, least + k * step);
      if (k > 0) least += (k - 1) * step + 1;
      else break;
    }
    return most;
  }
  // The values of a bucket: from lo to hi.
  __device__ __forceinline__ void range_of(unsigned bucket, float& lo, float& hi) {
    const double width = OCTAVE / 64 / w.c;
    const unsigned top = key_of((float)w.top), bottom = key_of(-INFINITY);
    auto guess = [&](unsigned b) { return key_of((float)(w.top - ((double)b - 0.5 / (OCTAVE / 64)) * width)); };
    // the largest of the bucket is one below the least of the buckets in front of it
    const unsigned first = least_key([&](unsigned k) { return w.bucket(of_key(k)) <= bucket; }, bottom, top, guess(bucket + 1));
    const unsigned behind = bucket == 0 ? top + 1 : least_key([&](unsigned k) { return w.bucket(of_key(k)) < bucket; }, bottom, top, guess(bucket));
    lo = of_key(first), hi = of_key(behind - 1);
  }

  // Not above 0 from lo to hi (of which -inf is none: it has no weight); without a branch
  __device__ __forceinline__ static float outside(float x, float lo, float hi) { return fmaxf(x - hi, fmaxf(lo, -3.4028235e38f) - x); }

  // Where the sum reaches the target, among the tokens with logits from `from` to `to`, `count` and `mass` before them: the entry (falling key, index), and the weights up to and with it.
  __device__ __forceinline__ void resolve(float from, float to, bool by_count, u64 target, u64 count, u64 mass, bool want_index, u64& entry, u64& mass_upto) {
    const auto in = [&](float x) __attribute__((always_inline)) { return x >= from && x <= to; };
    int n = gather_within([&](float x) __attribute__((always_inline)) { return outside(x, from, to); });
    if (n <= LIST) {
      order(n);
      reach(n, by_count, target, count, mass, entry, mass_upto);
      return;
    }
    // many: by the bits of their keys, between the least and the largest of them
    __syncthreads();
    if (threadIdx.x == 0) s.words[2] = ~0u, s.words[3] = 0;
    __syncthreads();
    unsigned lo = ~0u, hi = 0;
    row.all([&](float x, int, int) {
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
      row.all([&](float x, int, int) {
        const unsigned k = key_of(x);
        if (k >= lo && k <= hi) {
          if (const u64 wt = w.of(x)) atomicAdd(&s.finer[(hi - k) >> shift], wt);
          atomicAdd(&s.finer_count[(hi - k) >> shift], 1u);
        }
      });
      __syncthreads();
      const int b = bucket_of(s.finer, s.finer_count, by_count, target, count, mass);
      hi -= (unsigned)b << shift;
      if (hi - lo >= 1u << shift) lo = hi - ((1u << shift) - 1);
      n = gather([&](float x) { return key_of(x) >= lo && key_of(x) <= hi; });
      if (n <= LIST) {
        order(n);
        reach(n, by_count, target, count, mass, entry, mass_upto);
        return;
      }
    }
  }
};

// What a row is sampled by.
struct Settings {
  float temperature, top_p, min_p, u;
  int top_k, frac;
  bool cut_k, cut_p, cut_m;
  u64 one, least;   // a weight of 1; the least weight that min_p keeps
  __device__ __forceinline__ Settings(const SampleParams& p, int r)
      : temperature(p.temperature ? p.temperature[r] : p.temperature_all), top_p(p.top_p ? p.top_p[r] : p.top_p_all), min_p(p.min_p ? p.min_p[r] : p.min_p_all), u(p.u[r]),
        top_k(p.top_k ? p.top_k[r] : p.top_k_all), frac(p.frac), cut_k(top_k > 0 && top_k < p.vocab), cut_p(top_p < 1.f), cut_m(min_p > 0.f), one(1ull << p.frac),
        least(cut_m ? (u64)fmin(ceil((double)min_p * (double)one), 9e18) : 0) {}
  // all that may be among the first top_k are few, and nothing else need have a weight formed
  __device__ __forceinline__ bool few() const { return cut_k && top_k <= LIST / 2; }
  // the weights with which top_p is reached, of those kept so far, and the random number's
  __device__ __forceinline__ u64 target_p(u64 kept) const {
    const u64 p64 = part(top_p);
    return max((u64)1, __umul64hi(p64, kept) + (p64 * kept != 0));
  }
  __device__ __forceinline__ u64 target_u(u64 kept) const { return u < 1.f ? min(__umul64hi(part(u), kept) + 1, kept) : kept; }
  // x 2^64 of a number below 1, without what is below 1; 0 of negative ones and NaN
  __device__ __forceinline__ static u64 part(float x) {
    const unsigned bits = __builtin_bit_cast(unsigned, x), mantissa = (bits & 0x7fffff) | 0x800000;
    const int shift = (int)(bits >> 23) - 127 + 64 - 23;   // at most 40
    return x > 0.f && shift > -24 ? shift >= 0 ? (u64)mantissa << shift : (u64)mantissa >> -shift : 0;
  }
  __device__ __forceinline__ Weights weights(float top, const double* table) const {
    return Weights{OCTAVE * 1.4426950408889634 / (double)temperature, (double)top, __builtin_bit_cast(double, (u64)(1023 + 52 - frac) << 52), top, table};
  }
};
// The least entry's token, or none.
__device__ __forceinline__ void write_first(const SampleParams& p, int r, bool none, u64 entry) {
  if (threadIdx.x != 0) return;
  p.tokens[r] = none ? -1 : (int64_t)(unsigned)entry;
  p.logprobs[r] = none ? -INFINITY : 0.f;
}
// log2 of the kept weights by 32 bits, y, and what is left of them: kept 2^-y = 1 + d, d of 2^-20 or less.
__device__ __forceinline__ void write(const SampleParams& p, int r, const Weights& w, u64 entry, u64 kept) {
  if (threadIdx.x != 0) return;
  p.tokens[r] = (int64_t)(unsigned)entry;
  const double y = __log2f((float)kept);
  unsigned n;
  const double d = (double)kept * w.power(y * OCTAVE, n) - 1.0, log2w = -w.steps(of_key(~(unsigned)(entry >> 32))) / OCTAVE;
  p.logprobs[r] = (float)((log2w + p.frac - y) * 0.6931471805599453 - (d - 0.5 * d * d));
}
// The largest of a row, for all threads.
template <typename R> __device__ __forceinline__ float largest_of(const R& row, float* wave_max) {
  float x = -INFINITY;
  row.all([&](float y, int, int) { x = fmaxf(x, y); });   // of a NaN and a number the number
#pragma unroll
  for (int d = 1; d < 64; d *= 2) x = fmaxf(x, __shfl_xor(x, d, 64));
  if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = x;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < R::THREADS / 64; k++) x = fmaxf(x, wave_max[k]);
  return x;
}
// The largest logit is +inf: those are equals with all of the weight.
template <typename S> __device__ __forceinline__ void sample_infinite(const SampleParams& p, int r, const Settings& set, S& a, Shared& s) {
  const int n = a.gather([&](float x) __attribute__((always_inline)) { return x == INFINITY; });
  u64 kept = (u64)n << set.frac;
  const auto first_with = [&](u64 sum) { return (sum + set.one - 1) >> set.frac; };
  if (set.cut_k) kept = min(kept, (u64)set.top_k << set.frac);
  if (set.cut_p) kept = min(kept, first_with(set.target_p(kept)) << set.frac);
  if (set.least > set.one) kept = set.one;
  const u64 entry = a.nth_listed(n, INFINITY, (unsigned)first_with(set.target_u(kept)));
  if (threadIdx.x == 0) p.tokens[r] = (int64_t)(unsigned)entry, p.logprobs[r] = (float)-log((double)(kept >> set.frac));
}
// 2^(-j / OCTAVE), by the series of exp around the middle: twelve terms of |x| < 0.35 leave 2^-51.  (Out of memory the table would be the first thing that a block waits for.)
template <typename T> __device__ __forceinline__ void fill_table(Shared& s) {
  for (int j = threadIdx.x; j < OCTAVE; j += THREADS_OF<T>) {
    const double x = (OCTAVE / 2 - j) * (0.6931471805599453 / OCTAVE);
    double y = 1.0;
#pragma unroll
    for (int k = 12; k > 0; k--) y = fma(y * x, 1.0 / k, 1.0);
    s.table[j] = y * 0.7071067811865476;
  }
}

// The window of counted values: bits base .. base + VALUES / 2 - 1 of either sign, below 2^most, a multiple of 128 (of which all have one exponent).
__device__ __forceinline__ unsigned base_of(int most) { return (unsigned)max(128, (most + 127) * 128 - VALUES / 2); }
constexpr int USUAL = 7;   // logits below 128: the largest need not be known to count them

constexpr int VALUES_EACH = VALUES / THREADS_OF<bf16>;   // values of a thread, of one exponent
static_assert(128 % VALUES_EACH == 0 && VALUES_EACH == 16, "values of one exponent; lanes of a row sum");

// Tokens nearer to 0 than the window keep weights of their own: their sums to s.small.
template <typename S, typename R> __device__ __forceinline__ void add_small(const Settings& set, Shared& s, S& a, const R& row, unsigned base) {
  u64 mass = 0, over = 0;
  unsigned count = 0;
  row.matches([&](float x) { return (__builtin_bit_cast(unsigned, x) >> 16 & 0x7fff) < base; }, [&](float x, int) {
    const u64 wt = a.w.of(x);
    mass += wt, over += wt >= set.least ? wt : 0, count++;
  });
  if (count) {
    atomicAdd(&s.small[0], mass), atomicAdd(&s.small[1], over);
    atomicAdd(&s.small_tokens, count);
  }
}
// The cuts, then the token, by the thread's numbers of tokens by value, which s.count has too, in a window from `base` on: its value and its number among those with it, or (`listed`) its
// entry.  `small`: s.small has what is nearer to 0.  Not WHOLE: false, where a place is among those, which a's row has not all of.
template <bool WHOLE, typename S>
__device__ __forceinline__ bool choose_value(const Settings& set, Shared& s, S& a, unsigned base, float top, const unsigned (&tokens)[VALUES_EACH], bool small, float& x, unsigned& nth,
                                             bool& listed, u64& entry, u64& kept) {
  constexpr int EACH = VALUES_EACH;
  const int tid = threadIdx.x;
  // ---- weights by value: those of a thread are evenly spaced, so that one is a constant times the one before
  const int v0 = tid * EACH;
  const bool positive = v0 < VALUES / 2;
  const unsigned bits = positive ? base + (VALUES / 2 - 1 - v0) : base + (v0 - VALUES / 2);   // of the first one; each has one less, or, among the negative ones, one more
  const float x0 = __builtin_bit_cast(float, bits << 16 | (positive ? 0u : 0x80000000u));
  u64 mass_here = 0, m, c = 0, all = 0, over = 0;
  unsigned tokens_here = 0;
#pragma unroll
  for (int k = 0; k < EACH; k++) tokens_here += tokens[k];
  const int skip = x0 > top ? abs((int)bits - (int)(__builtin_bit_cast(unsigned, top) >> 16 & 0x7fff)) : 0;   // values above the largest: nobody's
  double first = 0.0, ratio = 0.0;   // of value `skip`; of a step of this exponent
  if (__any(tokens_here != 0)) {
    unsigned n;
    // (up to fifteen factors' errors add up in a weight: three terms, for 2^-44)
    first = a.w.template power<3>(a.w.steps(fminf(x0, top)), n);
    ratio = a.w.template power<3>(fmin(__builtin_bit_cast(double, (u64)(1023 - 134 + (bits >> 7)) << 52) * a.w.c, 60.0 * OCTAVE), n);
    double weight = first;
#pragma unroll
    for (int k = 0; k < EACH; k++) {
      const u64 wt = a.w.whole(weight), sum = wt * tokens[k];
      mass_here += sum, over += wt >= set.least ? sum : 0;
      weight *= k < skip ? 1.0 : ratio;
    }
  }
  // tokens next to 0 are behind the last positive value's
  const bool next_to_0 = small && v0 == VALUES / 2 - EACH;
  m = block_scan<bf16>(s, mass_here + (next_to_0 ? s.small[0] : 0), kept);
  if (set.cut_k) c = block_scan<bf16>(s, tokens_here + (next_to_0 ? s.small_tokens : 0), all);
  if (set.cut_m) {
    u64 heavy;
    block_scan<bf16>(s, over, heavy);
    over = max(set.one, heavy + s.small[1]);   // the first one at any rate
  }
  // ---- the cuts, then the token
  for (int step = set.cut_k ? 0 : set.cut_p ? 1 : 2; step < 3; step++) {
    if (step == 0 && all < (u64)set.top_k) continue;   // all that have a weight
    if (step == 1 && !set.cut_p) continue;
    if (step == 2 && set.cut_m) kept = min(kept, over);
    const u64 target = step == 0 ? (u64)set.top_k : step == 1 ? set.target_p(kept) : set.target_u(kept);
    const bool by_count = step == 0;
    __syncthreads();
    // found: the value's bits and the number of its token, the weights up to and with that one; or the tokens next to 0, with the sums before them
    const bool here = by_count ? c < target && c + tokens_here >= target : m < target && m + mass_here >= target;
    if (const u64 those = __ballot(here)) {   // one thread's: 16 lanes take a value of it each
      const int lane = tid & 63, from = __ffsll(those) - 1, k = lane & (EACH - 1), skipped = __builtin_amdgcn_readlane(skip, from);
      const unsigned its_bits = __builtin_amdgcn_readlane(bits, from), its_first = (tid - lane + from) * EACH, number = s.count[its_first + k];
      const double its_ratio = __builtin_bit_cast(double, read_lane(__builtin_bit_cast(u64, ratio), from));
      double weight = __builtin_bit_cast(double, read_lane(__builtin_bit_cast(u64, first), from));
#pragma unroll
      for (int j = 0; j < EACH - 1; j++) weight *= j < skipped || j >= k ? 1.0 : its_ratio;
      const u64 wt = a.w.whole(weight), mass = wt * number, upto = read_lane(m, from) + row_scan(mass), count = read_lane(c, from) + row_scan(number);
      if (lane < EACH && (by_count ? count - number < target && count >= target : upto - mass < target && upto >= target)) {
        unsigned nth = (unsigned)(target - (count - number));
        if (!by_count) {   // the least with nth wt >= what is missing
          const u64 missing = target - (upto - mass);
          nth = max(1u, (unsigned)((double)missing * __builtin_amdgcn_rcp((double)wt)));
          while (nth * wt < missing) nth++;
          while ((nth - 1) * wt >= missing) nth--;
        }
        s.found[0] = (u64)(its_first < VALUES / 2 ? its_bits - k : (its_bits + k) | 0x8000u) << 32 | nth, s.found[1] = upto - mass + nth * wt, s.words[1] = 0;
      }
    }
    if (next_to_0 && !here && (by_count ? c + tokens_here < target && c + tokens_here + s.small_tokens >= target : m + mass_here < target && m + mass_here + s.small[0] >= target)) {
      s.found[0] = c + tokens_here, s.found[1] = m + mass_here, s.words[1] = 1;
    }
    __syncthreads();
    u64 upto = s.found[1];
    const u64 found = s.found[0];
    if (s.words[1]) {
      if (!WHOLE) return false;
      const unsigned key = key_of(__builtin_bit_cast(float, (base - 1) << 16));
      a.resolve(of_key(~key), of_key(key), by_count, target, found, s.found[1], step == 2, entry, upto);
      listed = true;
    } else {
      x = __builtin_bit_cast(float, (unsigned)(found >> 32) << 16), nth = (unsigned)found;
      listed = false;
    }
    if (step < 2) kept = min(kept, upto);
  }
  return true;
}

// A whole row.
template <int NV>
__device__ __forceinline__ void sample_values_row(const SampleParams& p, int r, const Settings& set, Shared& s) {
  constexpr int EACH = VALUES_EACH;
  const int tid = threadIdx.x;
  Row<bf16, NV> row(static_cast<const bf16*>(p.logits) + r * p.row_stride, p.vocab);
  fill_table<bf16>(s);
  Sampler<bf16, NV> a{s, row, set.weights(0.f, s.table)};

  // ---- tokens by value, in a window that may have to be another one once the largest value is known
  unsigned tokens[EACH], base;   // of a thread's values
  float top = 0.f;
  int most = USUAL;
  for (bool again = false;; again = true) {
    base = base_of(most);
    for (int b = tid; b < VALUES / 4; b += THREADS_OF<bf16>) reinterpret_cast<u32x4*>(s.count)[b] = u32x4{0, 0, 0, 0};
    if (tid == 0) s.words[0] = ~0u, s.words[1] = 0, s.small[0] = s.small[1] = 0, s.small_tokens = 0;
    __syncthreads();
    unsigned least;
    int greatest;
    row.count_values(s.count, base, least, greatest);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) least = min(least, (unsigned)__shfl_xor((int)least, d, 64)), greatest = max(greatest, __shfl_xor(greatest, d, 64));
    if ((tid & 63) == 0) {
      atomicMin(&s.words[0], least);
      if (greatest >= 0) atomicMax(&s.words[1], (unsigned)greatest + 1);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EACH; k += 4) {
      const u32x4 four = *reinterpret_cast<const u32x4*>(&s.count[tid * EACH + k]);
#pragma unroll
      for (int e = 0; e < 4; e++) tokens[k + e] = four[e];
    }
    if (again) break;
    const unsigned positive = s.words[1];   // bits of the largest one, and 1
    top = __builtin_bit_cast(float, (positive - 1) << 16);
    const bool seen = positive > 0 && positive <= base + VALUES / 2;   // else all are negative, or it is beyond the window: infinite or NaN perhaps
    if (!seen) top = largest_of(row, s.wave_max);
    if (top == -INFINITY) {
      write_first(p, r, true, 0);
      return;
    }
    if (!(set.temperature > 0.f)) break;
    if (top == INFINITY) {
      sample_infinite(p, r, set, a, s);
      return;
    }
    // 36 T below the largest there is none that has a weight
    if (fabsf(top) + 36.f * set.temperature < (float)(1 << USUAL) && (seen || top < 0.f)) break;
    most = ilogb(fmin((double)fabsf(top) + 36.0 * (double)set.temperature, 0x1p127)) + 1;
    __syncthreads();
  }
  float x = top;        // the value of the token, and which one of those with it
  unsigned nth = 1;
  bool listed = false;   // the token is in `entry`
  u64 entry = 0, kept = 0;
  if (set.temperature > 0.f) {
    a.w.top = top, a.w.topf = top;
    const bool small = s.words[0] < base;
    if (small) {   // nearer to 0 than the window
      add_small(set, s, a, row, base);
      __syncthreads();
    }
    choose_value<true>(set, s, a, base, top, tokens, small, x, nth, listed, entry, kept);
  }
  if (!listed) entry = a.pick(x, nth);
  if (set.temperature > 0.f) write(p, r, a.w, entry, kept);
  else write_first(p, r, false, entry);
}

template <int NV>
__global__ __launch_bounds__(THREADS_OF<bf16>) void sample_values_kernel(const SampleParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  sample_values_row<NV>(p, blockIdx.x, Settings(p, blockIdx.x), *reinterpret_cast<Shared*>(smem));
}

// ---- fp32
// A whole row.
template <typename T>
__device__ __forceinline__ void sample_row(const SampleParams& p, int r, const Settings& set, Shared& s) {
  const int tid = threadIdx.x;
  Row<T> row(static_cast<const T*>(p.logits) + r * p.row_stride, p.vocab);
  fill_table<T>(s);
  for (int b = tid; b < BUCKETS; b += THREADS_OF<T>) s.mass[b] = 0, s.count[b] = 0;
  const float largest = largest_of(row, s.wave_max);
  Sampler<T> a{s, row, set.weights(largest, s.table)};
  if (largest == -INFINITY || !(set.temperature > 0.f)) {   // nothing to choose from, or nothing but the first
    write_first(p, r, largest == -INFINITY, largest == -INFINITY ? 0 : a.pick(largest, 1));
    return;
  }
  if (largest == INFINITY) {
    sample_infinite(p, r, set, a, s);
    return;
  }
  u64 entry = 0, kept = 0;
  // ---- few: all that may be among the first top_k into the list
  bool done = false;
  if (set.few()) {
    a.count_buckets();
    __syncthreads();
    const int n = a.gather_first(set.top_k);
    done = n <= LIST;
    if (done) {
      entry = a.among_first(n, set, kept);
    } else {
      __syncthreads();
      for (int b = tid; b < BUCKETS; b += THREADS_OF<T>) s.count[b] = 0;
      __syncthreads();
    }
  }
  // ---- sums of the weights by buckets of all
  if (!done) {
    u64 over = a.add_weights(set.cut_m, set.least);
    if (set.cut_k) {
      unsigned last = 0;
      row.all([&](float x, int, int) {
        unsigned b;
        const u64 wt = a.w.of(x, b);
        if (b == BUCKETS - 1) last += wt != 0;
        else atomicAdd(&s.count[b], 1u);
      });
      if (last) atomicAdd(&s.count[BUCKETS - 1], last);
    }
    __syncthreads();
    constexpr int EACH = BUCKETS / THREADS_OF<T>;
    unsigned tokens[EACH];
    u64 weights[EACH], mass_here = 0, tokens_here = 0, m, c = 0, all = 0, heavy;
#pragma unroll
    for (int k = 0; k < EACH; k++) {
      weights[k] = s.mass[tid * EACH + k], tokens[k] = s.count[tid * EACH + k];
      mass_here += weights[k], tokens_here += tokens[k];
    }
    m = block_scan<T>(s, mass_here, kept);
    if (set.cut_k) c = block_scan<T>(s, tokens_here, all);
    if (set.cut_m) {
      block_scan<T>(s, over, heavy);
      over = max(set.one, heavy);   // the first one at any rate
    }
    if (!set.cut_k) {
      Ends q;
      const u64 most = set.cut_m ? over : ~0ull;
      const int n = a.gather_ends(set, m, weights, kept, most, q);
      done = n <= LIST;
      if (done) entry = a.among_ends(n, set, most, q, kept);
    }
    for (int step = done ? 3 : set.cut_k ? 0 : set.cut_p ? 1 : 2; step < 3; step++) {
      if (step == 0 && all < (u64)set.top_k) continue;   // all that have a weight
      if (step == 1 && !set.cut_p) continue;
      if (step == 2 && set.cut_m) kept = min(kept, over);
      const u64 target = step == 0 ? (u64)set.top_k : step == 1 ? set.target_p(kept) : set.target_u(kept);
      u64 count = 0, mass = 0, upto;
      const unsigned b = a.template slot_of<EACH>(step == 0, target, tid * EACH, c, m, tokens, weights, count, mass);
      float lo, hi;
      a.range_of(b, lo, hi);
      a.resolve(lo, hi, step == 0, target, count, mass, step == 2, entry, upto);
      if (step < 2) kept = min(kept, upto);
    }
  }
  write(p, r, a.w, entry, kept);
}

template <typename T>
__global__ __launch_bounds__(THREADS_OF<T>) void sample_kernel(const SampleParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  sample_row<T>(p, blockIdx.x, Settings(p, blockIdx.x), *reinterpret_cast<Shared*>(smem));
}

// ---- few long rows: a row in slices, a block each, in launches between which all slices' results are there
template <typename T> __device__ __forceinline__ Row<T> slice_of(const SampleParams& p, int r, int j) {
  return Row<T>(static_cast<const T*>(p.logits) + r * p.row_stride + j * p.slice, min(p.slice, p.vocab - j * p.slice));
}
__device__ __forceinline__ float largest_slice(const SampleParams& p, int r) {
  const int lane = threadIdx.x & 63;
  float x = lane < p.slices ? p.largest[r * p.slices + lane] : -INFINITY;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) x = fmaxf(x, __shfl_xor(x, d, 64));
  return x;
}
// Sums over a row's slices of N vectors of a thread, SIDE slices' loads at once.
template <int N, typename V> __device__ __forceinline__ void add_slices(V (&sum)[N], const V* from, int pitch, int slices) {
  constexpr int SIDE = 4;
  for (int k = 0; k < slices; k += SIDE) {
    V x[SIDE][N];
#pragma unroll
    for (int q = 0; q < SIDE; q++)
#pragma unroll
      for (int e = 0; e < N; e++) x[q][e] = from[(int64_t)min(k + q, slices - 1) * pitch + e];
#pragma unroll
    for (int q = 0; q < SIDE; q++)
#pragma unroll
      for (int e = 0; e < N; e++) sum[e] += k + q < slices ? x[q][e] : V{};
  }
}
// bf16: the slices' tokens by value,
__global__ __launch_bounds__(THREADS_OF<bf16>) void sample_counts_kernel(const SampleParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  const int r = blockIdx.x / p.slices, j = blockIdx.x - r * p.slices, tid = threadIdx.x;
  Row<bf16> row = slice_of<bf16>(p, r, j);
  for (int b = tid; b < VALUES / 4; b += THREADS_OF<bf16>) reinterpret_cast<u32x4*>(s.count)[b] = u32x4{0, 0, 0, 0};
  if (tid == 0) s.words[0] = ~0u, s.words[1] = 0;
  __syncthreads();
  unsigned least;
  int greatest;
  row.count_values(s.count, base_of(USUAL), least, greatest);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) least = min(least, (unsigned)__shfl_xor((int)least, d, 64)), greatest = max(greatest, __shfl_xor(greatest, d, 64));
  if ((tid & 63) == 0) {
    atomicMin(&s.words[0], least);
    if (greatest >= 0) atomicMax(&s.words[1], (unsigned)greatest + 1);
  }
  __syncthreads();
  for (int b = tid; b < VALUES / 4; b += THREADS_OF<bf16>) reinterpret_cast<u32x4*>(p.counts + (int64_t)blockIdx.x * VALUES)[b] = reinterpret_cast<u32x4*>(s.count)[b];
  if (tid == 0) p.ends[blockIdx.x] = make_int2((int)s.words[0], (int)s.words[1]);
}
// and the token: every block finds its value and the slice that has it, which looks for it.  Rows for which that will not do -- the largest is not a positive one below 128, or the token is
// one next to 0 -- one block, all of it.
__global__ __launch_bounds__(THREADS_OF<bf16>) void sample_counted_kernel(const SampleParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  const int r = blockIdx.x / p.slices, j = blockIdx.x - r * p.slices, tid = threadIdx.x;
  const Settings set(p, r);
  const unsigned base = base_of(USUAL), *counts = p.counts + (int64_t)r * p.slices * VALUES;
  const int lane = tid & 63;
  const int2 ends = p.ends[r * p.slices + min(lane, p.slices - 1)];
  u32x4 fours[VALUES_EACH / 4] = {};
  add_slices(fours, reinterpret_cast<const u32x4*>(counts + tid * VALUES_EACH), VALUES / 4, p.slices);
  unsigned least = (unsigned)ends.x, positive = (unsigned)ends.y, tokens[VALUES_EACH];
#pragma unroll
  for (int d = 1; d < 64; d *= 2) least = min(least, (unsigned)__shfl_xor((int)least, d, 64)), positive = max(positive, (unsigned)__shfl_xor((int)positive, d, 64));
#pragma unroll
  for (int k = 0; k < VALUES_EACH; k++) tokens[k] = fours[k / 4][k % 4];
  const float top = __builtin_bit_cast(float, (positive - 1) << 16);   // as in a whole row
  const bool seen = positive > base && positive <= base + VALUES / 2, greedy = !(set.temperature > 0.f);
  bool whole = !seen || (!greedy && !(top + 36.f * set.temperature < (float)(1 << USUAL)));
  if (whole && j != 0) return;
  Row<bf16> row = slice_of<bf16>(p, r, j);
  Sampler<bf16> a{s, row, set.weights(top, s.table)};
  float x = top;
  unsigned nth = 1;
  u64 entry = 0, kept = 0;
  if (!greedy && !whole) {
    bool listed;
    fill_table<bf16>(s);
#pragma unroll
    for (int q = 0; q < VALUES_EACH / 4; q++) reinterpret_cast<u32x4*>(s.count)[tid * (VALUES_EACH / 4) + q] = fours[q];
    if (tid == 0) s.small[0] = s.small[1] = 0, s.small_tokens = 0;
    __syncthreads();
    for (int k = 0; least < base && k < p.slices; k++)
      if ((unsigned)p.ends[r * p.slices + k].x < base) add_small(set, s, a, slice_of<bf16>(p, r, k), base);
    __syncthreads();
    whole = !choose_value<false>(set, s, a, base, top, tokens, least < base, x, nth, listed, entry, kept);
  }
  if (whole) {
    __syncthreads();
    if (j == 0) sample_values_row<0>(p, r, set, s);
    return;
  }
  // the slices' numbers of it, in 16 lanes
  const unsigned bits = __builtin_bit_cast(unsigned, x) >> 16, d = (bits & 0x7fff) - base, place = bits & 0x8000 ? VALUES / 2 + d : VALUES / 2 - 1 - d;
  const unsigned mine = lane < p.slices ? counts[lane * VALUES + place] : 0, upto = (unsigned)row_scan(mine);
  const int of = __ffsll(__ballot(lane < p.slices && upto >= nth)) - 1;
  if (of != j) return;
  nth -= __builtin_amdgcn_readlane(upto - mine, of);
  entry = a.pick(x, nth) + (unsigned)(j * p.slice);
  if (greedy) write_first(p, r, false, entry);
  else write(p, r, a.w, entry, kept);
}
// fp32: the slices' largest,
__global__ __launch_bounds__(THREADS_OF<float>) void sample_largest_kernel(const SampleParams p) {
  __shared__ float wave_max[THREADS_OF<float> / 64];
  const int r = blockIdx.x / p.slices, j = blockIdx.x - r * p.slices;
  const Row<float> row = slice_of<float>(p, r, j);
  const float x = largest_of(row, wave_max);
  if (threadIdx.x == 0) p.largest[blockIdx.x] = x;
  if (threadIdx.x == 0 && j == 0) p.listed[r] = 0;
}
// their sums by buckets,
__device__ __forceinline__ bool in_slices(const Settings& set, float largest) {
  return set.temperature > 0.f && fabsf(largest) < INFINITY && (set.few() || !set.cut_k);
}
__global__ __launch_bounds__(THREADS_OF<float>) void sample_buckets_kernel(const SampleParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  const int r = blockIdx.x / p.slices, j = blockIdx.x - r * p.slices, tid = threadIdx.x;
  const Settings set(p, r);
  const float largest = largest_slice(p, r);
  if (!in_slices(set, largest)) return;
  const bool few = set.few();
  Row<float> row = slice_of<float>(p, r, j);
  Sampler<float> a{s, row, set.weights(largest, s.table)};
  if (!few) fill_table<float>(s);
  for (int b = tid; b < BUCKETS; b += THREADS_OF<float>) s.mass[b] = 0, s.count[b] = 0;
  __syncthreads();
  if (few) {
    a.count_buckets();
    __syncthreads();
    for (int b = tid; b < BUCKETS / 4; b += THREADS_OF<float>) reinterpret_cast<u32x4*>(p.mass + (int64_t)blockIdx.x * BUCKETS)[b] = reinterpret_cast<u32x4*>(s.count)[b];
  } else {
    u64 over = a.add_weights(set.cut_m, set.least), heavy;
    block_scan<float>(s, over, heavy);
    if (tid == 0) p.over[blockIdx.x] = heavy;
    for (int b = tid; b < BUCKETS / 2; b += THREADS_OF<float>) reinterpret_cast<u32x4*>(p.mass + (int64_t)blockIdx.x * BUCKETS)[b] = reinterpret_cast<u32x4*>(s.mass)[b];
  }
}
// what each has in the buckets that matter, which every block finds for itself,
__global__ __launch_bounds__(THREADS_OF<float>) void sample_slices_kernel(const SampleParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  const int r = blockIdx.x / p.slices, j = blockIdx.x - r * p.slices, tid = threadIdx.x;
  const Settings set(p, r);
  const float largest = largest_slice(p, r);
  Row<float> row = slice_of<float>(p, r, j);
  Sampler<float> a{s, row, set.weights(largest, s.table)};
  if (largest == -INFINITY || !(set.temperature > 0.f)) {   // nothing, or the first: in the first slice that has it
    int first = 0;
    while (p.largest[r * p.slices + first] != largest) first++;
    if (j == first) write_first(p, r, largest == -INFINITY, largest == -INFINITY ? 0 : a.pick(largest, 1) + (unsigned)(j * p.slice));
    return;
  }
  if (!in_slices(set, largest)) return;
  RowEnds e{};
  e.most = ~0ull;
  const u64* mass = p.mass + (int64_t)r * p.slices * BUCKETS;
  int n;
  if (set.few()) {
    typedef unsigned part __attribute__((ext_vector_type(BUCKETS / THREADS_OF<float>)));
    part sum[1] = {};
    add_slices(sum, reinterpret_cast<const part*>(mass) + tid, BUCKETS * (int)(sizeof(u64) / sizeof(part)), p.slices);
    reinterpret_cast<part*>(s.count)[tid] = sum[0];
    __syncthreads();
    n = a.gather_first(set.top_k);
  } else {
    constexpr int EACH = BUCKETS / THREADS_OF<float>;
    u64 weights[EACH] = {}, here = 0;
    add_slices(weights, mass + tid * EACH, BUCKETS, p.slices);
#pragma unroll
    for (int i = 0; i < EACH; i++) s.mass[tid * EACH + i] = weights[i], here += weights[i];
    const u64 m = block_scan<float>(s, here, e.kept);
    if (set.cut_m) {
      block_scan<float>(s, tid < p.slices ? p.over[r * p.slices + tid] : 0, e.most);
      e.most = max(set.one, e.most);   // the first one at any rate
    }
    n = a.gather_ends(set, m, weights, e.kept, e.most, e.q);
  }
  if (tid == 0) s.words[2] = atomicAdd(&p.listed[r], (unsigned)n);
  if (tid == 0 && j == 0) p.ends_of_rows[r] = e;
  __syncthreads();
  const unsigned to = s.words[2];
  if (n <= LIST && to + n <= LIST)
    for (int k = tid; k < n; k += THREADS_OF<float>) p.lists[(int64_t)r * LIST + to + k] = s.list[k] + (unsigned)(j * p.slice);
}
// and the token among them.  A row for which that will not do: all of it.
__global__ __launch_bounds__(THREADS_OF<float>) void sample_listed_kernel(const SampleParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  const int r = blockIdx.x, tid = threadIdx.x;
  const Settings set(p, r);
  const float largest = largest_slice(p, r);
  if (largest == -INFINITY || !(set.temperature > 0.f)) return;
  const unsigned n = p.listed[r];
  if (!in_slices(set, largest) || n > LIST) {
    sample_row<float>(p, r, set, s);
    return;
  }
  Row<float> row(static_cast<const float*>(p.logits) + r * p.row_stride, p.vocab);
  Sampler<float> a{s, row, set.weights(largest, s.table)};
  for (int k = tid; k < (int)n; k += THREADS_OF<float>) s.list[k] = p.lists[(int64_t)r * LIST + k];
  const RowEnds e = p.ends_of_rows[r];
  fill_table<float>(s);
  __syncthreads();
  u64 kept = e.kept;
  const u64 entry = set.few() ? a.among_first((int)n, set, kept) : a.among_ends((int)n, set, e.most, e.q, kept);
  write(p, r, a.w, entry, kept);
}

template <typename T, typename K> int launch(K kernel, const SampleParams& p, int blocks, hipStream_t st) {
  if (int rc = ody_allow_dynamic_lds(reinterpret_cast<const void*>(kernel), sizeof(Shared), "ody_sample")) return rc;
  ODY_LAUNCH("sample", st, kernel, dim3((unsigned)blocks), dim3(THREADS_OF<T>), sizeof(Shared), p);
  return ody_check_launch("sample");
}

// fp32 rows of fewer logits go by 512 threads, whose barriers and joined results cost less (us by 512 / 1024: 64 rows of 4000 10.6 / 12.0, of 12000 14.7 / 14.9, of 24000 19.8 / 19.1).
constexpr int SHORT = 12288;
// How rows are divided: long ones into slices, at most one a compute unit; of bf16 fewer, as each block reads the counts of all.  us by a block a row / in slices, top_p 0.9: fp32,
// one row of 66000 31.8 / 24.3, of 80000 34.6 / 23.7, of 250000 87.5 / 28.0; 16 of 66000 32.0 / 32.2, of 80000 35.8 / 32.3, of 128000 52.6 / 32.8; 64 of 80000 37.2 / 32.5, of 128000 54.6 / 40.6, 128 61.6 / 59.8;
// bf16, one of 70000 19.8 / 16.9, of 250000 42.9 / 19.5; 8 of 128000 30.0 / 19.9, 64 34.3 / 26.4, 128 35.4 / 28.9.
// fp32 rows of a small top_k and greedy ones are read twice and little else: in slices from FEW on (one of 66000 with top_k 20 18.5 / 19.5, of 98000 22.9 / 19.6, of 250000 47.3 / 21.1; 16 of 66000 19.1 / 24.4,
// of 98000 23.4 / 24.5; greedy, one of 70000 10.3 / 12.1), if one number for all says so; where each has its own they may all be such, and many rows lose more so than others gain (4 of 66000, top_k 0 and 20 in
// turn 28.7 / 23.7, all 20 18.8 / 20.6; 16 28.9 / 27.7 and 19.0 / 24.4; 64 29.0 / 29.6 and 19.0 / 23.6).  A large top_k for all is nothing for slices (in_slices): one row of 70000 with top_k 4000 57.3 / 65.8.
constexpr int LONG = 65536, FEW = 98304;
int least_of(int rows, int vocab, bool greedy, bool each, int top_k) {   // the least of fp32 rows that go in slices
  if (greedy || (each && rows >= 16)) return FEW;
  if (each || top_k <= 0 || top_k >= vocab) return LONG;
  return top_k <= LIST / 2 ? FEW : vocab + 1;
}
struct Plan {
  int slices, slice;
  size_t ends, mass, over, largest, listed, bytes;   // places in the workspace, behind the lists (fp32) or the counts (bf16)
};
Plan plan(int rows, int vocab, int dtype, int least) {
  Plan q{};
  q.slices = std::min(dtype == ODY_F32 ? 16 : rows > 8 ? 4 : 8, 256 / rows);
  if (vocab < least || q.slices < (dtype == ODY_F32 ? 4 : 2)) return Plan{1, vocab, 0, 0, 0, 0, 0, 0};
  q.slice = ((vocab + q.slices - 1) / q.slices + 7) / 8 * 8;
  q.slices = (vocab + q.slice - 1) / q.slice;
  const size_t all = (size_t)rows * q.slices;
  if (dtype == ODY_BF16) {
    q.ends = all * VALUES * sizeof(unsigned), q.bytes = q.ends + all * sizeof(int2);
    return q;
  }
  q.mass = (size_t)rows * LIST * sizeof(u64), q.ends = q.mass + all * BUCKETS * sizeof(u64), q.over = q.ends + rows * sizeof(RowEnds);
  q.largest = q.over + all * sizeof(u64), q.listed = q.largest + all * sizeof(float), q.bytes = q.listed + rows * sizeof(unsigned);
  return q;
}

}  // namespace

extern "C" size_t ody_sample_workspace_bytes(int rows, int vocab, int dtype) { return rows > 0 && vocab > 0 ? plan(rows, vocab, dtype, LONG).bytes : 0; }

extern "C" int ody_sample(const void* logits, const float* u, const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                          float temperature_all, int top_k_all, float top_p_all, float min_p_all, int64_t* tokens, float* logprobs, int rows, int vocab,
                          int64_t row_stride, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  ODY_REQUIRE(logits && u && tokens && logprobs, ODY_ERR_NULL, "ody_sample: logits, u, tokens or logprobs is NULL");
  ODY_REQUIRE(rows > 0 && vocab > 0 && rows < 1 << 22 && vocab <= MOST, ODY_ERR_BAD_SHAPE, "ody_sample: %d rows of %d logits (fewer than 2^22 of at most %d)", rows, vocab, MOST);
  ODY_REQUIRE(row_stride >= vocab || rows == 1, ODY_ERR_BAD_SHAPE, "ody_sample: rows overlap (stride %lld)", (long long)row_stride);
  ODY_REQUIRE(dtype == ODY_BF16 || dtype == ODY_F32, ODY_ERR_UNSUPPORTED, "ody_sample: dtype %d unknown", dtype);
  ODY_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (dtype == ODY_BF16 ? 1 : 3)) == 0, ODY_ERR_MISALIGNED, "ody_sample: logits are not aligned to their size");
  const Plan q = plan(rows, vocab, dtype, dtype == ODY_F32 ? least_of(rows, vocab, !temperature && !(temperature_all > 0.f), top_k != nullptr, top_k_all) : LONG);
  ODY_REQUIRE(q.bytes == 0 || (workspace && workspace_bytes >= q.bytes && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0), ODY_ERR_WORKSPACE,
              "ody_sample: a workspace of %zu bytes, 256-byte aligned, is needed, %zu given", q.bytes, workspace_bytes);
  const int frac = std::min(50, __builtin_clzll((u64)vocab + 1));   // (vocab + 1) 2^frac is below 2^64
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  const SampleParams p{logits, row_stride, u, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all, top_k_all, tokens, logprobs, vocab,
                       frac, q.slices, q.slice, reinterpret_cast<u64*>(ws + q.mass), reinterpret_cast<u64*>(ws + q.over), reinterpret_cast<unsigned*>(ws), reinterpret_cast<int2*>(ws + q.ends),
                       reinterpret_cast<float*>(ws + q.largest), reinterpret_cast<unsigned*>(ws + q.listed), reinterpret_cast<RowEnds*>(ws + q.ends), reinterpret_cast<u64*>(ws)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == ODY_F32 && q.slices == 1) return vocab < SHORT ? launch<ShortRow>(&sample_kernel<ShortRow>, p, rows, st) : launch<float>(&sample_kernel<float>, p, rows, st);
  if (dtype == ODY_F32) {
    ODY_LAUNCH("sample_largest", st, sample_largest_kernel, dim3((unsigned)(rows * q.slices)), dim3(THREADS_OF<float>), 0, p);
    if (int rc = ody_check_launch("sample_largest")) return rc;
    if (int rc = launch<float>(&sample_buckets_kernel, p, rows * q.slices, st)) return rc;
    if (int rc = launch<float>(&sample_slices_kernel, p, rows * q.slices, st)) return rc;
    return launch<float>(&sample_listed_kernel, p, rows, st);
  }
  if (q.slices > 1) {
    if (int rc = launch<bf16>(&sample_counts_kernel, p, rows * q.slices, st)) return rc;
    return launch<bf16>(&sample_counted_kernel, p, rows * q.slices, st);
  }
  const int turns = (vocab + 14 + THREADS_OF<bf16> * 8 - 1) / (THREADS_OF<bf16> * 8);   // however rows are aligned
  if (turns <= 8) return launch<bf16>(&sample_values_kernel<8>, p, rows, st);   // longer rows are counted while they arrive (256 of 128000: 45 us, 51 out of registers)
  return launch<bf16>(&sample_values_kernel<0>, p, rows, st);
}
