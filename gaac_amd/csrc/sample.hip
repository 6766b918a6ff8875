// One token per row of logits: temperature, top-k, top-p, min-p, and a given random number u in [0, 1).
//   w_i = exp((x_i - max) / T).  Order: x descending, then index ascending.  Kept: the first k in the order; of these the shortest prefix whose sum of w is at
//   least p times theirs; of these the ones with w >= min_p (the maximum has 1).  Token: the first i, by index, at which the running sum of the kept w
//   exceeds u times their total.  T not positive: the first maximum.  Nothing but -inf (a NaN counts as one): -1.
//
// Which token comes is a whole number, so it must not depend on the order in which a sum is taken: weights are computed in 64 bits and held as multiples of 2^-43 of the
// largest in 64-bit integers (2^20 of them fit).  Their sums are exact; against the definition a weight is off by 2^-44 (and 0 below that), a sum over n tokens by n * 2^-44 at
// most, 2^-24 for 2^20 of them, which is u's own last bit.  A share (p or u times a sum) is rounded to 53 bits, 2^-53 of it.
// What is kept is a prefix of the order, so it is found as a key (the bits of x, in order) and the number of its equals that are kept: counts and sums by bins
// of (max - x), then the elements of the bin where the limit falls (with a k: all up to it), in order: up to 64 of them sorted by a wave, up to 1024 by the block, up to 8192
// by ever finer bins of their keys, more by such bins over the row.  Three launches: the row's maximum; bins; and the limits, the sums of segments and the token by the last of the row's blocks to
// arrive.  A row of one segment takes one launch, bins and candidates in LDS.
//
// What bounds it: for few rows the chain of launches and of dependent steps in the last block (4 rows of 128256 in bf16, 1 MB, top-k 50: 16.6 us; kernels 3.0, 4.9 and 9.7,
// launch 1.6 of each); for many the weights in 64 bits, computed twice for each element that can be kept, and atomic additions to bins (64
// mixed rows of 128256 in fp32, 33 MB: 52.3 us; kernels 7.0, 17.2 and 28.2; the read alone 5.5).
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "gaac_capi.h"
#include "../../include/gaac_hip.h"

namespace {

constexpr int NT = 512, SEG = NT * 8, BINS = 2048, MAX_V = 1 << 20, MAX_SEGS = MAX_V / SEG;      // a segment is a block's: 8 elements a thread
constexpr int BLOCKS = 512;
constexpr int ROOM = 8192;      // elements of a row that are looked at one by one, at most
constexpr int SORTED = 2 * NT;      // and of these so many by sorting them
static_assert(MAX_SEGS <= NT && 2 * SORTED <= BINS);
typedef unsigned long long u64;
template <int N> struct Number { static constexpr int value = N; };
typedef unsigned u4 __attribute__((ext_vector_type(4)));

// Order of floats as that of unsigned numbers; -0 and NaN have been taken away.
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __builtin_bit_cast(unsigned, x);
  return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) { return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k); }

template <typename T> __device__ __forceinline__ float number(T v) {
  const float x = (float)v;
  return x != x ? -__builtin_inff() : x + 0.f;      // -0 + 0 = +0: equal numbers have equal keys
}

// The row as segments from the 16-byte boundary at or below its start; a thread has 8 elements in a row.  Elements before and behind the row are -inf.
template <typename T> struct Row {
  const T* base;      // aligned
  int shift, V;       // row element i is base[shift + i]
  __device__ __forceinline__ Row(const T* start, int V_) : shift((int)(reinterpret_cast<uintptr_t>(start) % 16 / sizeof(T))), V(V_) { base = start - shift; }
  __device__ __forceinline__ int segs() const { return (shift + V + SEG - 1) / SEG; }
  __device__ __forceinline__ int index(int seg, int i) const { return seg * SEG + threadIdx.x * 8 + i; }      // of element i of the thread, counted from base
  struct Raw { T v[8]; };      // as they lie in memory: what is fetched ahead is not looked at
  __device__ __forceinline__ Raw fetch(int seg) const {
    constexpr int G = 16 / sizeof(T);      // elements of a 16-byte load
    Raw r;
#pragma unroll
    for (int part = 0; part < 8 / G; ++part) {
      const int at = index(seg, part * G);
      if (at >= shift && at + G <= shift + V) {
        const u4 raw = *reinterpret_cast<const u4*>(base + at);
        __builtin_memcpy(r.v + part * G, &raw, 16);
      } else {
#pragma unroll
        for (int i = 0; i < G; ++i) r.v[part * G + i] = at + i >= shift && at + i < shift + V ? base[at + i] : (T)-__builtin_inff();
      }
    }
    return r;
  }
  static __device__ __forceinline__ void numbers(const Raw& r, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = number(r.v[i]);
  }
  __device__ __forceinline__ void load(int seg, float (&x)[8]) const { numbers(fetch(seg), x); }
  // f(seg, x) for every step-th segment of n from `first` on, the next one in flight meanwhile; r: the first
  template <typename F> __device__ __forceinline__ void each_segment(int n, int first, int step, Raw r, F f) const {
    for (int seg = first; seg < n; seg += step) {
      float x[8];
      numbers(r, x);
      if (seg + step < n) r = fetch(seg + step);
      f(seg, x);
    }
  }
};

// exp(y), y <= 0, from z = y * 256 / ln 2: the whole part n of z by a table of the 256 roots of 2 in LDS and the exponent, times the series of exp to r^4 of the rest,
// r = (z - n) ln 2 / 256 (|r| <= 0.0014: what is left is below 1e-16).  z's own rounding is one of 2^-53 of y, and below -31 all is less than half of 2^-43.
// (64 roots, a series to r^5 and r in two steps: 64 mixed rows of 128256 56.3 us, so 52.3; the series to r^11 without a table some 7 more.)
constexpr int ROOTS = 256;
constexpr double LN2 = 0.6931471805599453, STEP = LN2 / ROOTS;
__device__ __forceinline__ void fill_roots(double* table) {      // 2^(j / 256) = exp(j ln 2 / 256) by its series
  if (threadIdx.x < ROOTS) {
    const double x = threadIdx.x * STEP;
    double e = 1;
#pragma unroll
    for (int k = 17; k > 0; --k) e = __builtin_fma(e, x * (1.0 / k), 1.0);
    table[threadIdx.x] = e;
  }
}
__device__ __forceinline__ double exp_of(double z, const double* table) {
  z = __builtin_fmax(z, -31.0 / STEP);      // (also where it is NaN)
  const double n = __builtin_rint(z), f = z - n;
  const int i = (int)n;
  double q = __builtin_fma(f, STEP * STEP * STEP * STEP / 24, STEP * STEP * STEP / 6);
  q = __builtin_fma(q, f, STEP * STEP / 2);
  q = __builtin_fma(q, f, STEP);
  const double t = table[i & (ROOTS - 1)], e = __builtin_fma(t * q, f, t);
  const u64 bits = __builtin_bit_cast(u64, e);
  return __builtin_bit_cast(double, (u64)((unsigned)(bits >> 32) + ((unsigned)(i & -ROOTS) << 12)) << 32 | (unsigned)bits);      // + i / 256 in the exponent
}
// As a multiple of 2^-43: the sum with 2^9, whose last bit that is, rounds to it.
__device__ __forceinline__ u64 fixed(double w) { return __builtin_bit_cast(u64, w + 512.0) - __builtin_bit_cast(u64, 512.0); }

struct Weights {      // of a row
  float top;
  double scale;      // 1 / (T STEP)
  const double* roots;
  __device__ __forceinline__ Weights(float top_, float t, const double* r) : top(top_), scale(1.0 / (double)t * (1.0 / STEP)), roots(r) {}
  __device__ __forceinline__ double operator()(float x) const { return x == top ? 1.0 : exp_of(((double)x - (double)top) * scale, roots); }      // (-inf: less than half of 2^-43)
};

// Inclusive sums over the wave in the vector unit: shifts within rows of 16 lanes, then the last lane of a row to the next ones.
template <int CTRL, int ROWS> __device__ __forceinline__ unsigned moved(unsigned x) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS> __device__ __forceinline__ u64 moved(u64 x) { return (u64)moved<CTRL, ROWS>((unsigned)(x >> 32)) << 32 | moved<CTRL, ROWS>((unsigned)x); }
template <typename U> __device__ __forceinline__ U wave_scan(U x) {
  x += moved<0x111, 0xf>(x); x += moved<0x112, 0xf>(x); x += moved<0x114, 0xf>(x); x += moved<0x118, 0xf>(x);
  x += moved<0x142, 0xa>(x); x += moved<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ u64 lane(u64 x, int i) { return (u64)(unsigned)__builtin_amdgcn_readlane((int)(x >> 32), i) << 32 | (unsigned)__builtin_amdgcn_readlane((int)x, i); }
__device__ __forceinline__ u64 larger(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 wave_max(u64 x) {      // in lane 63
  x = larger(x, moved<0x111, 0xf>(x)); x = larger(x, moved<0x112, 0xf>(x)); x = larger(x, moved<0x114, 0xf>(x)); x = larger(x, moved<0x118, 0xf>(x));
  x = larger(x, moved<0x142, 0xa>(x)); return larger(x, moved<0x143, 0xc>(x));
}

constexpr int WAVES = NT / 64;
struct Shared {
  u64 mass[BINS];           // of bins; candidates in order
  unsigned count[BINS];
  double roots[ROOTS];
  u64 seg_mass[MAX_SEGS];
  unsigned seg_ties[MAX_SEGS];
  u64 wave_mass[WAVES];
  unsigned wave_count[WAVES];
  u64 before_mass;
  unsigned before_count, found_count;
  int found, last;
};

// Inclusive prefix sums over the block of each thread's (count, mass); returns those of all.
struct Sums { unsigned count; u64 mass; };
__device__ __forceinline__ Sums block_scan(Shared& sh, unsigned& count, u64& mass) {
  const int w = threadIdx.x >> 6;
  mass = wave_scan(mass);
  count = wave_scan(count);
  if ((threadIdx.x & 63) == 63) { sh.wave_mass[w] = mass; sh.wave_count[w] = count; }
  __syncthreads();
  Sums all{0, 0}, x[WAVES];
#pragma unroll
  for (int i = 0; i < WAVES; ++i) x[i] = {sh.wave_count[i], sh.wave_mass[i]};      // (all reads in flight together)
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    if (i == w) { count += all.count; mass += all.mass; }
    all.count += x[i].count; all.mass += x[i].mass;
  }
  __syncthreads();
  return all;
}

struct Limit { unsigned key, ties; };      // the key of the last element kept, and how many of its equals are kept; key 0: all

struct Bins {      // of max - x, 1/32 of the temperature (or of 1, if that is less) wide, 64 of it in all; never ascends with x
  float top, scale;
  __device__ __forceinline__ Bins(float top_, float t) : top(top_), scale(fmaxf(32.f / t, 32.f)) {}
  __device__ __forceinline__ int operator()(float x) const { return x == top ? 0 : (int)fminf((top - x) * scale, (float)(BINS - 1)); }
};

// Zero the bins / find the first of them at which the running count or sum reaches what is wanted: into sh.found (-1: none), before_count, before_mass.
__device__ __forceinline__ void clear_bins(Shared& sh) {
  for (int i = threadIdx.x; i < BINS; i += NT) { sh.mass[i] = 0; sh.count[i] = 0; }
  __syncthreads();
}
constexpr int PER = BINS / NT;      // bins of a thread
template <bool BY_MASS> __device__ unsigned find_bin(Shared& sh, const unsigned (&counts)[PER], const u64 (&masses)[PER], unsigned before_count, u64 before_mass, unsigned want_count, u64 want_mass) {
  unsigned count = 0;
  u64 mass = 0;
  for (int i = 0; i < PER; ++i) { count += counts[i]; mass += masses[i]; }
  const unsigned own_count = count;
  const u64 own_mass = mass;
  if (threadIdx.x == 0) sh.found = -1;
  const unsigned all = block_scan(sh, count, mass).count;
  count += before_count - own_count; mass += before_mass - own_mass;      // before this thread's bins
  for (int i = 0; i < PER; ++i) {
    const unsigned c = count + counts[i];
    const u64 m = mass + masses[i];
    if (BY_MASS ? mass < want_mass && m >= want_mass : count < want_count && c >= want_count) {
      sh.found = threadIdx.x * PER + i; sh.before_count = count; sh.before_mass = mass; sh.found_count = counts[i];
    }
    count = c; mass = m;
  }
  __syncthreads();
  return all;
}

// The first element in the order at which the running count reaches want_count (BY_MASS false) or the running sum of weights reaches want_mass (true), among
// the elements with key above `from.key` and from.ties of its equals.  each(f) calls f(x) for the thread's share of the elements.
// bin0: the bin of max - x where it falls, if that is known.
template <bool BY_MASS, typename Each>
__device__ Limit find_limit(Shared& sh, Each each, const Weights& weight, const Bins& bin_of, Limit from, unsigned want_count, u64 want_mass, int bin0 = -1) {
  unsigned lo = 0, hi = 0xffffffffu, before_count = 0;
  u64 before_mass = 0;
  const float top = weight.top;
  const auto bounds = [&] {      // of the bin's keys, with room for the roundings of its index
    lo = 0; hi = key_of(top);
    if (__builtin_isfinite(top) && bin0 < BINS - 1) {
      const double a = (double)top - (bin0 + 1) / (double)bin_of.scale * (1 + 1e-6), b = (double)top - bin0 / (double)bin_of.scale * (1 - 1e-6);
      if (a > -3e38) lo = key_of((float)a + 0.f) - 2;
      if (b > -3e38) hi = min(key_of((float)b + 0.f) + 2, hi);
    }
    lo = max(lo, from.key); hi = max(hi, lo);
  };
  int level = 0;
  if (bin0 >= 0) { bounds(); level = 1; }
  for (;; ++level) {
    // level 0: bins of top - x; then bins of 2^s keys in [lo, hi]
    const int s = level == 0 ? 0 : max(0, 32 - __builtin_clz((hi - lo) | 1) - 11);
    clear_bins(sh);
    each([&](float x) {
      const unsigned k = key_of(x);
      if (x == -__builtin_inff() || k < from.key || k < lo || k > hi) return;
      const int b0 = bin_of(x);
      if (level > 0 && b0 != bin0) return;
      const int b = level == 0 ? b0 : (int)((hi - k) >> s);
      if constexpr (!BY_MASS) atomicAdd(&sh.count[b], 1u);
      else if (k != from.key) { const u64 m = fixed(weight(x)); if (m) atomicAdd(&sh.mass[b], m); }
    });
    __syncthreads();
    if constexpr (BY_MASS) {      // the equals of the limit that is there already: only the first of them are kept
      if (threadIdx.x == 0 && from.key != 0 && from.key >= lo && from.key <= hi) {
        const float x = value_of(from.key);
        const int b0 = bin_of(x);
        if (level == 0 || b0 == bin0) sh.mass[level == 0 ? b0 : (int)((hi - from.key) >> s)] += from.ties * fixed(weight(x));
      }
      __syncthreads();
    }
    unsigned counts[PER];
    u64 masses[PER];
    for (int i = 0; i < PER; ++i) { counts[i] = sh.count[threadIdx.x * PER + i]; masses[i] = sh.mass[threadIdx.x * PER + i]; }
    find_bin<BY_MASS>(sh, counts, masses, before_count, before_mass, want_count, want_mass);
    const int f = sh.found;
    if (f < 0) { __syncthreads(); return from; }      // not reached: all of them
    before_count = sh.before_count; before_mass = sh.before_mass;
    if (level == 0) {
      bin0 = f;
      bounds();
    } else {
      hi -= (unsigned)f << s;
      lo = max(lo, hi - ((1u << s) - 1));
      if (s == 0) break;
    }
    __syncthreads();
  }
  Limit r{hi, 0};
  if constexpr (BY_MASS) {
    const u64 m = max(fixed(weight(value_of(hi))), (u64)1), need = want_mass - before_mass;
    r.ties = (unsigned)min((need + m - 1) / m, (u64)0xffffffffu);
    if (hi == from.key) r.ties = min(r.ties, from.ties);
  } else {
    r.ties = want_count - before_count;
  }
  __syncthreads();
  return r;
}

__device__ __forceinline__ u64 share_of(float p, u64 total) {      // the least whole number that is at least p * total, and at least 1
  const double want = (double)p * (double)total;
  u64 m = want > 0 ? (u64)want : 0;
  if ((double)m < want) ++m;
  return m > 0 ? m : 1;
}

__device__ __forceinline__ u64 share_of_draw(float u, u64 total) {      // the token's is the first running sum above it
  const double want = (double)u * (double)total;
  return want > 0 ? (want < (double)total ? min((u64)want, total - 1) : total - 1) : 0;
}

struct Setting { const float* rows; float all; __device__ float operator()(int b) const { return rows ? rows[b] : all; } };
struct Args {
  const void* logits;
  long stride;
  int V, segs;      // segments of a row, at most
  const float* u;
  Setting temperature, top_p, min_p;
  const int* top_k_rows;
  int top_k;
  long* out;
  uint8_t* work;
};

// What a row's blocks leave for each other (in a.work, set up by the first launch).
struct Work {
  u64 *best, *seg_mass, *mass, *candidates;
  unsigned *count, *ticket, *n;
  static __host__ __device__ long bytes(int segs) { return 16l * segs + 12l * BINS + 8l * ROOM + 16; }
  __device__ Work(const Args& a, int b) {
    uint8_t* p = a.work + b * bytes(a.segs);
    best = reinterpret_cast<u64*>(p); seg_mass = best + a.segs; mass = seg_mass + a.segs; candidates = mass + BINS;
    count = reinterpret_cast<unsigned*>(candidates + ROOM); ticket = count + BINS; n = ticket + 1;
  }
};

struct Settings {
  float t, p, min_p;
  int k;      // 0: none
  __device__ __forceinline__ Settings(const Args& a, int b) : t(a.temperature(b)), p(a.top_p(b)) {
    const float m = a.min_p(b);
    min_p = m > 1 ? 1 : m;
    k = a.top_k_rows ? a.top_k_rows[b] : a.top_k;
    if (k <= 0 || k >= a.V) k = 0;
  }
  __device__ __forceinline__ bool greedy() const { return !(t > 0); }
  __device__ __forceinline__ bool cut() const { return k > 0 || p < 1; }
};

// To and from other blocks of the row, past the caches.
template <typename U> __device__ __forceinline__ void put(U* p, U v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename U> __device__ __forceinline__ U get(const U* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// max of key << 32 | ~index over the block
__device__ __forceinline__ u64 block_best(Shared& sh, u64 best) {
  best = wave_max(best);
  if ((threadIdx.x & 63) == 63) sh.wave_mass[threadIdx.x >> 6] = best;
  __syncthreads();
  best = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) best = larger(best, sh.wave_mass[i]);
  __syncthreads();
  return best;
}
template <typename T> __device__ __forceinline__ u64 segment_best(const Row<T>& row, int seg, const float (&x)[8]) {
  u64 best = 0;
  for (int i = 0; i < 8; ++i) {
    const u64 e = (u64)key_of(x[i]) << 32 | (unsigned)~row.index(seg, i);
    best = best > e ? best : e;
  }
  return best;
}
// The rows that need no weights: true if it is done.
template <typename T> __device__ __forceinline__ bool easy(const Args& a, int b, const Row<T>& row, const Settings& set, u64 best, bool writes) {
  const bool none = value_of((unsigned)(best >> 32)) == -__builtin_inff();
  if (!none && !set.greedy()) return false;
  if (writes && threadIdx.x == 0) a.out[b] = none ? -1 : (long)(unsigned)~(unsigned)best - row.shift;
  return true;
}

// The limit by looking at every element, as often as it takes.
template <typename Each> __device__ Limit full_limit(Shared& sh, Each each, const Settings& set, const Weights& weight, const Bins& bins) {
  Limit limit{0, 0};
  if (set.k > 0) limit = find_limit<false>(sh, each, weight, bins, limit, (unsigned)set.k, 0);
  if (set.p < 1) {
    u64 mass = 0;
    unsigned count = 0;
    each([&](float x) { if (key_of(x) > limit.key) mass += fixed(weight(x)); });
    const u64 total = block_scan(sh, count, mass).mass + (limit.key ? limit.ties * fixed(weight(value_of(limit.key))) : 0);
    limit = find_limit<true>(sh, each, weight, bins, limit, 0, share_of(set.p, total));
  }
  return limit;
}
__device__ __forceinline__ u64 kept_mass(const float (&x)[8], const Weights& weight, const Settings& set, unsigned above, unsigned& ties) {
  u64 mass = 0;
  for (int i = 0; i < 8; ++i) {
    const unsigned key = key_of(x[i]);
    ties += key == above;
    if (key <= above) continue;
    const double e = weight(x[i]);
    if (!(e < set.min_p)) mass += fixed(e);
  }
  return mass;
}

// x of the lane whose number differs in bit S: within rows of 16 lanes by data parallel moves (4: all three low bits turned, then the lower two back), across them by swaps
// of rows and halves.
template <int S> __device__ __forceinline__ unsigned across(unsigned x) {
  const auto dpp = [](unsigned v, auto ctrl) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xf, 0xf, false); };
  if constexpr (S == 1) return dpp(x, Number<0xb1>{});
  else if constexpr (S == 2) return dpp(x, Number<0x4e>{});
  else if constexpr (S == 4) return dpp(dpp(x, Number<0x141>{}), Number<0x1b>{});
  else if constexpr (S == 8) return dpp(x, Number<0x128>{});
  else if constexpr (S == 16) { const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false); return threadIdx.x & 16 ? r[0] : r[1]; }
  else { const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false); return threadIdx.x & 32 ? r[0] : r[1]; }
}
// The steps of stride S, S / 2 .. 1 of a bitonic merge of `size` places (i: the thread's), which descend where i & size is 0.
template <int S> __device__ __forceinline__ void merge_in_wave(u64& x, int i, int size) {
  const u64 y = (u64)across<S>((unsigned)(x >> 32)) << 32 | across<S>((unsigned)x);
  if ((y > x) == (((i & S) == 0) == ((i & size) == 0))) x = y;
  if constexpr (S > 1) merge_in_wave<S / 2>(x, i, size);
}
// The n numbers of a wave, those of lanes from n on being 0, in descending order where i & the number of lanes is 0.
template <int SIZE> __device__ __forceinline__ void sort_in_wave(u64& x, int i, int n = 64) {
  if constexpr (SIZE > 2) sort_in_wave<SIZE / 2>(x, i, n);
  if (n > SIZE / 2) merge_in_wave<SIZE / 2>(x, i, SIZE);
}
// Puts up to SORTED numbers in descending order, x[j] being place threadIdx.x + j * NT; also where the result points to, in LDS.  A bitonic sort in registers: strides below
// 64 within a wave, 64 to 256 through LDS, two buffers in turn so that a step takes one barrier, 512 within a thread (53
// numbers 2.0 us and 335 4.0, with all steps through LDS 4.3 and 7.5).
__device__ const u64* put_in_order(Shared& sh, u64 (&x)[2], int n) {
  const int t = threadIdx.x;
  const bool two = n > NT;
  u64* buffer = sh.mass;
  if (t - t % 64 < n) sort_in_wave<64>(x[0], t);
  if (two) sort_in_wave<64>(x[1], t + NT);
  for (int size = 128; size < 2 * n && size <= SORTED; size *= 2) {
    int s = size / 2;
    if (s == NT) {
      if (x[0] < x[1]) { const u64 y = x[0]; x[0] = x[1]; x[1] = y; }
      s /= 2;
    }
    for (; s >= 64; s /= 2) {
      buffer[t] = x[0];
      if (two) buffer[t + NT] = x[1];
      __syncthreads();
      for (int j = 0; j < 2; ++j) {
        if (j == 1 && !two) break;
        const int i = t + j * NT;
        const u64 y = buffer[i ^ s];
        if ((y > x[j]) == (((i & s) == 0) == ((i & size) == 0))) x[j] = y;
      }
      buffer = buffer == sh.mass ? sh.mass + SORTED : sh.mass;
    }
    merge_in_wave<32>(x[0], t, size);
    if (two) merge_in_wave<32>(x[1], t + NT, size);
  }
  buffer[t] = x[0];
  if (two) buffer[t + NT] = x[1];
  __syncthreads();
  return buffer;
}

// Up to 64 candidates (key << 32 | index; what is wanted of them as in candidate_limit), a lane each, by a wave without a barrier: x in order, the weight, its multiple of
// 2^-43, and how many are kept before min-p.
struct Few { u64 x, m; double w; int keep; };
__device__ __forceinline__ Few order_few(u64 candidate, int n, const Settings& set, const Weights& weight, u64 want) {
  const int l = threadIdx.x & 63, k = set.k > 0 ? min(set.k, n) : n;
  Few r{l < n ? candidate ^ 0xffffffffu : 0, 0, 0, k};
  sort_in_wave<64>(r.x, l, n);
  if (l < k) r.w = weight(value_of((unsigned)(r.x >> 32)));
  r.m = fixed(r.w);
  if (set.p < 1) {
    const u64 sum = wave_scan(r.m), target = set.k > 0 ? share_of(set.p, lane(sum, 63)) : want;
    const u64 here = __ballot(sum - r.m < target && sum >= target);
    if (here) r.keep = __builtin_ctzll(here) + 1;
  }
  return r;
}
// With a k, everything that may be kept is a candidate: the token of a row with up to 64 of them, by the first wave.  Index (below 2^20) and sum (up to 2^43) of a candidate are one
// number, which puts them in the order of the vocabulary (4 rows of 128256, k 50: 16.6 us; by the sums of segments and a second look at the token's 19.3).
__device__ __forceinline__ void draw_few(long* out, int shift, float u, u64 candidate, int n, const Settings& set, const Weights& weight) {
  constexpr u64 MASS = ((u64)1 << 44) - 1;
  if (threadIdx.x >= 64) return;
  const int l = threadIdx.x;
  const Few c = order_few(candidate, n, set, weight, 0);
  u64 y = l < c.keep && !(c.w < set.min_p) && c.m > 0 ? (c.x & 0xfffff) << 44 | c.m : 0;      // (x has the index inverted)
  sort_in_wave<64>(y, l, n);
  const u64 m = y & MASS, sum = wave_scan(m), total = lane(sum, 63), target = share_of_draw(u, total);
  if (sum - m <= target && target < sum) *out = (long)(~(unsigned)(y >> 44) & 0xfffff) - shift;
}

// The limit among n candidates (key << 32 | index): all elements of the order up to the limit, with a k, or all of the bin that it falls in, without; `want` is then
// what is wanted of their sum.  first: the lane's of the first 64; mine: the thread's of the first SORTED; values: room for all of them in LDS.
__device__ Limit candidate_limit(Shared& sh, u64 first, const u64 (&mine)[2], const u64* cand, int n, float* values, const Settings& set, const Weights& weight, const Bins& bins, u64 want, int bin) {
  if (n <= 64) {      // each wave by itself
    const Few c = order_few(first, n, set, weight, want);
    const unsigned key = (unsigned)(c.x >> 32), last = (unsigned)__builtin_amdgcn_readlane((int)key, c.keep - 1);
    return Limit{last, (unsigned)__builtin_popcountll(__ballot((int)(threadIdx.x & 63) < c.keep && key == last))};
  }
  if (n <= SORTED) {
    u64 x[2];      // places threadIdx.x and NT + threadIdx.x; descends in the order, none: last
    for (int j = 0; j < 2; ++j) x[j] = (int)threadIdx.x + j * NT < n ? mine[j] ^ 0xffffffffu : 0;
    const u64* sorted = put_in_order(sh, x, n);
    const bool two = n > NT;
    const int k = set.k > 0 ? min(set.k, n) : n;
    int keep = k;
    if (set.p < 1) {
      u64 m[2] = {0, 0}, mass[2], all = 0;
      unsigned none = 0;
      for (int j = 0; j < 2; ++j) {
        if (j == 1 && !two) break;
        if ((int)threadIdx.x + j * NT < k) m[j] = fixed(weight(value_of((unsigned)(x[j] >> 32))));
        mass[j] = m[j];
        const u64 sum = block_scan(sh, none, mass[j]).mass;
        mass[j] += all;
        all += sum;
      }
      const u64 target = set.k > 0 ? share_of(set.p, all) : want;
      if (threadIdx.x == 0) sh.found = k;
      __syncthreads();
      for (int j = 0; j < 2; ++j)
        if ((j == 0 || two) && mass[j] - m[j] < target && mass[j] >= target) sh.found = threadIdx.x + j * NT + 1;      // (with m 0: no place)
      __syncthreads();
      keep = sh.found;
    }
    const unsigned last = (unsigned)(sorted[keep - 1] >> 32);
    for (int j = 0; j < 2; ++j) {      // the first of the last one's equals
      const int i = threadIdx.x + j * NT;
      if (i < n && (unsigned)(x[j] >> 32) == last && (i == 0 || (unsigned)(sorted[i - 1] >> 32) != last)) sh.before_count = i;
    }
    __syncthreads();
    return Limit{last, keep - sh.before_count};
  }
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += NT) values[i] = value_of((unsigned)(get(cand + i) >> 32));      // (each thread reads its own)
  const auto each = [&](auto f) { for (int i = threadIdx.x; i < n; i += NT) f(values[i]); };
  return set.k > 0 ? full_limit(sh, each, set, weight, bins) : find_limit<true>(sh, each, weight, bins, Limit{0, 0}, 0, want, bin);
}

// The token: sh.seg_mass and sh.seg_ties hold, by segments, the kept sums above limit.key and the number of its equals.
template <typename T> __device__ void draw(Shared& sh, const Args& a, int b, float u, const Row<T>& row, const Settings& set, const Weights& weight, Limit limit) {
  constexpr int EACH = (MAX_SEGS + 63) / 64;      // segments of a lane: each wave looks for the token's by itself, without a barrier
  const int segs = row.segs(), l = threadIdx.x & 63;
  const double tie_weight = limit.key ? weight(value_of(limit.key)) : 0.0;
  const u64 tie_mass = tie_weight < set.min_p ? 0 : fixed(tie_weight);
  unsigned own_ties[EACH], ties = 0, lane_ties = 0;
  u64 own[EACH], mass = 0, lane_mass = 0;
  for (int i = 0; i < EACH; ++i) {
    const int s = l * EACH + i;
    own_ties[i] = s < segs ? sh.seg_ties[s] : 0;
    own[i] = s < segs ? sh.seg_mass[s] : 0;
    lane_ties += own_ties[i];
  }
  ties = wave_scan(lane_ties) - lane_ties;      // before the lane's, then before the segment found
  for (int i = 0; i < EACH; ++i) {
    own[i] += tie_mass * (ties >= limit.ties ? 0u : min(own_ties[i], limit.ties - ties));
    ties += own_ties[i];
    lane_mass += own[i];
  }
  ties -= lane_ties;
  mass = wave_scan(lane_mass);
  const u64 total = lane(mass, 63);
  mass -= lane_mass;
  const u64 target = share_of_draw(u, total);
  const bool here = mass <= target && target < mass + lane_mass;
  int at = 0;
  unsigned in_segment = 0;
  bool passed = false;
  for (int i = 0; i < EACH; ++i) {
    if (passed) continue;
    passed = target < mass + own[i];
    if (passed) { at = l * EACH + i; in_segment = own_ties[i]; }
    else { mass += own[i]; ties += own_ties[i]; }
  }
  const int src = __builtin_ctzll(__ballot(here));
  const int seg = __builtin_amdgcn_readlane(at, src);
  const u64 before_mass = lane(mass, src);
  const unsigned before_ties = __builtin_amdgcn_readlane(ties, src);
  const bool all_ties = before_ties + (unsigned)__builtin_amdgcn_readlane(in_segment, src) <= limit.ties;
  float x[8];
  row.load(seg, x);
  unsigned seen = before_ties, none = 0;
  if (!all_ties) {
    unsigned t = 0;
    for (int i = 0; i < 8; ++i) t += key_of(x[i]) == limit.key;
    seen -= t;
    u64 no_mass = 0;
    block_scan(sh, t, no_mass);
    seen += t;
  }
  u64 e[8], sum = 0;
  for (int i = 0; i < 8; ++i) {
    const unsigned key = key_of(x[i]);
    e[i] = 0;
    if (key == limit.key) { if (all_ties || seen++ < limit.ties) e[i] = tie_mass; }
    else if (key > limit.key) { const double y = weight(x[i]); if (!(y < set.min_p)) e[i] = fixed(y); }
    sum += e[i];
  }
  mass = sum;
  block_scan(sh, none, mass);
  u64 run = before_mass + mass - sum;
  for (int i = 0; i < 8; ++i) {
    if (run <= target && target < run + e[i]) a.out[b] = row.index(seg, i) - row.shift;
    run += e[i];
  }
}

// Whether this block is the last of its row to come here.  What the blocks leave for it they store past the caches (put, or an atomic), which is waited for here, and it
// reads them past the caches (get): a release and an acquire would write back and empty a whole L2 in each block.
__device__ __forceinline__ bool last_of_row(Shared& sh, const Work& work) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) sh.last = __hip_atomic_fetch_add(work.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  __syncthreads();
  return sh.last;
}

// The bin where the limit falls, in sh.found (-1: there are fewer than k): by count where there is a k, otherwise by sum, and then what is wanted of that bin's.
// up_to: with a k, the elements up to that bin.
__device__ __forceinline__ u64 find_cut(Shared& sh, const Settings& set, const unsigned (&counts)[PER], const u64 (&masses)[PER], unsigned& up_to) {
  up_to = 0;
  if (set.k > 0) {
    const unsigned all = find_bin<false>(sh, counts, masses, 0, 0, (unsigned)set.k, 0);
    up_to = sh.found < 0 ? all : sh.before_count + sh.found_count;
    return 0;
  }
  u64 m = 0;
  unsigned c = 0;
  for (int i = 0; i < PER; ++i) m += masses[i];
  const u64 want = share_of(set.p, block_scan(sh, c, m).mass);
  find_bin<true>(sh, counts, masses, 0, 0, 0, want);
  return want - sh.before_mass;
}

// First launch: the maximum of each segment; what the row's blocks add to later is zeroed.  A block takes every gridDim.x-th segment, in all launches.
template <typename T> __global__ __launch_bounds__(NT) void k_sample_max(Args a) {
  __shared__ Shared sh;
  const int b = blockIdx.y;
  const Row<T> row(static_cast<const T*>(a.logits) + b * a.stride, a.V);
  const Work work(a, b);
  const auto first = row.fetch(blockIdx.x);
  for (int i = blockIdx.x * NT + threadIdx.x; i < BINS; i += gridDim.x * NT) { work.mass[i] = 0; work.count[i] = 0; }
  if (blockIdx.x == 0 && threadIdx.x == 0) *work.ticket = *work.n = 0;
  row.each_segment(a.segs, blockIdx.x, gridDim.x, first, [&](int seg, const float (&x)[8]) {
    const u64 best = block_best(sh, segment_best(row, seg, x));
    if (threadIdx.x == 0) { work.best[seg] = best; work.seg_mass[seg] = 0; }
  });
}

__device__ __forceinline__ void add_to_bins(Shared& sh, const Settings& set, const Weights& weight, const Bins& bins, const float (&x)[8]) {
  for (int i = 0; i < 8; ++i) {
    const int bin = bins(x[i]);
    if (set.k > 0) {
      if (x[i] != -__builtin_inff()) atomicAdd(&sh.count[bin], 1u);
      continue;
    }
    const u64 m = fixed(weight(x[i]));
    if (m) atomicAdd(&sh.mass[bin], m);
  }
}

template <typename T> __device__ __forceinline__ void draw_kept(Shared& sh, const Args& a, int b, float u, const Row<T>& row, const Settings& set, const Weights& weight, const Work& work) {
  if (threadIdx.x < row.segs()) { sh.seg_mass[threadIdx.x] = get(work.seg_mass + threadIdx.x); sh.seg_ties[threadIdx.x] = 0; }
  __syncthreads();
  draw(sh, a, b, u, row, set, weight, Limit{0, 0});
}

// Second: rows that are cut get their bins (counts where there is a k, which leaves few elements to look at, otherwise sums), the others their token.
template <typename T> __global__ __launch_bounds__(NT) void k_sample_bins(Args a) {
  __shared__ Shared sh;
  const int b = blockIdx.y, l = threadIdx.x & 63;
  const Row<T> row(static_cast<const T*>(a.logits) + b * a.stride, a.V);
  const Work work(a, b);
  const Settings set(a, b);
  const float u = a.u[b];      // (fetched with the first loads)
  const auto first = row.fetch(blockIdx.x);
  fill_roots(sh.roots);
  const u64 best = block_best(sh, threadIdx.x < a.segs ? work.best[threadIdx.x] : 0);
  if (easy(a, b, row, set, best, blockIdx.x == 0)) return;
  const Weights weight(value_of((unsigned)(best >> 32)), set.t, sh.roots);
  if (set.cut()) {
    const Bins bins(weight.top, set.t);
    clear_bins(sh);
    row.each_segment(a.segs, blockIdx.x, gridDim.x, first, [&](int, const float (&x)[8]) { add_to_bins(sh, set, weight, bins, x); });
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += NT) {
      if (sh.count[i]) atomicAdd(&work.count[i], sh.count[i]);
      if (sh.mass[i]) atomicAdd(&work.mass[i], sh.mass[i]);
    }
    return;
  }
  row.each_segment(a.segs, blockIdx.x, gridDim.x, first, [&](int seg, const float (&x)[8]) {
    unsigned ties = 0;
    const u64 mass = wave_scan(kept_mass(x, weight, set, 0, ties));
    if (l == 63 && mass) atomicAdd(&work.seg_mass[seg], mass);
  });
  if (last_of_row(sh, work)) draw_kept(sh, a, b, u, row, set, weight, work);
}

// Third: the bin where the limit falls; its elements (with k: all up to it) become candidates, of what stands before it the segments' sums are taken.  The
// row's last block finds the limit among the candidates and draws.
template <typename T> __global__ __launch_bounds__(NT) void k_sample_draw(Args a) {
  __shared__ Shared sh;
  __shared__ float values[ROOM];
  const int b = blockIdx.y, l = threadIdx.x & 63;
  const Row<T> row(static_cast<const T*>(a.logits) + b * a.stride, a.V);
  const Settings set(a, b);
  if (!set.cut() || set.greedy()) return;
  const Work work(a, b);
  const float u = a.u[b];
  const auto first = row.fetch(blockIdx.x);
  fill_roots(sh.roots);
  unsigned counts[PER];
  u64 masses[PER];
  for (int i = 0; i < PER; ++i) {
    counts[i] = set.k > 0 ? work.count[threadIdx.x * PER + i] : 0;
    masses[i] = set.k > 0 ? 0 : work.mass[threadIdx.x * PER + i];
  }
  const u64 best = block_best(sh, threadIdx.x < a.segs ? work.best[threadIdx.x] : 0);
  if (easy(a, b, row, set, best, false)) return;
  const Weights weight(value_of((unsigned)(best >> 32)), set.t, sh.roots);
  const Bins bins(weight.top, set.t);
  unsigned up_to_k;
  const u64 want = find_cut(sh, set, counts, masses, up_to_k);
  const int f = sh.found < 0 ? BINS - 1 : sh.found;      // fewer than k: all of them
  const bool few = up_to_k <= ROOM;
  row.each_segment(few ? a.segs : 0, blockIdx.x, gridDim.x, first, [&](int seg, const float (&x)[8]) {
    u64 mass = 0;
    unsigned mine = 0, take = 0;
    for (int i = 0; i < 8; ++i) {
      if (x[i] == -__builtin_inff()) continue;
      const int bin = bins(x[i]);
      if (set.k > 0 ? bin <= f : bin == f) { take |= 1u << i; ++mine; }
      else if (set.k == 0 && bin < f) { const double e = weight(x[i]); if (!(e < set.min_p)) mass += fixed(e); }
    }
    if (set.k == 0) {
      mass = wave_scan(mass);
      if (l == 63 && mass) atomicAdd(&work.seg_mass[seg], mass);
    }
    if (__ballot(mine > 0) == 0) return;
    const unsigned run = wave_scan(mine);
    unsigned at = 0;
    if (l == 63) at = atomicAdd(work.n, run);
    at = (unsigned)__builtin_amdgcn_readlane((int)at, 63) + run - mine;
    for (int i = 0; i < 8; ++i)
      if (take >> i & 1) { if (at < ROOM) put(work.candidates + at, (u64)key_of(x[i]) << 32 | (unsigned)row.index(seg, i)); ++at; }
  });
  if (!last_of_row(sh, work)) return;
  const int segs = row.segs();
  const u64 seg_mass = threadIdx.x < segs ? get(work.seg_mass + threadIdx.x) : 0, mine[2] = {get(work.candidates + threadIdx.x), get(work.candidates + NT + threadIdx.x)};      // (some of it unset: how many there are comes with it)
  const u64 first_few = get(work.candidates + l);
  const unsigned n = few ? get(work.n) : up_to_k;
  if (set.k > 0 && n <= 64) {
    draw_few(a.out + b, row.shift, u, first_few, (int)n, set, weight);
    return;
  }
  Limit limit;
  if (n <= ROOM) {
    if (threadIdx.x < segs) { sh.seg_mass[threadIdx.x] = seg_mass; sh.seg_ties[threadIdx.x] = 0; }
    limit = candidate_limit(sh, first_few, mine, work.candidates, (int)n, values, set, weight, bins, want, f);
    __syncthreads();
    const auto keep = [&](u64 c) {
      const unsigned key = (unsigned)(c >> 32);
      if (key < limit.key) return;
      const int s = (unsigned)c / SEG;
      if (key == limit.key) { atomicAdd(&sh.seg_ties[s], 1u); return; }
      const double e = weight(value_of(key));
      if (!(e < set.min_p)) atomicAdd(&sh.seg_mass[s], fixed(e));
    };
    for (int j = 0; j < 2; ++j) if (threadIdx.x + j * NT < n) keep(mine[j]);
#pragma unroll 4
    for (int i = threadIdx.x + SORTED; i < (int)n; i += NT) keep(get(work.candidates + i));
  } else {
    limit = full_limit(sh, [&](auto f) {
      for (int s = 0; s < segs; ++s) {
        float y[8];
        row.load(s, y);
        for (int i = 0; i < 8; ++i) f(y[i]);
      }
    }, set, weight, bins);
    for (int s = 0; s < segs; ++s) {
      float x[8];
      row.load(s, x);
      unsigned ties = 0;
      u64 sum = kept_mass(x, weight, set, limit.key, ties);
      const Sums all = block_scan(sh, ties, sum);
      if (threadIdx.x == 0) { sh.seg_mass[s] = all.mass; sh.seg_ties[s] = all.count; }
    }
  }
  __syncthreads();
  draw(sh, a, b, u, row, set, weight, limit);
}

// Rows of one segment, in one launch: the same steps by one block, with the bins and candidates in LDS.
template <typename T> __global__ __launch_bounds__(NT) void k_sample_short(Args a) {
  __shared__ Shared sh;
  __shared__ u64 cand[SEG];
  __shared__ float values[SEG];
  __shared__ int n;
  const int b = blockIdx.y, l = threadIdx.x & 63;
  const Row<T> row(static_cast<const T*>(a.logits) + b * a.stride, a.V);
  const Settings set(a, b);
  const float u = a.u[b];      // (fetched with the first loads)
  float x[8];
  row.load(0, x);
  fill_roots(sh.roots);
  if (threadIdx.x == 0) n = 0;
  const u64 best = block_best(sh, segment_best(row, 0, x));
  if (easy(a, b, row, set, best, true)) return;
  const Weights weight(value_of((unsigned)(best >> 32)), set.t, sh.roots);
  Limit limit{0, 0};
  if (set.cut()) {
    const Bins bins(weight.top, set.t);
    clear_bins(sh);
    add_to_bins(sh, set, weight, bins, x);
    __syncthreads();
    unsigned counts[PER];
    u64 masses[PER];
    for (int i = 0; i < PER; ++i) { counts[i] = sh.count[threadIdx.x * PER + i]; masses[i] = sh.mass[threadIdx.x * PER + i]; }
    unsigned up_to_k;
    const u64 want = find_cut(sh, set, counts, masses, up_to_k);
    const int f = sh.found < 0 ? BINS - 1 : sh.found;
    for (int i = 0; i < 8; ++i) {
      if (x[i] == -__builtin_inff()) continue;
      const int bin = bins(x[i]);
      if (set.k > 0 ? bin <= f : bin == f) cand[atomicAdd(&n, 1)] = (u64)key_of(x[i]) << 32 | (unsigned)row.index(0, i);
    }
    __syncthreads();
    if (set.k > 0 && n <= 64) {
      draw_few(a.out + b, row.shift, u, cand[l], n, set, weight);
      return;
    }
    const u64 mine[2] = {cand[threadIdx.x], cand[NT + threadIdx.x]};
    limit = candidate_limit(sh, cand[l], mine, cand, n, values, set, weight, bins, want, f);
  }
  unsigned ties = 0;
  u64 mass = kept_mass(x, weight, set, limit.key, ties);
  const Sums all = block_scan(sh, ties, mass);
  if (threadIdx.x == 0) { sh.seg_mass[0] = all.mass; sh.seg_ties[0] = all.count; }
  __syncthreads();
  draw(sh, a, b, u, row, set, weight, limit);
}

constexpr int ROWS = 1024, SHORT_ROWS = 65535;      // rows of a launch, at most: there is work memory for so many
int segments(int V) { return (V + 7 + SEG - 1) / SEG; }      // whatever the rows' alignment
long work_needed(int B, int V) { return segments(V) == 1 ? 0 : min(B, ROWS) * Work::bytes(segments(V)); }

template <typename T> int launch(Args a, int B, bool cut, hipStream_t stream) {
  const int rows = a.segs == 1 ? SHORT_ROWS : ROWS;
  for (int b = 0; b < B; b += rows) {
    const int n = min(B - b, rows);
    // two blocks a CU: each starts with the row's maxima or bins, which costs as much as several segments (64 rows of 128256 by top-p: 42.2 us, 51.1 with 256 blocks, 48.2 with 1024)
    const dim3 grid(min(a.segs, max(BLOCKS / n, 1)), n);
    if (a.segs == 1) {
      k_sample_short<T><<<grid, NT, 0, stream>>>(a);
    } else {
      k_sample_max<T><<<grid, NT, 0, stream>>>(a);
      k_sample_bins<T><<<grid, NT, 0, stream>>>(a);
      if (cut) k_sample_draw<T><<<grid, NT, 0, stream>>>(a);
    }
    a.logits = static_cast<const T*>(a.logits) + n * a.stride;
    a.u += n; a.out += n;
    for (Setting* s : {&a.temperature, &a.top_p, &a.min_p}) if (s->rows) s->rows += n;
    if (a.top_k_rows) a.top_k_rows += n;
  }
  return gaac::launch_status("gaac_sample");
}

}  // namespace

extern "C" int gaac_sample(int type, const void* logits, long row_stride, int B, int V, const float* u, const float* temperature_rows, float temperature, const int* top_k_rows, int top_k,
                           const float* top_p_rows, float top_p, const float* min_p_rows, float min_p, void* work, long work_bytes, int64_t* out, void* stream) {
  GAAC_REQUIRE(logits != nullptr && u != nullptr && out != nullptr, "gaac_sample: null pointer");
  GAAC_REQUIRE(type >= 0 && type <= 2, "gaac_sample: type must be 0 (bf16), 1 (fp16) or 2 (fp32)");
  GAAC_REQUIRE(B > 0 && V > 0 && V <= MAX_V - 16 && row_stride >= 0, "gaac_sample: bad sizes (%d rows of %d logits, at most %d)", B, V, MAX_V - 16);
  GAAC_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (type == 2 ? 4 : 2) == 0, "gaac_sample: logits are not aligned to their type");
  const int segs = segments(V);
  GAAC_REQUIRE(reinterpret_cast<uintptr_t>(work) % 8 == 0 && work_bytes >= work_needed(B, V) && (work != nullptr || segs == 1), "gaac_sample: %ld bytes of work memory, aligned to 8, are too few", work_bytes);
  const Args a{logits, row_stride, V, segs, u, {temperature_rows, temperature}, {top_p_rows, top_p}, {min_p_rows, min_p}, top_k_rows, top_k, (long*)out, (uint8_t*)work};
  const bool cut = top_k_rows != nullptr || top_p_rows != nullptr || (top_k > 0 && top_k < V) || top_p < 1;
  if (type == 0) return launch<__bf16>(a, B, cut, (hipStream_t)stream);
  if (type == 1) return launch<_Float16>(a, B, cut, (hipStream_t)stream);
  return launch<float>(a, B, cut, (hipStream_t)stream);
}
