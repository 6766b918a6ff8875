// One token per row of logits: temperature, top-k, top-p, min-p, and a given random number u in [0, 1).
//   w_i = exp((x_i - max) / T).  Order: x descending, then index ascending.  Kept: the first k in the order; of these the shortest prefix whose sum of w is at
//   least p times theirs; of these the ones with w >= min_p (the maximum has 1).  Token: the first i, by index, at which the running sum of the kept w
//   exceeds u times their total.  T not positive: the first maximum.  Nothing but -inf (a NaN counts as one): -1.
//
// Which token comes is a whole number, so a sum that is off in its last bits is an error: weights are computed in 64 bits and held as multiples of 2^-43
// in 64-bit integers (2^20 of them fit), whose sums are exact in any order.
// What is kept is a prefix of the order, so it is found as a key (the bits of x, in order) and the number of its equals that are kept: counts and sums by bins
// of (max - x), then by ever finer bins of the key within the bin where the limit falls.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "gaac_capi.h"
#include "../../include/gaac_hip.h"

namespace {

constexpr int NT = 1024, BINS = 2048, CHUNK = 512, MAX_V = 1 << 20, MAX_CHUNKS = MAX_V / CHUNK;
static_assert(MAX_CHUNKS <= BINS);
typedef unsigned long long u64;
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

// The row as chunks of 512 elements from the 16-byte boundary at or below its start; a lane has 8 in a row.  Elements before and behind the row are -inf.
template <typename T> struct Row {
  const T* base;      // aligned
  int shift, V;       // row element i is base[shift + i]
  __device__ __forceinline__ int chunks() const { return (shift + V + CHUNK - 1) / CHUNK; }
  __device__ __forceinline__ void load(int chunk, int l, float (&x)[8]) const {
    constexpr int G = 16 / sizeof(T);      // elements of a 16-byte load
    for (int part = 0; part < 8 / G; ++part) {
      const int at = chunk * CHUNK + l * 8 + part * G;
      if (at >= shift && at + G <= shift + V) {
        const u4 raw = *reinterpret_cast<const u4*>(base + at);
        T v[G];
        __builtin_memcpy(v, &raw, 16);
        for (int i = 0; i < G; ++i) x[part * G + i] = number(v[i]);
      } else {
        for (int i = 0; i < G; ++i) x[part * G + i] = at + i >= shift && at + i < shift + V ? number(base[at + i]) : -__builtin_inff();
      }
    }
  }
};

// exp(y), y <= 0, as a multiple of 2^-43: y = n ln 2 + r, the series of exp to r^11 (|r| <= 0.35: what is left is below 1e-14), and the sum with 2^9, whose
// last bit is 2^-43, rounds to it.
__device__ __forceinline__ double exp64(double y) {
  if (!(y > -31.0)) return 0.0;
  const double n = __builtin_rint(y * 1.4426950408889634);
  const double r = __builtin_fma(n, -5.5459262969660605e-09, __builtin_fma(n, -0.693147175014019, y));      // ln 2 = 27 bits of it and the rest
  double e = 1.0 / 39916800;
  e = __builtin_fma(e, r, 1.0 / 3628800);
  e = __builtin_fma(e, r, 1.0 / 362880);
  e = __builtin_fma(e, r, 1.0 / 40320);
  e = __builtin_fma(e, r, 1.0 / 5040);
  e = __builtin_fma(e, r, 1.0 / 720);
  e = __builtin_fma(e, r, 1.0 / 120);
  e = __builtin_fma(e, r, 1.0 / 24);
  e = __builtin_fma(e, r, 1.0 / 6);
  e = __builtin_fma(e, r, 0.5);
  e = __builtin_fma(e, r, 1.0);
  e = __builtin_fma(e, r, 1.0);
  return __builtin_bit_cast(double, __builtin_bit_cast(u64, e) + ((u64)(long long)n << 52));
}
__device__ __forceinline__ u64 fixed(double w) { return __builtin_bit_cast(u64, w + 512.0) - __builtin_bit_cast(u64, 512.0); }

struct Weights {      // of a row
  float top;
  double inv_t;
  __device__ __forceinline__ double operator()(float x) const {
    if (x == top) return 1.0;
    return x == -__builtin_inff() ? 0.0 : exp64(((double)x - (double)top) * inv_t);
  }
};

__device__ __forceinline__ u64 wave_scan(u64 x, int l) {      // inclusive
  for (int o = 1; o < 64; o <<= 1) { const u64 y = __shfl_up(x, o); if (l >= o) x += y; }
  return x;
}

struct Shared {
  u64 mass[BINS];           // of bins; of chunks
  unsigned count[BINS];
  u64 wave_mass[16];
  unsigned wave_count[16];
  u64 best[16];
  u64 total;
  u64 before_mass;
  unsigned before_count;
  int found;
};

// Inclusive prefix sums over the block of each thread's (count, mass); afterwards sh.total and the last thread's count are complete.
__device__ __forceinline__ void block_scan(Shared& sh, unsigned& count, u64& mass) {
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  mass = wave_scan(mass, l);
  count = (unsigned)wave_scan(count, l);
  if (l == 63) { sh.wave_mass[w] = mass; sh.wave_count[w] = count; }
  __syncthreads();
  for (int i = 0; i < w; ++i) { mass += sh.wave_mass[i]; count += sh.wave_count[i]; }
  __syncthreads();
}

// Where a limit falls: the key of the last element kept, how many of its equals are, and count and sum of what stands before that key.
struct Limit { unsigned key, ties; };

// The first element in the order at which the running count reaches `count` (BY_MASS false) or the running sum of weights reaches `mass` (true), among the
// elements with key above `from.key` and from.ties of its equals.
template <bool BY_MASS, typename T>
__device__ Limit find_limit(Shared& sh, const Row<T>& row, const Weights& weight, float bin_scale, Limit from, unsigned want_count, u64 want_mass) {
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, chunks = row.chunks();
  unsigned lo = 0, hi = 0xffffffffu, before_count = 0;
  u64 before_mass = 0;
  int bin0 = -1;
  const float top = weight.top;
  const auto bin_of = [&](float x) { return x == top ? 0 : (int)fminf((top - x) * bin_scale, (float)(BINS - 1)); };      // never ascends with x
  for (int level = 0;; ++level) {
    // level 0: bins of top - x; then bins of 2^s keys in [lo, hi]
    const int s = level == 0 ? 0 : max(0, 32 - __builtin_clz((hi - lo) | 1) - 11);
    for (int i = threadIdx.x; i < BINS; i += NT) { sh.mass[i] = 0; sh.count[i] = 0; }
    __syncthreads();
    for (int c = w; c < chunks; c += NT / 64) {
      float x[8];
      row.load(c, l, x);
      for (int i = 0; i < 8; ++i) {
        const unsigned k = key_of(x[i]);
        if (x[i] == -__builtin_inff() || k < from.key || k < lo || k > hi) continue;
        const int b0 = bin_of(x[i]);
        if (level > 0 && b0 != bin0) continue;
        const int b = level == 0 ? b0 : (int)((hi - k) >> s);
        atomicAdd(&sh.count[b], 1u);
        if constexpr (BY_MASS) if (k != from.key) { const u64 m = fixed(weight(x[i])); if (m) atomicAdd(&sh.mass[b], m); }
      }
    }
    __syncthreads();
    if constexpr (BY_MASS) {      // the equals of the limit that is there already: only the first of them are kept
      if (threadIdx.x == 0 && from.key != 0 && from.key >= lo && from.key <= hi) {
        const float x = value_of(from.key);
        const int b0 = bin_of(x);
        if (level == 0 || b0 == bin0) sh.mass[level == 0 ? b0 : (int)((hi - from.key) >> s)] += from.ties * fixed(weight(x));
      }
      __syncthreads();
    }
    unsigned count = 0;
    u64 mass = 0;
    const int b0 = threadIdx.x * (BINS / NT);
    for (int i = 0; i < BINS / NT; ++i) { count += sh.count[b0 + i]; mass += sh.mass[b0 + i]; }
    const unsigned own_count = count;
    const u64 own_mass = mass;
    if (threadIdx.x == 0) sh.found = -1;
    block_scan(sh, count, mass);
    count += before_count - own_count; mass += before_mass - own_mass;      // before this thread's bins
    for (int i = 0; i < BINS / NT; ++i) {
      const bool reached = BY_MASS ? mass < want_mass && mass + sh.mass[b0 + i] >= want_mass : count < want_count && count + sh.count[b0 + i] >= want_count;
      if (reached) { sh.found = b0 + i; sh.before_count = count; sh.before_mass = mass; }
      count += sh.count[b0 + i]; mass += sh.mass[b0 + i];
    }
    __syncthreads();
    const int f = sh.found;
    if (f < 0) return from.key ? from : Limit{0, 0};      // not reached: all of them
    before_count = sh.before_count; before_mass = sh.before_mass;
    if (level == 0) {
      bin0 = f;
      if (__builtin_isfinite(top) && f < BINS - 1) {      // bounds of the bin's keys, with room for the roundings of its index
        const double a = (double)top - (f + 1) / (double)bin_scale * (1 + 1e-6), b = (double)top - f / (double)bin_scale * (1 - 1e-6);
        lo = key_of((float)a + 0.f) - 2; hi = min(key_of((float)b + 0.f) + 2, key_of(top));
        if (!(a > -3e38)) lo = 0;
      } else {
        lo = 0; hi = key_of(top);
      }
      lo = max(lo, from.key); hi = max(hi, lo);
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

struct Setting { const float* rows; float all; __device__ float operator()(int b) const { return rows ? rows[b] : all; } };
struct Args {
  const void* logits;
  long stride;
  int V;
  const float* u;
  Setting temperature, top_p, min_p;
  const int* top_k_rows;
  int top_k;
  long* out;
};

template <typename T> __global__ __launch_bounds__(NT) void k_sample(Args a) {
  __shared__ Shared sh;
  const int b = blockIdx.x, l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const T* start = static_cast<const T*>(a.logits) + b * a.stride;
  const int shift = (int)(reinterpret_cast<uintptr_t>(start) % 16 / sizeof(T));
  const Row<T> row{start - shift, shift, a.V};
  const int chunks = row.chunks();
  // the maximum, and the first place that has it
  u64 best = 0;
  for (int c = w; c < chunks; c += NT / 64) {
    float x[8];
    row.load(c, l, x);
    for (int i = 0; i < 8; ++i) {
      const u64 e = (u64)key_of(x[i]) << 32 | (unsigned)~(c * CHUNK + l * 8 + i);
      best = best > e ? best : e;
    }
  }
  for (int o = 32; o > 0; o >>= 1) { const u64 y = __shfl_xor(best, o); best = best > y ? best : y; }
  if (l == 0) sh.best[w] = best;
  __syncthreads();
  for (int i = 0; i < NT / 64; ++i) best = best > sh.best[i] ? best : sh.best[i];
  const float top = value_of((unsigned)(best >> 32)), t = a.temperature(b);
  if (top == -__builtin_inff()) { if (threadIdx.x == 0) a.out[b] = -1; return; }
  if (!(t > 0)) { if (threadIdx.x == 0) a.out[b] = (long)(unsigned)~(unsigned)best - shift; return; }
  const Weights weight{top, 1.0 / (double)t};
  const float bin_scale = fmaxf(32.f / t, 32.f), p = a.top_p(b), m = a.min_p(b), min_p = m > 1 ? 1 : m;
  const int k = a.top_k_rows ? a.top_k_rows[b] : a.top_k;
  Limit limit{0, 0};      // key 0: none
  if (k > 0 && k < a.V) limit = find_limit<false>(sh, row, weight, bin_scale, limit, (unsigned)k, 0);
  if (p < 1) {
    // the sum that p is a share of
    u64 mass = 0;
    for (int c = w; c < chunks; c += NT / 64) {
      float x[8];
      row.load(c, l, x);
      for (int i = 0; i < 8; ++i) if (key_of(x[i]) > limit.key) mass += fixed(weight(x[i]));
    }
    unsigned count = 0;
    block_scan(sh, count, mass);
    if (threadIdx.x == NT - 1) sh.total = mass;
    __syncthreads();
    u64 total = sh.total;
    if (limit.key) total += limit.ties * fixed(weight(value_of(limit.key)));
    const double want = (double)p * (double)total;
    u64 target = want > 0 ? (u64)want : 0;
    if ((double)target < want) ++target;
    limit = find_limit<true>(sh, row, weight, bin_scale, limit, 0, target > 0 ? target : 1);
  }
  // sums of what is kept, by chunks
  for (int c = w; c < chunks; c += NT / 64) {
    float x[8];
    row.load(c, l, x);
    u64 mass = 0;
    unsigned ties = 0;
    for (int i = 0; i < 8; ++i) {
      const unsigned key = key_of(x[i]);
      if (key < limit.key) continue;
      if (key == limit.key) { ++ties; continue; }
      const double e = weight(x[i]);
      if (!(e < min_p)) mass += fixed(e);
    }
    for (int o = 32; o > 0; o >>= 1) { mass += __shfl_xor(mass, o); ties += __shfl_xor(ties, o); }
    if (l == 0) { sh.mass[c] = mass; sh.count[c] = ties; }
  }
  __syncthreads();
  const double tie_weight = limit.key ? weight(value_of(limit.key)) : 0.0;
  const u64 tie_mass = tie_weight < min_p ? 0 : fixed(tie_weight);
  constexpr int PER = (MAX_CHUNKS + NT - 1) / NT;
  unsigned ties = 0;
  u64 mass = 0;
  for (int i = 0; i < PER; ++i) { const int c = threadIdx.x * PER + i; if (c < chunks) ties += sh.count[c]; }
  const unsigned own_ties = ties;
  block_scan(sh, ties, mass);
  ties -= own_ties;
  const unsigned first_ties = ties;
  const auto kept_mass = [&](int c, unsigned before) { return sh.mass[c] + tie_mass * (before >= limit.ties ? 0u : min(sh.count[c], limit.ties - before)); };
  mass = 0;
  for (int i = 0; i < PER; ++i) { const int c = threadIdx.x * PER + i; if (c < chunks) { mass += kept_mass(c, ties); ties += sh.count[c]; } }
  const u64 own_mass = mass;
  unsigned none = 0;
  block_scan(sh, none, mass);
  if (threadIdx.x == NT - 1) sh.total = mass;
  __syncthreads();
  const u64 total = sh.total;
  const double want = (double)a.u[b] * (double)total;
  u64 target = want > 0 ? (want < (double)total ? (u64)want : total - 1) : 0;      // the first running sum above it
  target = min(target, total - 1);
  u64 at = mass - own_mass;
  ties = first_ties;
  for (int i = 0; i < PER; ++i) {
    const int c = threadIdx.x * PER + i;
    if (c >= chunks) break;
    const u64 m = kept_mass(c, ties);
    if (at <= target && target < at + m) { sh.found = c; sh.before_mass = at; sh.before_count = ties; }
    at += m; ties += sh.count[c];
  }
  __syncthreads();
  if (w != 0) return;
  const int c = sh.found;
  float x[8];
  row.load(c, l, x);
  unsigned lane_ties = 0;
  for (int i = 0; i < 8; ++i) lane_ties += key_of(x[i]) == limit.key;
  unsigned seen = sh.before_count + (unsigned)wave_scan(lane_ties, l) - lane_ties;
  u64 e[8], sum = 0;
  for (int i = 0; i < 8; ++i) {
    const unsigned key = key_of(x[i]);
    e[i] = 0;
    if (key == limit.key) { if (seen++ < limit.ties) e[i] = tie_mass; }
    else if (key > limit.key) { const double y = weight(x[i]); if (!(y < min_p)) e[i] = fixed(y); }
    sum += e[i];
  }
  u64 run = sh.before_mass + wave_scan(sum, l) - sum;
  for (int i = 0; i < 8; ++i) {
    if (run <= target && target < run + e[i]) a.out[b] = (long)c * CHUNK + l * 8 + i - shift;
    run += e[i];
  }
}

}  // namespace

extern "C" int gaac_sample(int type, const void* logits, long row_stride, int B, int V, const float* u, const float* temperature_rows, float temperature, const int* top_k_rows, int top_k,
                           const float* top_p_rows, float top_p, const float* min_p_rows, float min_p, int64_t* out, void* stream) {
  GAAC_REQUIRE(logits != nullptr && u != nullptr && out != nullptr, "gaac_sample: null pointer");
  GAAC_REQUIRE(type >= 0 && type <= 2, "gaac_sample: type must be 0 (bf16), 1 (fp16) or 2 (fp32)");
  GAAC_REQUIRE(B > 0 && V > 0 && V <= MAX_V - 16 && row_stride >= 0, "gaac_sample: bad sizes (%d rows of %d logits, at most %d)", B, V, MAX_V - 16);
  GAAC_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (type == 2 ? 4 : 2) == 0, "gaac_sample: logits are not aligned to their type");
  const Args a{logits, row_stride, V, u, {temperature_rows, temperature}, {top_p_rows, top_p}, {min_p_rows, min_p}, top_k_rows, top_k, (long*)out};
  if (type == 0) k_sample<__bf16><<<B, NT, 0, (hipStream_t)stream>>>(a);
  else if (type == 1) k_sample<_Float16><<<B, NT, 0, (hipStream_t)stream>>>(a);
  else k_sample<float><<<B, NT, 0, (hipStream_t)stream>>>(a);
  return gaac::launch_status("gaac_sample");
}
