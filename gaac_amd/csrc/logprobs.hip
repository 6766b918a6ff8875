// Log probabilities of given tokens, their ranks, the entropy of the rows, and the likeliest alternatives, from logits.
//   p_i = exp(x_i - max) / S, S = sum of exp(x_i - max);  log p_i = (x_i - max) - log S;  entropy = log S - sum of exp(x_i - max) (x_i - max) / S
// One read of the logits: a block takes a segment of 8192 of a row into registers, its maximum, and with it the sums of e^d and of d e^d; segments are joined with the factors
// e^(max of one - max of all).  The order of tokens is x descending, then index ascending: as one 64-bit key, in which no two tokens are alike.  Each wave takes the
// largest x of every lane, and of these 64 the n-th largest, n an eighth of `top`: the least of the block's eight is a bound that `top` tokens at least reach and few others (alternatives lie far apart, most lanes have
// one), and these few are ranked by counting.  Where many reach it, as with tokens that are alike, the bound is one of keys: the larger of that, and of what `top` lanes of one wave reach.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "gaac_capi.h"
#include "../../include/gaac_hip.h"

namespace {

constexpr int THREADS = 512, WAVES = THREADS / 64, EACH = 16, SEGMENT = THREADS * EACH, MAX_TOP = 64, MAX_VOCAB = (1 << 20) - 16;
typedef unsigned long long u64;
typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ void load16(const __bf16* p, float* x) { const bf8 v = *reinterpret_cast<const bf8*>(p); for (int i = 0; i < 8; ++i) x[i] = (float)v[i]; }
__device__ __forceinline__ void load16(const _Float16* p, float* x) { const h8 v = *reinterpret_cast<const h8*>(p); for (int i = 0; i < 8; ++i) x[i] = (float)v[i]; }
__device__ __forceinline__ void load16(const float* p, float* x) { const f4 v = *reinterpret_cast<const f4*>(p); for (int i = 0; i < 4; ++i) x[i] = v[i]; }

// e^d for -104 <= d <= 0.  The product is rounded to 24 bits: e^d is off by |d| 2^-24 of itself, as much as by the rounding of d, a difference of 32-bit numbers.  What is far below the maximum adds little to a sum
// unless there are e^|d| of its kind, so |d| is 14 at most where it counts: 2^-20, less than a logarithm of that size is rounded by.  (The product in two parts: four more instructions a logit, 104 us instead of 97 for 777 x 128256 in fp32 with 5 alternatives.)
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * 1.44269502f); }
__device__ __forceinline__ float cleaned(float x) { return x != x ? -__builtin_inff() : x; }      // NaN: a token that never comes
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < __builtin_inff(); }
__device__ __forceinline__ float distance(float x, float top) { return x == top ? 0.f : x - top; }      // (also where both are infinite)

// The place in the order of tokens: larger is earlier.
__device__ __forceinline__ unsigned order_of(float x) {
  const unsigned b = __builtin_bit_cast(unsigned, x == 0.f ? 0.f : x);      // (-0 is 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ u64 key_of(float x, int index) { return (u64)order_of(x) << 32 | (unsigned)~index; }
__device__ __forceinline__ float value_of(u64 key) {
  const unsigned b = (unsigned)(key >> 32);
  return __builtin_bit_cast(float, b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int index_of(u64 key) { return (int)~(unsigned)key; }

// Over the wave, for all lanes, in the vector unit: rotations within 16 lanes, then halves swapped.
typedef unsigned u2 __attribute__((ext_vector_type(2)));
template <int CTRL, typename T> __device__ __forceinline__ T rotated(T x) { return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false)); }
template <typename T, typename F> __device__ __forceinline__ T over_wave(T x, F f) {
  x = f(x, rotated<0x128>(x)); x = f(x, rotated<0x124>(x)); x = f(x, rotated<0x122>(x)); x = f(x, rotated<0x121>(x));
  unsigned w = __builtin_bit_cast(unsigned, x);
  u2 p = __builtin_bit_cast(u2, __builtin_amdgcn_permlane16_swap(w, w, false, false));
  x = f(__builtin_bit_cast(T, (unsigned)p[0]), __builtin_bit_cast(T, (unsigned)p[1]));
  w = __builtin_bit_cast(unsigned, x);
  p = __builtin_bit_cast(u2, __builtin_amdgcn_permlane32_swap(w, w, false, false));
  return f(__builtin_bit_cast(T, (unsigned)p[0]), __builtin_bit_cast(T, (unsigned)p[1]));
}
__device__ __forceinline__ float wave_max(float x) { return over_wave(x, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float wave_sum(float x) { return over_wave(x, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ int wave_sum(int x) { return over_wave(x, [](int a, int b) { return a + b; }); }

// The n-th largest of the wave's 64 words, its BITS upper bits; if there are equal ones, all of them count.
template <int BITS = 32> __device__ __forceinline__ unsigned nth_of(unsigned x, int n) {
  unsigned t = 0;
  for (int b = 31; b >= 32 - BITS; --b) {
    const unsigned trial = t | 1u << b;
    if (__popcll(__ballot(x >= trial)) >= n) t = trial;
  }
  return t;
}
__device__ __forceinline__ u64 nth_of(u64 x, int n) {
  const unsigned high = (unsigned)(x >> 32), h = nth_of(high, n);
  if (__popcll(__ballot(high >= h)) == n) return (u64)h << 32;
  return (u64)h << 32 | nth_of(high == h ? (unsigned)x : 0u, n - __popcll(__ballot(high > h)));
}

struct Sums { float max, sum, weighted; int above; };      // above: tokens before the given one

struct Out { float* logprob; int64_t* rank; float* entropy; float* top_logprobs; int64_t* top_tokens; };

__device__ __forceinline__ void write_row(const Out& o, long row, int token, int V, float x, const Sums& s) {
  const float log_sum = logf(s.sum);
  const bool inside = token >= 0 && token < V, alive = s.max > -__builtin_inff();
  o.logprob[row] = inside && alive ? distance(x, s.max) - log_sum : __builtin_nanf("");
  o.rank[row] = inside ? s.above : -1;
  o.entropy[row] = alive ? log_sum - s.weighted / s.sum : __builtin_nanf("");
}
__device__ __forceinline__ void write_top(const Out& o, long at, u64 key, const Sums& s) {
  o.top_logprobs[at] = s.max > -__builtin_inff() ? distance(value_of(key), s.max) - logf(s.sum) : __builtin_nanf("");
  o.top_tokens[at] = index_of(key);
}

// Places of c keys in their order, by counting: wave w compares with every WIDTH-th.  places: zeros.
template <int WIDTH> __device__ __forceinline__ void count_places(const u64* keys, int c, int* places) {
  const int l = threadIdx.x & 63;
  for (int i = l; i < c; i += 64) {
    const u64 k = keys[i];
    int before = 0, j = threadIdx.x >> 6;
    for (; j + 7 * WIDTH < c; j += 8 * WIDTH) {      // eight reads on their way
#pragma unroll
      for (int n = 0; n < 8; ++n) before += keys[j + n * WIDTH] > k;
    }
    for (; j < c; j += WIDTH) before += keys[j] > k;
    if (WIDTH == 1) places[i] = before; else if (before > 0) atomicAdd(&places[i], before);
  }
}

constexpr int most_ranked(int top) { return 2 * top + 64; }
constexpr int most_found(int top) { return WAVES * EACH * top; }      // keys at or above a bound of keys: no wave has more than `top` lanes there, each with its EACH tokens

// Work memory of a row and segment: its sums, and behind those of all rows its `top` best keys.  What bounds it is the blocks' way from load to store, four
// blocks a CU at once: instructions and waits (without alternatives 777 x 128256 take 73 us in fp32, 65 in bf16; with 5 97 and 91).  What is the same for a wave is counted by the scalar unit (ballots), and the given token's
// logit is waited for behind the maximum.  Blocks that take several segments and read the next one ahead need 83 registers, three blocks a CU: 148 instead of 97.
template <typename T>
__global__ __launch_bounds__(THREADS) void k_logprobs(const T* logits, long row_stride, int V, const int64_t* tokens, int top, int segments, Sums* sums, u64* best, Out out) {
  constexpr int PER = 16 / sizeof(T), RUNS = EACH / PER;
  __shared__ float red[3][WAVES];
  __shared__ int above_of[WAVES];
  __shared__ unsigned value_of_wave[WAVES];
  __shared__ u64 key_of_wave[2 * WAVES];
  __shared__ int count;
  extern __shared__ u64 found[];      // most_found keys, then as many places
  int* places = reinterpret_cast<int*>(found + most_found(top));
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, segment = blockIdx.x % segments, first = segment * SEGMENT, n = min(V - first, SEGMENT);
  const long row = blockIdx.x / segments;
  const T* src = logits + row * row_stride + first;
  const bool aligned = reinterpret_cast<uintptr_t>(src) % 16 == 0;
  const int slot = n < SEGMENT ? l * WAVES + wave : (int)threadIdx.x;      // (a short segment is spread over all waves: the bound below goes by the one that has the least)
  if (threadIdx.x == 0) count = 0;
  const long given = tokens[row];
  const int token = given >= 0 && given < V ? (int)given : -1;
  float x[EACH];
  if (aligned && n == SEGMENT) {
#pragma unroll
    for (int r = 0; r < RUNS; ++r) load16(src + (r * THREADS + threadIdx.x) * PER, x + r * PER);
  } else {
#pragma unroll
    for (int r = 0; r < RUNS; ++r) {
      const int at = (r * THREADS + slot) * PER;
      if (aligned && at + PER <= n) load16(src + at, x + r * PER);
      else {
#pragma unroll
        for (int i = 0; i < PER; ++i) x[r * PER + i] = at + i < n ? (float)src[at + i] : -__builtin_inff();
      }
    }
  }
  const T at_token = logits[row * row_stride + max(token, 0)];      // (read last, and waited for only after the maximum)
  const auto index = [&](int i) { return (i / PER * THREADS + slot) * PER + i % PER; };
  float m = -__builtin_inff();
  bool odd = false;      // a NaN among them
#pragma unroll
  for (int i = 0; i < EACH; i += 2) odd |= __builtin_isunordered(x[i], x[i + 1]);
  if (__any(odd)) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) x[i] = cleaned(x[i]);
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) m = fmaxf(m, x[i]);
  const float best_of_wave = wave_max(m);
  const int share = (top + WAVES - 1) / WAVES;
  if (top > 0) {
    const unsigned bound = share == 1 ? order_of(best_of_wave) : nth_of<16>(order_of(m), share);
    if (l == 0) value_of_wave[wave] = bound;
  }
  m = best_of_wave;
  if (l == 0) red[0][wave] = m;
  __syncthreads();
  for (int i = 0; i < WAVES; ++i) m = fmaxf(m, red[0][i]);
  float sum = 0, weighted = 0;
  int above = 0;
  if (finite(m)) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {      // (what is masked: e^-104 is 0)
      const float d = fmaxf(x[i] - m, -104.f), e = exp_of(d);
      sum += e;
      weighted = __builtin_fmaf(e, d, weighted);
    }
  } else if (m > 0.f) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) sum += x[i] == m ? 1.f : 0.f;
  }
  const float mine = token >= 0 ? cleaned((float)at_token) : 0.f;
  const auto below = [](float v) { return v == 0.f ? -1.40129846e-45f : __builtin_bit_cast(float, __builtin_bit_cast(int, v) + (v > 0.f ? -1 : 1)); };      // the next one below
  if (finite(mine) && (token < first || token >= first + SEGMENT)) {      // before the token whatever is not smaller, behind it what is larger; what is behind the row's end is -inf
    const float limit = token < first ? mine : below(mine);
#pragma unroll
    for (int i = 0; i < EACH; ++i) above += __popcll(__ballot(x[i] > limit));
  } else {
#pragma unroll
    for (int i = 0; i < EACH; ++i) above += __popcll(__ballot(index(i) < n && (x[i] > mine || (x[i] == mine && first + index(i) < token))));
  }
  sum = wave_sum(sum); weighted = wave_sum(weighted);
  if (l == 0) { red[1][wave] = sum; red[2][wave] = weighted; above_of[wave] = above; }
  u64 bound = 0;
  if (top > 0) {
    unsigned b = value_of_wave[0];
    for (int i = 1; i < WAVES; ++i) b = min(b, value_of_wave[i]);
    bound = (u64)max(b, order_of(-__builtin_inff())) << 32;      // (with its upper bits only it may lie below -inf, where no number is)
    const float limit = value_of(bound);
    int reach = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) reach += __popcll(__ballot(x[i] >= limit));
    if (l == 0 && reach > 0) atomicAdd(&count, reach);
  }
  __syncthreads();
  Sums s{m, 0.f, 0.f, 0};
  for (int i = 0; i < WAVES; ++i) { s.sum += red[1][i]; s.weighted += red[2][i]; s.above += above_of[i]; }
  if (threadIdx.x == 0) {
    if (segments == 1) write_row(out, row, token, V, mine, s); else sums[(long)row * segments + segment] = s;
  }
  if (top == 0) return;
  const int reached = count;
  __syncthreads();
  if (threadIdx.x == 0) count = 0;
  if (reached > 4 * top + 128 || reached > most_found(top)) {      // many alike
    u64 b = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const u64 k = index(i) < n ? key_of(x[i], first + index(i)) : 0;
      b = k > b ? k : b;
    }
    const u64 all = nth_of(b, top), part = nth_of(b, share);
    if (l == 0) { key_of_wave[wave] = all; key_of_wave[WAVES + wave] = part; }
    __syncthreads();
    bound = key_of_wave[WAVES];
    for (int i = 1; i < WAVES; ++i) bound = min(bound, key_of_wave[WAVES + i]);
    for (int i = 0; i < WAVES; ++i) bound = max(bound, key_of_wave[i]);
  }
  __syncthreads();
  const float limit = bound == 0 ? -__builtin_inff() : value_of(bound);      // (0: fewer than `top` lanes have a token)
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (x[i] >= limit && index(i) < n) {
      const u64 k = key_of(x[i], first + index(i));
      if (k >= bound) {
        const int at = atomicAdd(&count, 1);
        found[at] = k; places[at] = 0;
      }
    }
  __syncthreads();
  const int c = count;
  count_places<WAVES>(found, c, places);
  __syncthreads();
  u64* mine_best = best + ((long)row * segments + segment) * top;
  for (int i = threadIdx.x; i < c; i += THREADS) {
    const int before = places[i];
    if (before < top) {
      if (segments == 1) write_top(out, row * top + before, found[i], s); else mine_best[before] = found[i];
    }
  }
  if (segments > 1) for (int i = c + threadIdx.x; i < top; i += THREADS) mine_best[i] = 0;      // a last segment with fewer tokens
}

// A bound that at least n and at most `most` of c different keys in LDS reach (or all that are not 0, where they are fewer), by a wave: bit by bit the largest that n reach, until they are few enough.
__device__ __forceinline__ u64 key_bound(const u64* keys, int c, int n, int most) {
  u64 t = 0;
  for (int b = 63; b >= 0; --b) {
    const u64 trial = t | 1ull << b;
    int reach = 0;
#pragma unroll 4
    for (int i = threadIdx.x & 63; i < c; i += 64) reach += keys[i] >= trial;
    reach = wave_sum(reach);
    if (reach >= n) t = trial;
    if (reach >= n && reach <= most) break;
  }
  return t;
}

// Joins a row's segments, a wave a row.  Every segment's list is sorted: the least of their n-th keys, n = top / segments rounded up, is a bound that `top` keys at least reach.  Those that do are ranked by
// counting; where they are many more (a short last segment, or likely tokens in one place), those that reach the `top`-th of the lanes' best keys, and where these are too many as well, a bound found bit by bit.
template <typename T>
__global__ __launch_bounds__(64) void k_logprobs_merge(const T* logits, long row_stride, int V, const int64_t* tokens, int top, int segments, const Sums* sums, const u64* best, Out out) {
  extern __shared__ u64 keys[];      // of all segments, then those that are ranked, then their places
  const long row = blockIdx.x;
  const int l = threadIdx.x, c = segments * top, most = most_ranked(top);
  const Sums* mine = sums + row * segments;
  const long given = tokens[row];
  const int token = given >= 0 && given < V ? (int)given : -1;
#pragma unroll 4
  for (int i = l; i < c; i += 64) keys[i] = best[row * c + i];
  const Sums none{-__builtin_inff(), 0.f, 0.f, 0}, t0 = l < segments ? mine[l] : none, t1 = l + 64 < segments ? mine[l + 64] : none;      // (up to 128 segments)
  const float x = token >= 0 ? cleaned((float)logits[row * row_stride + token]) : 0.f;
  Sums s{wave_max(fmaxf(t0.max, t1.max)), 0.f, 0.f, t0.above + t1.above};
  const auto add = [&](const Sums& t) {
    const float d = fmaxf(distance(t.max, s.max), -104.f), e = exp_of(d);
    if (t.max > -__builtin_inff()) { s.sum += e * t.sum; s.weighted += e * __builtin_fmaf(d, t.sum, t.weighted); }
  };
  add(t0); add(t1);
  s.sum = wave_sum(s.sum); s.weighted = wave_sum(s.weighted); s.above = wave_sum(s.above);
  if (l == 0) write_row(out, row, token, V, x, s);
  if (top == 0) return;
  __syncthreads();
  u64* found = keys + c;
  int* places = reinterpret_cast<int*>(found + most);
  const int nth = (top + segments - 1) / segments - 1;
  u64 bound = min(l < segments ? keys[l * top + nth] : ~0ull, l + 64 < segments ? keys[(l + 64) * top + nth] : ~0ull);
  for (int o = 32; o > 0; o >>= 1) bound = min(bound, (u64)__shfl_xor(bound, o));
  const auto too_many = [&] {
    int reached = 0;
#pragma unroll 4
    for (int i = l; i < c; i += 64) reached += keys[i] >= bound;
    return wave_sum(reached) > most;
  };
  if (too_many()) {
    u64 b = 0;
#pragma unroll 4
    for (int i = l; i < c; i += 64) b = max(b, keys[i]);
    bound = max(bound, nth_of(b, top));
    if (too_many()) bound = key_bound(keys, c, top, most);
  }
  int held = 0;
  for (int i0 = 0; i0 < c; i0 += 64) {
    const u64 k = i0 + l < c ? keys[i0 + l] : 0;
    const u64 here = __ballot(k != 0 && k >= bound);
    if (k != 0 && k >= bound) found[held + __popcll(here & ((1ull << l) - 1))] = k;
    held += __popcll(here);
  }
  __syncthreads();
  count_places<1>(found, held, places);
  for (int i = l; i < held; i += 64)
    if (places[i] < top) write_top(out, row * top + places[i], found[i], s);
}

template <typename T> void launch(const void* logits, long row_stride, int B, int V, const int64_t* tokens, int top, void* work, const Out& out, hipStream_t stream) {
  const int segments = (V + SEGMENT - 1) / SEGMENT;
  Sums* sums = static_cast<Sums*>(work);
  u64* best = reinterpret_cast<u64*>(sums + (long)B * segments);
  k_logprobs<T><<<(unsigned)B * segments, THREADS, 12 * most_found(top), stream>>>(static_cast<const T*>(logits), row_stride, V, tokens, top, segments, sums, best, out);
  if (segments > 1) k_logprobs_merge<T><<<B, 64, 8 * segments * top + 12 * most_ranked(top), stream>>>(static_cast<const T*>(logits), row_stride, V, tokens, top, segments, sums, best, out);
}

}  // namespace

extern "C" int gaac_logprobs(int type, const void* logits, long row_stride, int B, int V, const int64_t* tokens, int top, void* work, long work_bytes, float* logprob, int64_t* rank, float* entropy,
                             float* top_logprobs, int64_t* top_tokens, void* stream) {
  GAAC_REQUIRE(logits != nullptr && tokens != nullptr && logprob != nullptr && rank != nullptr && entropy != nullptr, "gaac_logprobs: null pointer");
  GAAC_REQUIRE(type >= 0 && type <= 2, "gaac_logprobs: type must be 0 (bf16), 1 (fp16) or 2 (fp32)");
  GAAC_REQUIRE(B > 0 && V > 0 && V <= MAX_VOCAB && (long)B * ((V + SEGMENT - 1) / SEGMENT) <= 1 << 22, "gaac_logprobs: bad sizes (%d rows of %d logits, up to 2^22 segments of %d and rows of %d)", B, V, SEGMENT, MAX_VOCAB);
  GAAC_REQUIRE(top >= 0 && top <= MAX_TOP && top <= V && (top == 0 || (top_logprobs != nullptr && top_tokens != nullptr)), "gaac_logprobs: up to %d alternatives, no more than there are logits (%d of %d)", MAX_TOP, top, V);
  const long segments = (V + SEGMENT - 1) / SEGMENT, need = segments == 1 ? 0 : B * segments * (16 + 8l * top);
  GAAC_REQUIRE(need == 0 || (work != nullptr && reinterpret_cast<uintptr_t>(work) % 16 == 0 && work_bytes >= need), "gaac_logprobs: needs %ld bytes of work memory, 16-byte aligned", need);
  GAAC_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (type == 2 ? 4 : 2) == 0, "gaac_logprobs: logits are not aligned");
  const Out out{logprob, rank, entropy, top_logprobs, top_tokens};
  if (type == 0) launch<__bf16>(logits, row_stride, B, V, tokens, top, work, out, (hipStream_t)stream);
  else if (type == 1) launch<_Float16>(logits, row_stride, B, V, tokens, top, work, out, (hipStream_t)stream);
  else launch<float>(logits, row_stride, B, V, tokens, top, work, out, (hipStream_t)stream);
  return gaac::launch_status("gaac_logprobs");
}
