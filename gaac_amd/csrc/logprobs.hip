// Log probabilities of given tokens, their ranks, the entropy of the rows, and the likeliest alternatives, from logits.
//   p_i = exp(x_i - max) / S, S = sum of exp(x_i - max);  log p_i = (x_i - max) - log S;  entropy = log S - sum of exp(x_i - max) (x_i - max) / S
// One read of the logits: a block takes a segment of 8192 of a row into registers, its maximum, and with it the sums of e^d and of d e^d; segments are joined with the factors
// e^(max of one - max of all).  The order of tokens is x descending, then index ascending: as one 64-bit key, in which no two tokens are alike.  Each wave takes the
// best key of every lane; the `top`-th best of these 64 is a bound that `top` tokens at least reach, the largest bound of the block's waves leaves little more than that
// (alternatives lie far apart, most lanes have one), and these few are ranked by counting.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "gaac_capi.h"
#include "../../include/gaac_hip.h"

namespace {

constexpr int THREADS = 512, WAVES = THREADS / 64, EACH = 16, SEGMENT = THREADS * EACH, MAX_TOP = 64, MAX_VOCAB = (1 << 20) - 16, MERGE = 256;
typedef unsigned long long u64;
typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ void load16(const __bf16* p, float* x) { const bf8 v = *reinterpret_cast<const bf8*>(p); for (int i = 0; i < 8; ++i) x[i] = (float)v[i]; }
__device__ __forceinline__ void load16(const _Float16* p, float* x) { const h8 v = *reinterpret_cast<const h8*>(p); for (int i = 0; i < 8; ++i) x[i] = (float)v[i]; }
__device__ __forceinline__ void load16(const float* p, float* x) { const f4 v = *reinterpret_cast<const f4*>(p); for (int i = 0; i < 4; ++i) x[i] = v[i]; }

// e^d for d <= 0: the product with log2(e) in two parts, the second by the first two terms of its series (off by 2^-23 of itself, where one part alone would lose d's last bits).
__device__ __forceinline__ float exp_of(float d) {
  const float t = d * 1.44269502f, r = __builtin_fmaf(d, 1.44269502f, -t) + d * 1.92596303e-8f;
  const float e = __builtin_amdgcn_exp2f(t);
  return d > -104.f ? __builtin_fmaf(e, r * 0.693147181f, e) : 0.f;
}
__device__ __forceinline__ float cleaned(float x) { return x != x ? -__builtin_inff() : x; }      // NaN: a token that never comes
__device__ __forceinline__ float distance(float x, float top) { return x == top ? 0.f : x - top; }      // (also where both are infinite)

// The place in the order of tokens: larger is earlier.
__device__ __forceinline__ u64 key_of(float x, int index) {
  const unsigned b = __builtin_bit_cast(unsigned, x == 0.f ? 0.f : x);      // (-0 is 0)
  return (u64)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (unsigned)~index;
}
__device__ __forceinline__ float value_of(u64 key) {
  const unsigned b = (unsigned)(key >> 32);
  return __builtin_bit_cast(float, b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int index_of(u64 key) { return (int)~(unsigned)key; }

__device__ __forceinline__ float wave_max(float x) { for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o)); return x; }
__device__ __forceinline__ float wave_sum(float x) { for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o); return x; }
__device__ __forceinline__ int wave_sum(int x) { for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o); return x; }

// The n-th largest of the wave's 64 words; if there are equal ones, all of them count.
__device__ __forceinline__ unsigned nth_of(unsigned x, int n) {
  unsigned t = 0;
  for (int b = 31; b >= 0; --b) {
    const unsigned trial = t | 1u << b;
    if (__popcll(__ballot(x >= trial)) >= n) t = trial;
  }
  return t;
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

// Work memory of a row and segment: its sums, and behind those of all rows its `top` best keys.
template <typename T>
__global__ __launch_bounds__(THREADS) void k_logprobs(const T* logits, long row_stride, int V, const int64_t* tokens, int top, int segments, Sums* sums, u64* best, Out out) {
  constexpr int PER = 16 / sizeof(T), RUNS = EACH / PER;
  __shared__ float red[3][WAVES];
  __shared__ int above_of[WAVES];
  __shared__ u64 bound_of[WAVES];
  extern __shared__ u64 found[];      // a wave has `top` lanes at most at or above its bound, each with its EACH tokens
  __shared__ int count;
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, segment = blockIdx.x % segments, first = segment * SEGMENT, n = min(V - first, SEGMENT);
  const long row = blockIdx.x / segments;
  const T* src = logits + row * row_stride + first;
  const bool aligned = reinterpret_cast<uintptr_t>(src) % 16 == 0;
  if (threadIdx.x == 0) count = 0;
  float x[EACH];
#pragma unroll
  for (int r = 0; r < RUNS; ++r) {
    const int at = (r * THREADS + threadIdx.x) * PER;
    if (aligned && at + PER <= n) load16(src + at, x + r * PER);
    else {
#pragma unroll
      for (int i = 0; i < PER; ++i) x[r * PER + i] = at + i < n ? (float)src[at + i] : -__builtin_inff();
    }
  }
  const long given = tokens[row];
  const int token = given >= 0 && given < V ? (int)given : -1;
  const float mine = token >= 0 ? cleaned((float)logits[row * row_stride + token]) : 0.f;
  float m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < EACH; ++i) { x[i] = cleaned(x[i]); m = fmaxf(m, x[i]); }
  const auto index = [&](int i) { return (int)((i / PER * THREADS + threadIdx.x) * PER + i % PER); };
  m = wave_max(m);
  if (l == 0) red[0][wave] = m;
  __syncthreads();
  for (int i = 0; i < WAVES; ++i) m = fmaxf(m, red[0][i]);
  float sum = 0, weighted = 0;
  int above = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const float d = distance(x[i], m), e = exp_of(d);
    const bool alive = x[i] > -__builtin_inff();
    sum += alive ? e : 0.f;
    weighted += alive && e > 0.f ? e * d : 0.f;
    const int at = first + index(i);
    above += at < V && (x[i] > mine || (x[i] == mine && at < token));
  }
  sum = wave_sum(sum); weighted = wave_sum(weighted); above = wave_sum(above);
  u64 bound = 0;
  if (top > 0) {
    u64 b = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const u64 k = index(i) < n ? key_of(x[i], first + index(i)) : 0;
      b = k > b ? k : b;
    }
    const unsigned high = nth_of((unsigned)(b >> 32), top);
    const int before = __popcll(__ballot((unsigned)(b >> 32) > high));
    const unsigned low = nth_of((unsigned)(b >> 32) == high ? (unsigned)b : 0u, top - before);
    bound = (u64)high << 32 | low;
  }
  if (l == 0) { red[1][wave] = sum; red[2][wave] = weighted; above_of[wave] = above; bound_of[wave] = bound; }
  __syncthreads();
  Sums s{m, 0.f, 0.f, 0};
  for (int i = 0; i < WAVES; ++i) { s.sum += red[1][i]; s.weighted += red[2][i]; s.above += above_of[i]; bound = bound_of[i] > bound ? bound_of[i] : bound; }
  if (threadIdx.x == 0) {
    if (segments == 1) write_row(out, row, token, V, mine, s); else sums[(long)row * segments + segment] = s;
  }
  if (top == 0) return;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const u64 k = index(i) < n ? key_of(x[i], first + index(i)) : 0;
    if (k != 0 && k >= bound) found[atomicAdd(&count, 1)] = k;
  }
  __syncthreads();
  const int c = count;
  u64* mine_best = best + ((long)row * segments + segment) * top;
  for (int i = threadIdx.x; i < c; i += THREADS) {
    const u64 k = found[i];
    int before = 0;
    for (int j = 0; j < c; ++j) before += found[j] > k;
    if (before < top) {
      if (segments == 1) write_top(out, row * top + before, k, s); else mine_best[before] = k;
    }
  }
  if (segments > 1) for (int i = c + threadIdx.x; i < top; i += THREADS) mine_best[i] = 0;      // a last segment with fewer tokens
}

// Joins a row's segments.  Candidates are ranked by counting, behind a bound that leaves `top` of them at least.
template <typename T>
__global__ __launch_bounds__(MERGE) void k_logprobs_merge(const T* logits, long row_stride, int V, const int64_t* tokens, int top, int segments, const Sums* sums, const u64* best, Out out) {
  extern __shared__ u64 found[];
  const long row = blockIdx.x;
  const Sums* mine = sums + row * segments;
  const long given = tokens[row];
  const int token = given >= 0 && given < V ? (int)given : -1;
  Sums s{-__builtin_inff(), 0.f, 0.f, 0};
  for (int i = 0; i < segments; ++i) s.max = fmaxf(s.max, mine[i].max);
  for (int i = 0; i < segments; ++i) {
    const Sums t = mine[i];
    const float d = distance(t.max, s.max), e = t.max > -__builtin_inff() ? exp_of(d) : 0.f;
    if (e > 0.f) { s.sum += e * t.sum; s.weighted += e * __builtin_fmaf(d, t.sum, t.weighted); }
    s.above += t.above;
  }
  if (threadIdx.x == 0) write_row(out, row, token, V, token >= 0 ? cleaned((float)logits[row * row_stride + token]) : 0.f, s);
  if (top == 0) return;
  const int c = segments * top;
  for (int i = threadIdx.x; i < c; i += MERGE) found[i] = best[row * c + i];
  __syncthreads();
  for (int i = threadIdx.x; i < c; i += MERGE) {
    const u64 k = found[i];
    if (k == 0) continue;
    int before = 0;
    for (int j = 0; j < c; ++j) before += found[j] > k;
    if (before < top) write_top(out, row * top + before, k, s);
  }
}

template <typename T> void launch(const void* logits, long row_stride, int B, int V, const int64_t* tokens, int top, void* work, const Out& out, hipStream_t stream) {
  const int segments = (V + SEGMENT - 1) / SEGMENT;
  Sums* sums = static_cast<Sums*>(work);
  u64* best = reinterpret_cast<u64*>(sums + (long)B * segments);
  k_logprobs<T><<<(unsigned)B * segments, THREADS, sizeof(u64) * WAVES * EACH * top, stream>>>(static_cast<const T*>(logits), row_stride, V, tokens, top, segments, sums, best, out);
  if (segments > 1) k_logprobs_merge<T><<<B, MERGE, sizeof(u64) * segments * top, stream>>>(static_cast<const T*>(logits), row_stride, V, tokens, top, segments, sums, best, out);
}

}  // namespace

extern "C" int gaac_logprobs(int type, const void* logits, long row_stride, int B, int V, const int64_t* tokens, int top, void* work, long work_bytes, float* logprob, int64_t* rank, float* entropy,
                             float* top_logprobs, int64_t* top_tokens, void* stream) {
  GAAC_REQUIRE(logits != nullptr && tokens != nullptr && logprob != nullptr && rank != nullptr && entropy != nullptr, "gaac_logprobs: null pointer");
  GAAC_REQUIRE(type >= 0 && type <= 2, "gaac_logprobs: type must be 0 (bf16), 1 (fp16) or 2 (fp32)");
  GAAC_REQUIRE(B > 0 && B <= 1 << 23 && V > 0 && V <= MAX_VOCAB, "gaac_logprobs: bad sizes (%d rows of %d logits, up to 2^23 of %d)", B, V, MAX_VOCAB);
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
