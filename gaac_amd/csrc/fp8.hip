// Rows in 8 bits: their quantiser (with the residual's addition and the root-mean-square norm before it), the way back, and products of such rows with such weights.
//
// Format: 128 consecutive elements of a row are a block.  A block has one power of two 2^E, E the smallest integer with amax <= 448 * 2^E, from -117 to 119, held as the
// byte E + 127 (255: the block held a NaN or an infinity and reads as NaN), and e4m3 codes: the nearest to x * 2^-E, ties to the even code.  Scaling is by a power of two, so
// only that rounding is made, and every value is a normal number of bf16 (2^-126 to 448 * 2^119) or zero.  Elements behind the row's end are zero codes.
//
// 16 rows by one block are a tile, 2048 bytes in the order of the operands of the scaled 16x16x128 product, a lane's 16 bytes next to each other: row m, element
// 32 g + 16 j + i of the block at byte 1024 j + 16 (16 g + m) + i.  (Which elements of a block a lane group has is free, as long as both operands agree: they share one power of
// two.)  The tiles of a block of K lie in a row, those of the next block
// behind them: blocks of threads that go along K together read memory in one piece.  The exponent bytes of four blocks are a dword, byte s that of block 4 q + s, dword [q][row]: the
// instruction picks the byte, so a dword serves four products.  Weights of a gated pair alternate: tile 2 t holds 16 rows of the gate, tile 2 t + 1 the same rows of the other.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "gaac_capi.h"
#include "../../include/gaac_hip.h"

namespace {

constexpr int BLOCK = 128, TILE = 2048, MAX_K = 65536, MAX_NORM_K = 32768;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i8 __attribute__((ext_vector_type(8)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float bits(unsigned x) { return __builtin_bit_cast(float, x); }
__device__ __forceinline__ unsigned word(float x) { return __builtin_bit_cast(unsigned, x); }

__device__ __forceinline__ void load8(const __bf16* p, float (&x)[8]) { const bf8 v = *reinterpret_cast<const bf8*>(p); for (int i = 0; i < 8; ++i) x[i] = (float)v[i]; }
__device__ __forceinline__ void load8(const _Float16* p, float (&x)[8]) { const h8 v = *reinterpret_cast<const h8*>(p); for (int i = 0; i < 8; ++i) x[i] = (float)v[i]; }
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const f4 a = *reinterpret_cast<const f4*>(p), b = *reinterpret_cast<const f4*>(p + 4);
  for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
}
__device__ __forceinline__ void store8(__bf16* p, const float (&x)[8]) { bf8 v; for (int i = 0; i < 8; ++i) v[i] = (__bf16)x[i]; *reinterpret_cast<bf8*>(p) = v; }
__device__ __forceinline__ void store8(_Float16* p, const float (&x)[8]) { h8 v; for (int i = 0; i < 8; ++i) v[i] = (_Float16)x[i]; *reinterpret_cast<h8*>(p) = v; }
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<f4*>(p) = f4{x[0], x[1], x[2], x[3]};
  *reinterpret_cast<f4*>(p + 4) = f4{x[4], x[5], x[6], x[7]};
}
// The first n of 8 elements, zeros for the others; whole: all of them, from an aligned address.
template <typename T> __device__ __forceinline__ void load_some(const T* p, int n, bool whole, float (&x)[8]) {
  if (whole && n >= 8) return load8(p, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = i < n ? (float)p[i] : 0.f;
}
template <typename T> __device__ __forceinline__ void store_some(T* p, int n, bool whole, const float (&x)[8]) {
  if (whole && n >= 8) return store8(p, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) if (i < n) p[i] = (T)x[i];
}

// Largest magnitude as the bits of a float (those of a NaN above all others).
__device__ __forceinline__ unsigned magnitude8(const float (&x)[8]) {
  unsigned a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, word(x[i]) & 0x7fffffffu);
  return a;
}
// amax = m 2^e <= 448 * 2^E = 1.75 * 2^(E+8): one more where the mantissa is above 1.75.
__device__ __forceinline__ unsigned exponent_byte(unsigned a) { return a >= 0x7f800000u ? 255u : (unsigned)min(max((int)((a + 0x1fffffu) >> 23) - 8, 10), 246); }
__device__ __forceinline__ float inverse_scale(unsigned e) { return bits((254u - min(e, 246u)) << 23); }
__device__ __forceinline__ unsigned encode4(float a, float b, float c, float d) {
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}
// 8 codes; in a block that reads as NaN all of them are NaN.  Only blocks of the largest exponent can have elements beyond 448.
__device__ __forceinline__ u2 encode8(const float (&x)[8], unsigned e) {
  const float s = inverse_scale(e);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = x[i] * s;
  if (e >= 246u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = fminf(fmaxf(y[i], -448.f), 448.f);
  }
  const u2 w = {encode4(y[0], y[1], y[2], y[3]), encode4(y[4], y[5], y[6], y[7])};
  return e == 255u ? u2{0x7f7f7f7fu, 0x7f7f7f7fu} : w;
}
// Maximum over 16 lanes next to each other, in the vector unit.
template <int CTRL> __device__ __forceinline__ unsigned rotated(unsigned x) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false); }
__device__ __forceinline__ unsigned max16(unsigned x) {
  x = max(x, rotated<0x128>(x)); x = max(x, rotated<0x124>(x)); x = max(x, rotated<0x122>(x)); x = max(x, rotated<0x121>(x));      // row_ror 8, 4, 2, 1
  return x;
}
// Sum over the wave, for all lanes, in the vector unit: rotations within 16 lanes, then halves swapped.
template <int CTRL> __device__ __forceinline__ double rotated_sum(double x) {
  const u2 v = __builtin_bit_cast(u2, x);
  return x + __builtin_bit_cast(double, u2{rotated<CTRL>(v[0]), rotated<CTRL>(v[1])});
}
__device__ __forceinline__ double wave_sum(double x) {
  x = rotated_sum<0x128>(x); x = rotated_sum<0x124>(x); x = rotated_sum<0x122>(x); x = rotated_sum<0x121>(x);
  u2 v = __builtin_bit_cast(u2, x);
  u2 p = __builtin_bit_cast(u2, __builtin_amdgcn_permlane16_swap(v[0], v[0], false, false)), q = __builtin_bit_cast(u2, __builtin_amdgcn_permlane16_swap(v[1], v[1], false, false));
  x = __builtin_bit_cast(double, u2{p[0], q[0]}) + __builtin_bit_cast(double, u2{p[1], q[1]});
  v = __builtin_bit_cast(u2, x);
  p = __builtin_bit_cast(u2, __builtin_amdgcn_permlane32_swap(v[0], v[0], false, false)); q = __builtin_bit_cast(u2, __builtin_amdgcn_permlane32_swap(v[1], v[1], false, false));
  return __builtin_bit_cast(double, u2{p[0], q[0]}) + __builtin_bit_cast(double, u2{p[1], q[1]});
}

// y in 32 bits, rounded to an odd last bit where bits are lost: rounding once more, to 8 bits, then gives what rounding y itself would.  It matters only where the nearest number of 32 bits is a border between
// two codes, which has 19 zeros at its end.  The neighbour is taken by magnitude: what is rounded to 0 becomes the smallest number of y's sign, what is finite and rounded to infinity the largest.
__device__ __forceinline__ float to_odd(double y) {
  const float f = (float)y;
  const double d = fabs(y) - fabs((double)f);      // (NaN where y is infinite or NaN)
  const unsigned u = word(f);
  return !(d < 0.0 || d > 0.0) || (u & 1u) ? f : bits(d > 0.0 ? u + 1 : u - 1);
}

// ---------------------------------------------------------------------------------------------------- rows into 8 bits
struct RowsArgs {
  const void *x, *residual, *weight;
  void* sum;
  uint8_t *data, *exps;
  long x_rs, r_rs, pad;
  int K, nb, waves, tile_step, tile_first, first;
  float eps;
  bool whole;
};

// A block a row (for few rows without the norm: a part of a row), of `waves` waves; a lane takes CH runs of 8 elements, 16 lanes a block of 128.  Bound by HBM: 16384 x 4096 in bf16 52 us (201 MB, 3.9 TB/s; a large copy makes 4.7 to 5.2), with norm and residual 113 (470 MB,
// 4.2 TB/s); by launch and latency for a few rows (4 x 4096: 2.3, 3.6).  The sum of squares and the norm in 64 bits: a result next to the border between two
// codes is rounded as the formula says, of the sum of row and residual in 32 bits and of eps as a number of 32 bits.  With a residual that costs nothing beside the memory; without one the conversions show (8192 x 4096 35 us, 28 without the norm; 8192 x 14336 152, 88).  Pairs of 32-bit numbers took
// longer (registers: 16384 x 4096 with residual 121, 118 in 64 bits then).
template <typename T, bool NORM, int CH>
__global__ __launch_bounds__(1024) void k_fp8_rows(RowsArgs a) {
  __shared__ double sums[16];
  const int l = threadIdx.x & 63, part = threadIdx.x >> 6;
  // A cache line of the result has pieces of 8 rows.  Blocks go to the XCDs in turns, each of which has its own L2: the rows of a tile are those of blocks that go to the same one (16384 x 4096: 62 us
  // with rows in the blocks' order, 52 so).
  const int turn = blockIdx.x & ~127u, in_turn = blockIdx.x & 127u, row = (turn + 128 <= (int)gridDim.x ? turn + in_turn % 8 * 16 + in_turn / 8 : (int)blockIdx.x) + a.first;
  const T* src = static_cast<const T*>(a.x) + row * a.x_rs;
  const int from = NORM ? part : (int)blockIdx.y * a.waves + part, all = NORM ? a.waves : (int)gridDim.y * a.waves;
  const auto at = [&](int i) { return 8 * ((i * all + from) * 64 + l); };
  float x[CH][8];
#pragma unroll
  for (int i = 0; i < CH; ++i) load_some(src + at(i), a.K - at(i), a.whole, x[i]);
  if constexpr (NORM) {
    if (a.residual != nullptr) {
      const T* res = static_cast<const T*>(a.residual) + row * a.r_rs;
      T* out = static_cast<T*>(a.sum) + (long)row * a.K;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        float r[8];
        load_some(res + at(i), a.K - at(i), a.whole, r);
        for (int j = 0; j < 8; ++j) x[i][j] += r[j];
        store_some(out + at(i), a.K - at(i), a.whole, x[i]);
      }
    }
    float g[CH][8];      // (on their way while the sum is made)
#pragma unroll
    for (int i = 0; i < CH; ++i) load_some(static_cast<const T*>(a.weight) + at(i), a.K - at(i), a.whole, g[i]);
    double sum = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i)
      for (int j = 0; j < 8; ++j) sum = __builtin_fma((double)x[i][j], (double)x[i][j], sum);
    sum = wave_sum(sum);
    if (a.waves > 1) {
      if (l == 0) sums[part] = sum;
      __syncthreads();
      sum = 0;
      for (int i = 0; i < a.waves; ++i) sum += sums[i];
    }
    const double r = 1.0 / __builtin_sqrt(sum / a.K + (double)a.eps);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float y[8];
      unsigned least = ~0u;
      for (int j = 0; j < 8; ++j) { y[j] = (float)((double)x[i][j] * r * (double)g[i][j]); least = min(least, word(y[j]) & 0x7ffffu); }
      if (least == 0) for (int j = 0; j < 8; ++j) y[j] = to_odd((double)x[i][j] * r * (double)g[i][j]);
      for (int j = 0; j < 8; ++j) x[i][j] = at(i) + j < a.K ? y[j] : 0.f;      // (behind the row's end 0 * r may be a NaN)
    }
  }
  const long tile_row = (long)(row >> 4) * a.tile_step + a.tile_first;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = at(i) / 8, kb = c >> 4, p = c & 15;
    if (kb >= a.nb) continue;
    const unsigned e = exponent_byte(max16(magnitude8(x[i])));
    *reinterpret_cast<u2*>(a.data + (kb * (a.pad >> 4) + tile_row) * TILE + 1024 * (p >> 1 & 1) + 16 * (16 * (p >> 2) + (row & 15)) + 8 * (p & 1)) = encode8(x[i], e);
    if (p == 0) a.exps[((kb >> 2) * a.pad + 16 * tile_row + (row & 15)) * 4 + (kb & 3)] = (uint8_t)e;
  }
}

// The way back: a block of threads a tile, 16 lanes a row's 256 bytes.  Bound by HBM: 16384 x 4096 37 us (201 MB, 5.4 TB/s).
__global__ __launch_bounds__(256) void k_fp8_values(const uint8_t* data, const uint8_t* exps, long pad, int tile_step, int tile_first, long first, int M, int K, int nb, __bf16* out, long out_rs, bool whole) {
  const int p = threadIdx.x & 15, m = threadIdx.x >> 4, kb = blockIdx.x % nb;
  const long tile = first + blockIdx.x / nb, row = 16 * tile + m, tile_row = tile * tile_step + tile_first;
  if (row >= M) return;
  const u2 w = *reinterpret_cast<const u2*>(data + (kb * (pad >> 4) + tile_row) * TILE + 1024 * (p >> 1 & 1) + 16 * (16 * (p >> 2) + m) + 8 * (p & 1));
  const unsigned e = exps[((kb >> 2) * pad + 16 * tile_row + m) * 4 + (kb & 3)];
  const float s = bits(e << 23);
  float x[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[4 * i] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 0) * s; x[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 1) * s;
    x[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 2) * s; x[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 3) * s;
  }
  if (e == 255u) for (int i = 0; i < 8; ++i) x[i] = __builtin_nanf("");
  const int k = kb * BLOCK + 8 * p;
  store_some(out + row * out_rs + k, K - k, whole, x);
}

// ---------------------------------------------------------------------------------------------------- products
struct ProductArgs {
  const void* x;
  const unsigned* x_exps;
  const uint8_t* w;
  const unsigned* w_exps;
  void* out;
  long x_pad, w_pad, out_rs;
  int M, N, K, nb, tiles;      // tiles: of 16 weight rows
  bool whole;                  // four outputs at a time
};

// One block of K of a tile of weights by one of rows, byte S of both exponent words.  The scaled product adds eight elements' products as whole multiples of 2^-13 of the largest one's power of
// two, cutting what is below, and only these sums in 32 bits (found by trying: so does the product without scales).  Against the outputs' root mean square that is an error of 1.5e-5 for Gaussian rows and weights,
// 2.6e-5 to 4.5e-5 where some channels are 16 times larger, 6e-5 with channels from 2^-8 to 2^8 (root mean square; a single output up to 1.1e-3; K from 512 to 14336); bf16's rounding is 1.7e-3, fp16's 2.1e-4.  Outputs in 32 bits would show it, and so would what is rounded twice behind a sum (a gated block's inner result, where it crosses a border): for outputs in 32 bits, and where it costs nothing,
// the codes go as bf16 (EXACT), scale included, which holds them exactly, into products that are added in 32 bits, at half the rate.
template <int S> struct Byte { static constexpr int value = S; };
template <bool EXACT> struct Operand;
template <> struct Operand<false> {
  i8 v;
  unsigned e;
  template <int S> __device__ __forceinline__ static Operand of(u4 a, u4 b, unsigned e) { return {i8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]}, e}; }
};
template <> struct Operand<true> {
  bf8 v[4];
  template <int S> __device__ __forceinline__ static Operand of(u4 a, u4 b, unsigned e) {
    const float s = bits(S == 3 ? e >> 24 << 23 : (e >> 8 * S & 255u) << 23);
    Operand o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned lo = i < 2 ? a[2 * i] : b[2 * i - 4], hi = i < 2 ? a[2 * i + 1] : b[2 * i - 3];
      const bf2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false), q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
      const bf2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false), t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
      o.v[i] = bf8{p[0], p[1], q[0], q[1], r[0], r[1], t[0], t[1]};
    }
    return o;
  }
};
template <int S> __device__ __forceinline__ f4 product(const Operand<false>& w, const Operand<false>& x, f4 c) { return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, c, 0, 0, S, (int)w.e, S, (int)x.e); }
template <int S> __device__ __forceinline__ f4 product(const Operand<true>& w, const Operand<true>& x, f4 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], x.v[i], c, 0, 0, 0);
  return c;
}
template <bool EXACT, int S> __device__ __forceinline__ Operand<EXACT> operand(const uint8_t* tile, int l, unsigned e) {
  return Operand<EXACT>::template of<S>(*reinterpret_cast<const u4*>(tile + 16 * l), *reinterpret_cast<const u4*>(tile + 1024 + 16 * l), e);
}

__device__ __forceinline__ float silu(float g) { return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504f)); }

__device__ __forceinline__ void put4(__bf16* p, f4 v) { bf4 o; for (int i = 0; i < 4; ++i) o[i] = (__bf16)v[i]; *reinterpret_cast<bf4*>(p) = o; }
__device__ __forceinline__ void put4(_Float16* p, f4 v) { h4 o; for (int i = 0; i < 4; ++i) o[i] = (_Float16)v[i]; *reinterpret_cast<h4*>(p) = o; }
__device__ __forceinline__ void put4(float* p, f4 v) { *reinterpret_cast<f4*>(p) = v; }
template <typename O> __device__ __forceinline__ void put_some(O* p, f4 v, int n, bool whole) {
  if (whole && n >= 4) return put4(p, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) if (i < n) p[i] = (O)v[i];
}

// Outputs col .. col + 3 of a row; of a gated pair from both sums.
template <typename O, bool GATED> __device__ __forceinline__ void finish(const ProductArgs& a, int row, int col, f4 v, f4 up) {
  if constexpr (GATED) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = silu(v[k]) * up[k];
  }
  if (row < a.M && col < a.N) put_some(static_cast<O*>(a.out) + row * a.out_rs + col, v, a.N - col, a.whole);
}

// Few rows: the weights go by once.  A block has NT tiles of weights and MT of rows; its eight waves share the blocks of K out, four (a dword of exponents) at a time, and their sums meet in LDS, in
// the waves' order.  A wave holds the operands of AHEAD steps in registers, each set loaded again as soon as it is used: what bounds it is how many loads are on their way
// (a CU draws 145 GB/s from its L2 at most).  4 x 6144 x 4096 4.6 us (25.4 MB, 5.5 TB/s), 4 x 28672 x 4096 gated 20.4 (118 MB, 5.8), 48 x 4096 x 14336 13.4 (59 MB, 4.4), 200 x 4096 x 4096 in fp32 13.4 to 14.6 (480 TFLOP/s).
template <typename O, int MT, int NT, int AHEAD, bool GATED>
__global__ __launch_bounds__(512, 2) void k_fp8_stream(ProductArgs a) {
  static_assert(!GATED || NT % 2 == 0, "tiles of a gated pair alternate");
  constexpr bool EXACT = sizeof(O) == 4 || MT == 1;
  constexpr int WAVES = 8;
  __shared__ f4 part[WAVES][MT * NT][64];
  const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = l & 15, g = l >> 4;
  const uint8_t *w[NT], *x[MT];
  const unsigned *we[NT], *xe[MT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {      // (a tile behind the last one is the last one again, and written by nobody)
    const long t = min((int)blockIdx.x * NT + i, a.tiles - 1);
    w[i] = a.w + t * TILE; we[i] = a.w_exps + 16 * t;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const long t = min((int)blockIdx.y * MT + i, (a.M - 1) >> 4);
    x[i] = static_cast<const uint8_t*>(a.x) + t * TILE; xe[i] = a.x_exps + 16 * t;
  }
  struct Set { u4 w[NT][2], x[MT][2]; } set[AHEAD];
  unsigned ew[NT], ex[MT], next_w[NT], next_x[MT];
  const auto load = [&](Set& s, int kb) {
    const long at = min(kb, a.nb - 1);      // (behind the last block of K the last one again, which nobody uses)
#pragma unroll
    for (int i = 0; i < NT; ++i)
      for (int h = 0; h < 2; ++h) s.w[i][h] = *reinterpret_cast<const u4*>(w[i] + at * a.w_pad * BLOCK + 1024 * h + 16 * l);
#pragma unroll
    for (int i = 0; i < MT; ++i)
      for (int h = 0; h < 2; ++h) s.x[i][h] = *reinterpret_cast<const u4*>(x[i] + at * a.x_pad * BLOCK + 1024 * h + 16 * l);
  };
  const auto load_exps = [&](int q) {
#pragma unroll
    for (int i = 0; i < NT; ++i) next_w[i] = we[i][q * a.w_pad + m];
#pragma unroll
    for (int i = 0; i < MT; ++i) next_x[i] = xe[i][q * a.x_pad + m];
  };
  const auto next_exps = [&] {
#pragma unroll
    for (int i = 0; i < NT; ++i) ew[i] = next_w[i];
#pragma unroll
    for (int i = 0; i < MT; ++i) ex[i] = next_x[i];
  };
  f4 acc[MT][NT] = {};
  const auto step = [&](auto byte) {
    constexpr int S = decltype(byte)::value;
    const Set& s = set[S % AHEAD];
    Operand<EXACT> ow[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) ow[i] = Operand<EXACT>::template of<S>(s.w[i][0], s.w[i][1], ew[i]);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const Operand<EXACT> ox = Operand<EXACT>::template of<S>(s.x[j][0], s.x[j][1], ex[j]);
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[j][i] = product<S>(ow[i], ox, acc[j][i]);
    }
  };
  const int quads = (a.nb + 3) / 4;
  int q = wave;
  if (q < quads) {
    load_exps(q);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(set[i], 4 * q + i);
    __builtin_amdgcn_sched_barrier(0);
    for (; q + WAVES < quads; q += WAVES) {
      next_exps();
      load_exps(q + WAVES);
      const auto one = [&](auto byte) {
        constexpr int S = decltype(byte)::value;
        step(byte);
        load(set[S % AHEAD], S + AHEAD < 4 ? 4 * q + S + AHEAD : 4 * (q + WAVES) + S + AHEAD - 4);
        __builtin_amdgcn_sched_barrier(0);
      };
      one(Byte<0>{}); one(Byte<1>{}); one(Byte<2>{}); one(Byte<3>{});
    }
    next_exps();
    const int n = a.nb - 4 * q;
    step(Byte<0>{});
    if constexpr (AHEAD == 2) load(set[0], 4 * q + 2);
    __builtin_amdgcn_sched_barrier(0);
    if (n > 1) step(Byte<1>{});
    if constexpr (AHEAD == 2) load(set[1], 4 * q + 3);
    __builtin_amdgcn_sched_barrier(0);
    if (n > 2) step(Byte<2>{});
    __builtin_amdgcn_sched_barrier(0);
    if (n > 3) step(Byte<3>{});
  }
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int i = 0; i < NT; ++i) part[wave][j * NT + i][l] = acc[j][i];
  __syncthreads();
  constexpr int EACH = GATED ? NT / 2 : NT;      // outputs of a tile of rows, by 16
  for (int at = wave; at < MT * EACH; at += WAVES) {
    const int j = at / EACH, i = at % EACH;
    const auto sum = [&](int t) {
      f4 s = part[0][j * NT + t][l];
      for (int k = 1; k < WAVES; ++k) s += part[k][j * NT + t][l];
      return s;
    };
    const int row = 16 * ((int)blockIdx.y * MT + j) + m, col = 16 * ((int)blockIdx.x * EACH + i) + 4 * g;
    finish<O, GATED>(a, row, col, sum(GATED ? 2 * i : i), GATED ? sum(2 * i + 1) : f4{});
  }
}

// Many rows: tiles of both operands through LDS.  A block has WN x WM waves, a wave TN tiles of weights by TM of rows; a step is one block of K, whose tiles (whole kilobytes, in the
// operands' order) go straight into LDS while steps before are computed, in two to four buffers by turns.  256 x 256, two buffers: matrix unit and LDS share the time: a step is 2048 cycles of products on each SIMD's unit
// and moves 256 KB (64 in, 192 out) at 128 bytes a cycle, as many; 8192 x 28672 x 4096 812 to 825 us (2330 to 2370 TFLOP/s; the matrix units busy for 55 % of the cycles), 8192 x 8192 x 8192 403 (2730; the library's product 338 to 386).  Smaller blocks
// have four buffers, or two where two blocks share a CU: a step waits for HBM, 0.8 us with one step on its way, 0.45 with three.  192 rows x 128 of weights, three buffers (their turns and those of the exponents' bytes meet again after
// twelve steps): where it saves a round, 777 x 6144 x 4096 28.5 us (1370 TFLOP/s, 240 blocks; 37 with 336 of 128 x 128), 1536 x 4096 x 14336 84 (104).
typedef const __attribute__((address_space(1))) void* global_ptr;
typedef __attribute__((address_space(3))) void* lds_ptr;

template <typename O, int TN, int TM, int WN, int WM, int NBUF, bool GATED>
__global__ __launch_bounds__(64 * WN * WM, TN * TM == 64 ? 1 : 2) void k_fp8_tiles(ProductArgs a, int blocks_n, int blocks_m) {
  constexpr int W = WN * WM, TILES = WN * TN + WM * TM, LOADS = 2 * TILES / W, ROWS_W = 16 * WN * TN, ROWS = 16 * TILES;
  static_assert(2 * TILES % W == 0 && ROWS_W % 64 == 0 && ROWS % 64 == 0 && TN % 2 == 0 && NBUF >= 2 && NBUF <= 4, "every wave loads as many kilobytes; a wave loads the exponents of 64 rows of one operand; tiles of a gated pair alternate");
  constexpr bool EXACT = sizeof(O) == 4;
  __shared__ __attribute__((aligned(16))) uint8_t buf0[TILES * TILE];
  __shared__ __attribute__((aligned(16))) uint8_t buf1[TILES * TILE];
  __shared__ __attribute__((aligned(16))) uint8_t buf2[NBUF > 2 ? TILES * TILE : 16];
  __shared__ __attribute__((aligned(16))) uint8_t buf3[NBUF == 4 ? TILES * TILE : 16];
  __shared__ unsigned exps[2 * ROWS];
  const auto buffer = [&](auto byte) -> uint8_t* {
    constexpr int B = decltype(byte)::value % NBUF;
    if constexpr (B == 0) return buf0; else if constexpr (B == 1) return buf1; else if constexpr (B == 2) return buf2; else return buf3;
  };
  const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % WN, wm = wave / WN, m = l & 15, g = l >> 4;
  // Blocks that follow each other go to different XCDs: each XCD has a run of the tiles, in columns of 8 blocks of rows, so that what its L2 holds is used by all of its blocks.
  const int total = blocks_n * blocks_m, xcd = blockIdx.x & 7, each = total / 8, over = total % 8;
  const int id = xcd * each + min(xcd, over) + (int)(blockIdx.x >> 3);
  const int group = id / (8 * blocks_n), in_group = id - group * 8 * blocks_n, high = min(8, blocks_m - 8 * group);
  const int bm = 8 * group + in_group % high, bn = in_group / high;
  const int last_x = (a.M - 1) >> 4;
  const int last_q = (a.nb - 1) >> 2;
  const uint8_t* src[LOADS];
  long stride[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int c = wave * LOADS + i, t = c >> 1;
    src[i] = (t < WN * TN ? a.w + (long)min(bn * WN * TN + t, a.tiles - 1) * TILE : static_cast<const uint8_t*>(a.x) + (long)min(bm * WM * TM + t - WN * TN, last_x) * TILE) + 1024 * (c & 1);
    stride[i] = (t < WN * TN ? a.w_pad : a.x_pad) * BLOCK;
  }
  // (behind the last block of K the last one again, which nobody uses: no step is different from the others)
  int next = 0;
  const auto fetch_part = [&](uint8_t* to, int from_i, int end_i) {
#pragma unroll
    for (int i = from_i; i < end_i; ++i) {
      const uint8_t* from = src[i];
      asm("" : "+s"(from));
      __builtin_amdgcn_global_load_lds((global_ptr)(from + 16u * l), (lds_ptr)(to + (wave * LOADS + i) * 1024), 16, 0, 0);
      src[i] += next < a.nb - 1 ? stride[i] : 0;
    }
  };
  const auto fetch = [&](uint8_t* to) { fetch_part(to, 0, LOADS); ++next; };
  constexpr int PARTS = (ROWS / 64 + W - 1) / W;      // runs of 64 rows whose exponents a wave loads
  const unsigned* exps_src[PARTS];
  long exps_pad[PARTS];
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const int r = 64 * (i * W + wave);
    exps_pad[i] = r < ROWS_W ? a.w_pad : a.x_pad;
    exps_src[i] = (r < ROWS_W ? a.w_exps : a.x_exps) + min((r < ROWS_W ? (long)bn * ROWS_W + r : (long)bm * (ROWS - ROWS_W) + r - ROWS_W) + l, exps_pad[i] - 1);
  }
  const auto fetch_exps = [&](int q) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i)
      if (ROWS % (64 * W) == 0 || 64 * (i * W + wave) < ROWS)
        __builtin_amdgcn_global_load_lds((global_ptr)(exps_src[i] + min(q, last_q) * exps_pad[i]), (lds_ptr)(exps + (q & 1) * ROWS + 64 * (i * W + wave)), 4, 0, 0);
  };
  // A step's first operands are read while the last products of the step before run: the last TAIL tiles of weights go through the rows one row tile at a time, and each of these is then replaced by the next step's.
  // Before that all of a buffer has been read, so the barrier stands there, once a step, and the buffer is filled again behind it.
  constexpr int TAIL = 3, RING = 4;
  static_assert(TN % RING == 0, "the slot of a step's first tile is free while the last TAIL are in use");
  struct Raw { u4 a, b; };
  const auto read = [&](const uint8_t* tile) { return Raw{*reinterpret_cast<const u4*>(tile + 16 * l), *reinterpret_cast<const u4*>(tile + 1024 + 16 * l)}; };
  f4 acc[TM][TN] = {};
  Raw w[RING], x[TM];
  unsigned ew[TN], ex[TM], next_w[TN], next_x[TM];
  const auto read_exps = [&](int q) {
    const unsigned* e = exps + (q & 1) * ROWS;
#pragma unroll
    for (int i = 0; i < TN; ++i) next_w[i] = e[16 * (wn * TN + i) + m];
#pragma unroll
    for (int j = 0; j < TM; ++j) next_x[j] = e[ROWS_W + 16 * (wm * TM + j) + m];
  };
  // All of this wave's loads but those of the last NBUF - 2 steps are in LDS, all of its reads in registers; then the other waves' too.
  const auto barrier = [&] {
    constexpr int LATER = (NBUF - 2) * LOADS;
    __builtin_amdgcn_s_waitcnt(0x0070 | (LATER & 15) | (LATER >> 4) << 14);
    asm volatile("" ::: "memory"); __builtin_amdgcn_s_barrier(); asm volatile("" ::: "memory");
  };
  const int w_at = wn * TN * TILE, x_at = (WN * TN + wm * TM) * TILE;
  // Keeps products where they stand between reads and barrier.
  const auto pin = [&](f4& v) {
    if constexpr (TN * TM == 64) asm volatile("" : "+a"(v)); else asm volatile("" : "+v"(v));
  };
  const auto step = [&](auto byte, int kb) {
    constexpr int U = decltype(byte)::value, S = U % 4;
    uint8_t *now = buffer(Byte<U>{}), *then = buffer(Byte<U + 1>{});
    Operand<EXACT> ox[TM];
#pragma unroll
    for (int j = 0; j < TM; ++j) ox[j] = Operand<EXACT>::template of<S>(x[j].a, x[j].b, ex[j]);
#pragma unroll
    for (int i = 0; i < TN - TAIL; ++i) {
      w[(i + TAIL) % RING] = read(now + w_at + (i + TAIL) * TILE);
      const Operand<EXACT> ow = Operand<EXACT>::template of<S>(w[i % RING].a, w[i % RING].b, ew[i]);
#pragma unroll
      for (int j = 0; j < TM; ++j) acc[j][i] = product<S>(ow, ox[j], acc[j][i]);
#pragma unroll
      for (int j = 0; j < TM; ++j) pin(acc[j][i]);
      __builtin_amdgcn_sched_barrier(0);
    }
    barrier();
    if constexpr (S == 3) read_exps((kb >> 2) + 1);      // (before more is on its way into LDS: the compiler would wait for all of it)
    if constexpr (S == 0) fetch_exps((kb >> 2) + 1);
    Operand<EXACT> ow[TAIL];
#pragma unroll
    for (int i = 0; i < TAIL; ++i) ow[i] = Operand<EXACT>::template of<S>(w[(TN - TAIL + i) % RING].a, w[(TN - TAIL + i) % RING].b, ew[TN - TAIL + i]);
    w[0] = read(then + w_at);
#pragma unroll
    for (int j = 0; j < TM; ++j) {
#pragma unroll
      for (int i = 0; i < TAIL; ++i) acc[j][TN - TAIL + i] = product<S>(ow[i], ox[j], acc[j][TN - TAIL + i]);
#pragma unroll
      for (int i = 0; i < TAIL; ++i) pin(acc[j][TN - TAIL + i]);
      x[j] = read(then + x_at + j * TILE);
      fetch_part(now, LOADS * j / TM, LOADS * (j + 1) / TM);
      __builtin_amdgcn_sched_barrier(0);
    }
    ++next;
#pragma unroll
    for (int i = 1; i < TAIL; ++i) w[i] = read(then + w_at + i * TILE);
  };
  fetch_exps(0);
  fetch(buf0);
  fetch(buf1);
  if constexpr (NBUF > 2) fetch(buf2);
  if constexpr (NBUF == 4) fetch(buf3);
  __builtin_amdgcn_s_waitcnt(0x0070 | ((NBUF - 1) * LOADS & 15) | (NBUF - 1) * LOADS >> 4 << 14);
  __syncthreads();
  read_exps(0);
#pragma unroll
  for (int j = 0; j < TM; ++j) x[j] = read(buf0 + x_at + j * TILE);
#pragma unroll
  for (int i = 0; i < TAIL; ++i) w[i] = read(buf0 + w_at + i * TILE);
  const auto next_exps = [&] {
#pragma unroll
    for (int i = 0; i < TN; ++i) ew[i] = next_w[i];
#pragma unroll
    for (int j = 0; j < TM; ++j) ex[j] = next_x[j];
  };
  int kb = 0;
  if constexpr (NBUF == 3) {
    for (; kb + 12 <= a.nb; kb += 12) {
      next_exps();
      step(Byte<0>{}, kb); step(Byte<1>{}, kb + 1); step(Byte<2>{}, kb + 2); step(Byte<3>{}, kb + 3);
      next_exps();
      step(Byte<4>{}, kb + 4); step(Byte<5>{}, kb + 5); step(Byte<6>{}, kb + 6); step(Byte<7>{}, kb + 7);
      next_exps();
      step(Byte<8>{}, kb + 8); step(Byte<9>{}, kb + 9); step(Byte<10>{}, kb + 10); step(Byte<11>{}, kb + 11);
    }
    const int left = a.nb - kb;
    if (left >= 8) {
      next_exps();
      step(Byte<0>{}, kb); step(Byte<1>{}, kb + 1); step(Byte<2>{}, kb + 2); step(Byte<3>{}, kb + 3);
      next_exps();
      step(Byte<4>{}, kb + 4); step(Byte<5>{}, kb + 5); step(Byte<6>{}, kb + 6); step(Byte<7>{}, kb + 7);
      if (left > 8) {
        next_exps();
        step(Byte<8>{}, kb + 8);
        if (left > 9) step(Byte<9>{}, kb + 9);
        if (left > 10) step(Byte<10>{}, kb + 10);
      }
    } else if (left > 0) {
      next_exps();
      step(Byte<0>{}, kb);
      if (left > 1) step(Byte<1>{}, kb + 1);
      if (left > 2) step(Byte<2>{}, kb + 2);
      if (left > 3) {
        step(Byte<3>{}, kb + 3);
        if (left > 4) {
          next_exps();
          step(Byte<4>{}, kb + 4);
          if (left > 5) step(Byte<5>{}, kb + 5);
          if (left > 6) step(Byte<6>{}, kb + 6);
        }
      }
    }
  } else {
    for (; kb + 4 <= a.nb; kb += 4) {
      next_exps();
      step(Byte<0>{}, kb); step(Byte<1>{}, kb + 1); step(Byte<2>{}, kb + 2); step(Byte<3>{}, kb + 3);
    }
    if (kb < a.nb) {
      next_exps();
      step(Byte<0>{}, kb);
      if (kb + 1 < a.nb) step(Byte<1>{}, kb + 1);
      if (kb + 2 < a.nb) step(Byte<2>{}, kb + 2);
    }
  }
#pragma unroll
  for (int i = 0; i < TAIL; ++i) asm volatile("" : : "v"(w[i].a), "v"(w[i].b));
  __builtin_amdgcn_s_waitcnt(0x0070);      // no load of this block is on its way into LDS that another one may have by then
#pragma unroll
  for (int j = 0; j < TM; ++j)
#pragma unroll
    for (int i = 0; i < TN; i += GATED ? 2 : 1)
      finish<O, GATED>(a, 16 * ((bm * WM + wm) * TM + j) + m, 16 * (((bn * WN + wn) * TN + i) >> GATED) + 4 * g, acc[j][i], acc[j][GATED ? i + 1 : i]);
}

template <typename O, int TN, int TM, int WN, int WM, int NBUF> void launch_tiles(const ProductArgs& a, bool gated, hipStream_t s) {
  const int n = (a.tiles + WN * TN - 1) / (WN * TN), m = (a.M + 16 * WM * TM - 1) / (16 * WM * TM);
  if (gated) k_fp8_tiles<O, TN, TM, WN, WM, NBUF, true><<<n * m, 64 * WN * WM, 0, s>>>(a, n, m);
  else k_fp8_tiles<O, TN, TM, WN, WM, NBUF, false><<<n * m, 64 * WN * WM, 0, s>>>(a, n, m);
}
template <typename O, int MT, int NT, int AHEAD> void launch_stream(const ProductArgs& a, bool gated, hipStream_t s) {
  const dim3 grid((a.tiles + NT - 1) / NT, (a.M + 16 * MT - 1) / (16 * MT));
  if constexpr (NT % 2 == 0) {
    if (gated) return k_fp8_stream<O, MT, NT, AHEAD, true><<<grid, 512, 0, s>>>(a);
  }
  k_fp8_stream<O, MT, NT, AHEAD, false><<<grid, 512, 0, s>>>(a);
}

// Which form is taken: the one that should end first, its time being start + steps * (round * rounds + share * blocks / 256), rounds = blocks / 256 rounded up (a round: a block on each CU), steps the blocks of K
// that a wave goes through.  The constants, in us, are fitted to the times of all forms over 180 sizes (1 to 8192 rows by 1024 to 28672 x 512 to 14336); over these the chosen form takes 1.6 % longer than the
// best one in the mean (fp32: 0.6 % over 77), and over 112 with the form of 192 rows 1.3 % (2.8 without it); at worst 48 % (100 x 2048 x 512, 3.7 us for 2.5).  Over sizes outside of the fit, drawn from 1 to 8192 rows, 512 to 28672 outputs and 256 to
// 16384 inputs, 2.5 % in the mean and 23 % at worst (90 sizes; fp32 1.1 % and 19 %, gated 3.8 % and 41 %, 40 each); a tenth of them miss the best form by more than a tenth.  Up to 16 rows, and wherever a block has one tile of rows, the products are the exact ones for every type: the weights' way from memory hides most of them (8 x 4096 x 4096 4.9 us,
// 4.8 without; 8 x 28672 x 4096 23.6, 21.8).  Some of both sides, us, weights resident in turns (rows x N x K, outputs of 16 bits: stream of 1 x 1, 1 x 2, 2 x 2, 4 x 2 tiles | 64 x 64,
// 64 x 128, 128 x 128 with four buffers, with two, 256 x 256, 192 x 128 through LDS):
//   8 x 4096 x 4096  4.9 5.6             8 x 28672 x 4096  23.9 23.6                                 48 x 4096 x 14336  28 25 16.9 23 | 32 48 51 95 142
//   64 x 28672 x 4096  71 70 41 33 | 27 23.0 25 34 48            200 x 4096 x 4096  21 21 15 12 | 10.4 13 17 25 45             777 x 6144 x 4096  - - 56 49 | 41 41 37 35 51 28.5
//   1024 x 28672 x 4096  - - 520 328 | 213 212 151 149 113       2048 x 4096 x 14336  | 190 174 120 116 158                    8192 x 8192 x 8192  | 810 753 581 511 403
struct Form { int n, m, waves; float start, round, share; };      // tiles of weights and of rows a block, waves that share out K
constexpr Form FORMS[10] = {{1, 1, 8, .76f, .46f, .28f}, {2, 1, 8, 1.81f, .57f, .24f}, {2, 2, 8, 1.79f, .5f, .63f}, {2, 4, 8, 1.9f, .63f, 1.f},
                           {4, 4, 1, 3.97f, .28f, 0.f}, {8, 4, 1, 3.84f, .37f, .07f}, {8, 8, 1, 4.86f, .36f, .22f}, {8, 8, 1, 3.14f, .59f, .2f}, {16, 16, 1, 5.49f, 1.06f, .66f}, {8, 12, 1, 4.f, .44f, .4f}};
constexpr Form EXACT_FORMS[6] = {{1, 1, 8, .92f, .38f, .33f}, {2, 1, 8, .71f, .84f, .24f}, {2, 2, 8, .14f, .94f, .61f}, {2, 4, 8, .3f, .78f, 1.5f}, {4, 4, 1, 8.81f, .25f, .06f}, {8, 8, 1, 8.3f, .67f, .13f}};
// (Forms whose launch would have more than 65535 blocks in y or 2^32 threads in x are left out; the fourth never has.)
template <int COUNT> int form_of(const Form (&forms)[COUNT], const ProductArgs& a, bool gated) {
  int best = -1;
  float least = 0;
  for (int i = 0; i < (a.M <= 16 ? 2 : COUNT); ++i) {
    const Form& f = forms[i];
    if (gated && f.n % 2 != 0) continue;
    const long high = (a.M + 16 * f.m - 1) / (16 * f.m), blocks = (a.tiles + f.n - 1) / f.n * high;
    if (f.waves == 1 ? blocks >= 1 << 22 : high > 65535) continue;
    const int steps = f.waves == 1 ? a.nb : 4 * (((a.nb + 3) / 4 + f.waves - 1) / f.waves);
    const float time = f.start + steps * (f.round * ((blocks + 255) / 256) + f.share * blocks / 256.f);
    if (best < 0 || time < least) { best = i; least = time; }
  }
  return best;
}
int form_of(const ProductArgs& a, bool gated, bool exact) { return exact ? form_of(EXACT_FORMS, a, gated) : form_of(FORMS, a, gated); }
template <typename O> void launch_product(const ProductArgs& a, bool gated, hipStream_t s) {
  if constexpr (sizeof(O) == 4) {
    switch (form_of(a, gated, true)) {
      case 0: return launch_stream<O, 1, 1, 4>(a, gated, s);
      case 1: return launch_stream<O, 1, 2, 4>(a, gated, s);
      case 2: return launch_stream<O, 2, 2, 4>(a, gated, s);
      case 3: return launch_stream<O, 4, 2, 2>(a, gated, s);
      case 4: return launch_tiles<O, 4, 1, 1, 4, 4>(a, gated, s);
      default: return launch_tiles<O, 4, 4, 2, 2, 2>(a, gated, s);
    }
  } else {
    switch (form_of(a, gated, false)) {
      case 0: return launch_stream<O, 1, 1, 4>(a, gated, s);
      case 1: return launch_stream<O, 1, 2, 4>(a, gated, s);
      case 2: return launch_stream<O, 2, 2, 4>(a, gated, s);
      case 3: return launch_stream<O, 4, 2, 2>(a, gated, s);
      case 4: return launch_tiles<O, 4, 1, 1, 4, 4>(a, gated, s);
      case 5: return launch_tiles<O, 4, 1, 2, 4, 4>(a, gated, s);
      case 6: return launch_tiles<O, 4, 2, 2, 4, 4>(a, gated, s);
      case 7: return launch_tiles<O, 4, 2, 2, 4, 2>(a, gated, s);
      case 8: return launch_tiles<O, 8, 4, 2, 4, 2>(a, gated, s);
      default: return launch_tiles<O, 4, 3, 2, 4, 3>(a, gated, s);
    }
  }
}

constexpr int MOST_ROWS = 1 << 20, PART = 4;      // of one launch, of up to 1024 threads a row: a launch has less than 2^32 in x | waves of a part of a row
template <typename T, int CH> void launch_rows(RowsArgs a, int M, int parts, hipStream_t s) {
  for (a.first = 0; a.first < M; a.first += MOST_ROWS) {
    const int n = M - a.first < MOST_ROWS ? M - a.first : MOST_ROWS;
    if constexpr (CH < 8) {
      if (a.weight != nullptr) { k_fp8_rows<T, true, CH><<<n, 64 * a.waves, 0, s>>>(a); continue; }
    }
    k_fp8_rows<T, false, CH><<<dim3(n, parts), 64 * a.waves, 0, s>>>(a);
  }
}
// One run a lane for few rows, where latency counts, two for many (us, one / two runs, with the norm: 4 x 4096 4.0 / 4.8, 300 x 4096 6.3 / 6.9, 777 x 5000 12.5 / 10.9, 16384 x 4096 125 / 113); more only where a block's 16 waves
// would not do.  (The norm of 8 runs would not fit the registers.)  Few rows without the norm in parts of up to four waves, a block each (us, a block a row / in parts: 4 x 14336 2.9 / 2.2, 48 x 14336 3.9 / 3.1); many rows
// not: 2048 x 16384 25.9 / 30.0, as the parts of a row are then read far from each other.
template <typename T> void launch_rows(RowsArgs a, int M, hipStream_t s) {
  const auto waves = [&](int n) { return (a.nb * 16 + 64 * n - 1) / (64 * n); };
  int ch = (long)M * waves(1) <= 4096 ? 1 : 2, parts = 1;
  if (ch == 1 && a.weight == nullptr) parts = (waves(1) + PART - 1) / PART;
  while ((waves(ch) + parts - 1) / parts > 16) ch *= 2;
  a.waves = (waves(ch) + parts - 1) / parts;
  if (ch == 1) launch_rows<T, 1>(a, M, parts, s); else if (ch == 2) launch_rows<T, 2>(a, M, 1, s); else if (ch == 4) launch_rows<T, 4>(a, M, 1, s); else launch_rows<T, 8>(a, M, 1, s);
}

uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

}  // namespace

extern "C" int gaac_fp8_rows(int type, const void* x, long x_row_stride, const void* residual, long residual_row_stride, const void* weight, float eps, int M, int K, void* sum, void* data, void* exps,
                             long padded_rows, int tile_step, int tile_first, void* stream) {
  GAAC_REQUIRE(x != nullptr && data != nullptr && exps != nullptr, "gaac_fp8_rows: null pointer");
  GAAC_REQUIRE(type >= 0 && type <= 2, "gaac_fp8_rows: type must be 0 (bf16), 1 (fp16) or 2 (fp32)");
  GAAC_REQUIRE(M > 0 && M <= 1 << 24 && K > 0 && K <= MAX_K, "gaac_fp8_rows: bad sizes (%d rows of %d, up to 2^24 of %d)", M, K, MAX_K);
  GAAC_REQUIRE(weight == nullptr || K <= MAX_NORM_K, "gaac_fp8_rows: the norm takes rows of up to %d, not %d", MAX_NORM_K, K);
  GAAC_REQUIRE((residual == nullptr) == (sum == nullptr) && (residual == nullptr || weight != nullptr), "gaac_fp8_rows: a residual and its sum together, and with the norm's weight");
  GAAC_REQUIRE(tile_step >= 1 && tile_first >= 0 && tile_first < tile_step && padded_rows >= 16l * ((M + 15) / 16) * tile_step, "gaac_fp8_rows: bad sizes (%d rows in every %dth of tiles of %ld rows)", M, tile_step, padded_rows);
  GAAC_REQUIRE(address(data) % 16 == 0 && address(exps) % 4 == 0, "gaac_fp8_rows: data must be 16-byte aligned, exponents 4-byte");
  const int per = type == 2 ? 4 : 8;
  const bool whole = (address(x) | address(residual) | address(weight) | address(sum)) % 16 == 0 && (x_row_stride | residual_row_stride | K) % per == 0 && K % 8 == 0;
  const RowsArgs a{x, residual, weight, sum, static_cast<uint8_t*>(data), static_cast<uint8_t*>(exps), x_row_stride, residual_row_stride, padded_rows, K, (K + BLOCK - 1) / BLOCK, 1, tile_step, tile_first, 0, eps, whole};
  if (type == 0) launch_rows<__bf16>(a, M, (hipStream_t)stream);
  else if (type == 1) launch_rows<_Float16>(a, M, (hipStream_t)stream);
  else launch_rows<float>(a, M, (hipStream_t)stream);
  return gaac::launch_status("gaac_fp8_rows");
}

extern "C" int gaac_fp8_values(const void* data, const void* exps, long padded_rows, int tile_step, int tile_first, int M, int K, void* out, long out_row_stride, void* stream) {
  GAAC_REQUIRE(data != nullptr && exps != nullptr && out != nullptr, "gaac_fp8_values: null pointer");
  GAAC_REQUIRE(M > 0 && M <= 1 << 24 && K > 0 && K <= MAX_K, "gaac_fp8_values: bad sizes (%d rows of %d, up to 2^24 of %d)", M, K, MAX_K);
  GAAC_REQUIRE(tile_step >= 1 && tile_first >= 0 && tile_first < tile_step && padded_rows >= 16l * ((M + 15) / 16) * tile_step, "gaac_fp8_values: bad sizes (%d rows in every %dth of tiles of %ld rows)", M, tile_step, padded_rows);
  GAAC_REQUIRE(address(data) % 16 == 0 && address(exps) % 4 == 0, "gaac_fp8_values: data must be 16-byte aligned, exponents 4-byte");
  const int nb = (K + BLOCK - 1) / BLOCK;
  const bool whole = address(out) % 16 == 0 && out_row_stride % 8 == 0;
  const long tiles = (M + 15) / 16, most = (1 << 22) / nb;      // (a launch has less than 2^32 threads)
  for (long first = 0; first < tiles; first += most)
    k_fp8_values<<<(unsigned)((tiles - first < most ? tiles - first : most) * nb), 256, 0, (hipStream_t)stream>>>(static_cast<const uint8_t*>(data), static_cast<const uint8_t*>(exps), padded_rows, tile_step, tile_first, first, M, K,
                                                                                                               nb, static_cast<__bf16*>(out), out_row_stride, whole);
  return gaac::launch_status("gaac_fp8_values");
}

extern "C" int gaac_fp8_product(const void* x, const void* x_exps, const void* w, const void* w_exps, int M, int N, int K, int gated, int out_type, void* out, long out_row_stride, void* stream) {
  GAAC_REQUIRE(x != nullptr && x_exps != nullptr && w != nullptr && w_exps != nullptr && out != nullptr, "gaac_fp8_product: null pointer");
  GAAC_REQUIRE(out_type >= 0 && out_type <= 2, "gaac_fp8_product: type must be 0 (bf16), 1 (fp16) or 2 (fp32)");
  GAAC_REQUIRE(M > 0 && M <= 1 << 20 && K > 0 && K <= MAX_K && N > 0 && N <= 1 << 22, "gaac_fp8_product: bad sizes (%d rows of %d by %d)", M, K, N);
  GAAC_REQUIRE((address(x) | address(w)) % 16 == 0 && (address(x_exps) | address(w_exps)) % 4 == 0, "gaac_fp8_product: data must be 16-byte aligned, exponents 4-byte");
  const int size = out_type == 2 ? 4 : 2, tiles = (N + 15) / 16 * (gated ? 2 : 1);
  const bool whole = address(out) % (4 * size) == 0 && out_row_stride % 4 == 0;
  const ProductArgs a{x, static_cast<const unsigned*>(x_exps), static_cast<const uint8_t*>(w), static_cast<const unsigned*>(w_exps), out, 16l * ((M + 15) / 16), 16l * tiles, out_row_stride, M, N, K, (K + BLOCK - 1) / BLOCK, tiles, whole};
  if (out_type == 0) launch_product<__bf16>(a, gated != 0, (hipStream_t)stream);
  else if (out_type == 1) launch_product<_Float16>(a, gated != 0, (hipStream_t)stream);
  else launch_product<float>(a, gated != 0, (hipStream_t)stream);
  return gaac::launch_status("gaac_fp8_product");
}

extern "C" int gaac_fp8_product_form(int M, int N, int K, int gated, int out_type, int* form) {
  GAAC_REQUIRE(form != nullptr, "gaac_fp8_product_form: null pointer");
  GAAC_REQUIRE(out_type >= 0 && out_type <= 2, "gaac_fp8_product_form: type must be 0 (bf16), 1 (fp16) or 2 (fp32)");
  GAAC_REQUIRE(M > 0 && M <= 1 << 20 && K > 0 && K <= MAX_K && N > 0 && N <= 1 << 22, "gaac_fp8_product_form: bad sizes (%d rows of %d by %d)", M, K, N);
  ProductArgs a{};
  a.M = M; a.N = N; a.K = K; a.nb = (K + BLOCK - 1) / BLOCK; a.tiles = (N + 15) / 16 * (gated ? 2 : 1);
  *form = form_of(a, gated != 0, out_type == 2);
  return 0;
}
