// Rows in 8 bits: their quantiser (with the residual's addition and the root-mean-square norm before it), the way back, and products of such rows with such weights.
//
// Format: 128 consecutive elements of a row are a block.  A block has one power of two 2^E, E the smallest integer with amax <= 448 * 2^E, from -117 to 119, held as the
// byte E + 127 (255: the block held a NaN or an infinity and reads as NaN), and e4m3 codes: the nearest to x * 2^-E, ties to the even code.  Scaling is by a power of two, so
// only that rounding is made, and every value is a normal number of bf16 (2^-126 to 448 * 2^119) or zero.  Elements behind the row's end are zero codes.
//
// 16 rows by one block are a tile, 2048 bytes in the order of the operands of the scaled 16x16x128 product, a lane's 16 bytes next to each other: row m, element
// 32 g + 16 j + i of the block at byte 1024 j + 16 (16 g + m) + i.  (Which elements of a block a lane group has is free, as long as both operands agree: they share one power of
// two.)  A row of tiles is the blocks one after the other.  The exponent bytes of four blocks are a dword, byte s that of block 4 q + s, dword [q][row]: the
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
__device__ __forceinline__ double wave_sum(double x) {
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// ---------------------------------------------------------------------------------------------------- rows into 8 bits
struct RowsArgs {
  const void *x, *residual, *weight;
  void* sum;
  uint8_t *data, *exps;
  long x_rs, r_rs, pad;
  int M, K, nb, waves, tile_step, tile_first;
  float eps;
  bool whole;
};

// `waves` waves a row, a lane CH runs of 8 elements of it, 16 lanes a block.  The sum of squares and the norm in 64 bits, which cost nothing beside the memory: a result next to the border
// between two codes is then nearly always rounded as the formula says.
template <typename T, bool NORM, int CH>
__global__ __launch_bounds__(1024) void k_fp8_rows(RowsArgs a) {
  __shared__ double sums[16];
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, part = wave % a.waves, row = blockIdx.x * ((blockDim.x >> 6) / a.waves) + wave / a.waves;
  const bool there = row < a.M;
  const T* src = static_cast<const T*>(a.x) + row * a.x_rs;
  float x[CH][8];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int k = 8 * ((i * a.waves + part) * 64 + l);
    load_some(src + k, there ? a.K - k : 0, a.whole, x[i]);
  }
  if constexpr (NORM) {
    if (a.residual != nullptr) {
      const T* res = static_cast<const T*>(a.residual) + row * a.r_rs;
      T* out = static_cast<T*>(a.sum) + (long)row * a.K;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int k = 8 * ((i * a.waves + part) * 64 + l), n = there ? a.K - k : 0;
        float r[8];
        load_some(res + k, n, a.whole, r);
        for (int j = 0; j < 8; ++j) x[i][j] += r[j];
        store_some(out + k, n, a.whole, x[i]);
      }
    }
    double sum = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i)
      for (int j = 0; j < 8; ++j) sum = __builtin_fma((double)x[i][j], (double)x[i][j], sum);
    sum = wave_sum(sum);
    if (a.waves > 1) {
      if (l == 0) sums[wave] = sum;
      __syncthreads();
      sum = 0;
      for (int i = 0; i < a.waves; ++i) sum += sums[wave - part + i];
    }
    const double r = 1.0 / __builtin_sqrt(sum / a.K + (double)a.eps);
    const T* w = static_cast<const T*>(a.weight);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int k = 8 * ((i * a.waves + part) * 64 + l);
      float g[8];
      load_some(w + k, a.K - k, a.whole, g);
      for (int j = 0; j < 8; ++j) x[i][j] = (float)((double)x[i][j] * r * (double)g[j]);
    }
  }
  if (!there) return;
  const long tile_row = (long)(row >> 4) * a.tile_step + a.tile_first;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = (i * a.waves + part) * 64 + l, kb = c >> 4, p = c & 15;
    if (kb >= a.nb) continue;
    if constexpr (NORM) {      // (behind the row's end 0 * r may be a NaN)
      if (8 * c + 8 > a.K) for (int j = 0; j < 8; ++j) x[i][j] = 8 * c + j < a.K ? x[i][j] : 0.f;
    }
    const unsigned e = exponent_byte(max16(magnitude8(x[i])));
    *reinterpret_cast<u2*>(a.data + (tile_row * a.nb + kb) * TILE + 1024 * (p >> 1 & 1) + 16 * (16 * (p >> 2) + (row & 15)) + 8 * (p & 1)) = encode8(x[i], e);
    if (p == 0) a.exps[((kb >> 2) * a.pad + 16 * tile_row + (row & 15)) * 4 + (kb & 3)] = (uint8_t)e;
  }
}

// The way back: a block of threads a tile, 16 lanes a row's 256 bytes.
__global__ __launch_bounds__(256) void k_fp8_values(const uint8_t* data, const uint8_t* exps, long pad, int tile_step, int tile_first, int M, int K, int nb, __bf16* out, long out_rs, bool whole) {
  const int p = threadIdx.x & 15, m = threadIdx.x >> 4, kb = blockIdx.x % nb;
  const long tile = blockIdx.x / nb, row = 16 * tile + m, tile_row = tile * tile_step + tile_first;
  if (row >= M) return;
  const u2 w = *reinterpret_cast<const u2*>(data + (tile_row * nb + kb) * TILE + 1024 * (p >> 1 & 1) + 16 * (16 * (p >> 2) + m) + 8 * (p & 1));
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
  const void* x;             // rows in 8 bits, or as they come
  const unsigned* x_exps;
  const uint8_t* w;
  const unsigned* w_exps;
  void* out;
  long x_rs, x_pad, w_pad, out_rs;
  int M, N, K, nb, tiles;      // tiles: of 16 weight rows
  bool whole;                  // four outputs at a time
};

// One block of K of a tile of weights by one of rows, byte S of both exponent words.  The scaled product adds eight elements' products as whole multiples of 2^-13 of the largest one's power of
// two, cutting what is below, and only these sums in 32 bits (found by trying: so does the product without scales).  That is an error of 1.5e-5 to 3e-5 of the output's size, a sixtieth of bf16's rounding and an
// eighth of fp16's.  Outputs in 32 bits would show it: for them (EXACT) the codes go as bf16, scale included, which holds them exactly, into products that are added in 32 bits, at half the rate.
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

// Few rows: the weights go by once.  A block has NT tiles of weights and MT of rows; its eight waves share the blocks of K out, four (a dword of exponents) at a time, and their sums meet in LDS, in
// the waves' order.
template <typename O, int MT, int NT, bool GATED>
__global__ __launch_bounds__(512) void k_fp8_stream(ProductArgs a) {
  static_assert(!GATED || NT % 2 == 0, "tiles of a gated pair alternate");
  constexpr bool EXACT = sizeof(O) == 4;
  __shared__ f4 part[8][MT * NT][64];
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, m = l & 15, g = l >> 4;
  const uint8_t *w[NT], *x[MT];
  const unsigned *we[NT], *xe[MT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {      // (a tile behind the last one is the last one again, and written by nobody)
    const long t = min((int)blockIdx.x * NT + i, a.tiles - 1);
    w[i] = a.w + t * a.nb * TILE; we[i] = a.w_exps + 16 * t + m;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const long t = min((int)blockIdx.y * MT + i, (a.M - 1) >> 4);
    x[i] = static_cast<const uint8_t*>(a.x) + t * a.nb * TILE; xe[i] = a.x_exps + 16 * t + m;
  }
  f4 acc[MT][NT] = {};
  for (int q = wave; 4 * q < a.nb; q += 8) {
    unsigned ew[NT], ex[MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) ew[i] = we[i][q * a.w_pad];
#pragma unroll
    for (int i = 0; i < MT; ++i) ex[i] = xe[i][q * a.x_pad];
    const auto step = [&](auto byte) {
      constexpr int S = decltype(byte)::value;
      const long at = (long)(4 * q + S) * TILE;
      Operand<EXACT> ow[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) ow[i] = operand<EXACT, S>(w[i] + at, l, ew[i]);
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const Operand<EXACT> ox = operand<EXACT, S>(x[j] + at, l, ex[j]);
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[j][i] = product<S>(ow[i], ox, acc[j][i]);
      }
    };
    const int n = a.nb - 4 * q;
    if (n >= 4) {
      step(Byte<0>{}); step(Byte<1>{}); step(Byte<2>{}); step(Byte<3>{});
    } else {
      step(Byte<0>{});
      if (n > 1) step(Byte<1>{});
      if (n > 2) step(Byte<2>{});
    }
  }
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int i = 0; i < NT; ++i) part[wave][j * NT + i][l] = acc[j][i];
  __syncthreads();
  constexpr int EACH = GATED ? NT / 2 : NT;      // outputs of a tile of rows, by 16
  for (int at = wave; at < MT * EACH; at += 8) {
    const int j = at / EACH, i = at % EACH;
    const auto sum = [&](int t) {
      f4 s = part[0][j * NT + t][l];
      for (int k = 1; k < 8; ++k) s += part[k][j * NT + t][l];
      return s;
    };
    f4 v = sum(GATED ? 2 * i : i);
    if constexpr (GATED) {
      const f4 up = sum(2 * i + 1);
      for (int k = 0; k < 4; ++k) v[k] = silu(v[k]) * up[k];
    }
    const int row = 16 * ((int)blockIdx.y * MT + j) + m, col = 16 * ((int)blockIdx.x * EACH + i) + 4 * g;
    if (row < a.M && col < a.N) put_some(static_cast<O*>(a.out) + row * a.out_rs + col, v, a.N - col, a.whole);
  }
}

template <typename O> void launch_product(const ProductArgs& a, bool gated, hipStream_t s) {
  if (gated) {
    const int most = (a.tiles + 1) / 2;
    if (a.M <= 16) k_fp8_stream<O, 1, 2, true><<<dim3(most, 1), 512, 0, s>>>(a);
    else k_fp8_stream<O, 4, 2, true><<<dim3(most, (a.M + 63) / 64), 512, 0, s>>>(a);
  } else {
    if (a.M <= 16) k_fp8_stream<O, 1, 1, false><<<dim3(a.tiles, 1), 512, 0, s>>>(a);
    else k_fp8_stream<O, 4, 2, false><<<dim3((a.tiles + 1) / 2, (a.M + 63) / 64), 512, 0, s>>>(a);
  }
}

template <typename T, int CH> void launch_rows(const RowsArgs& a, int block, hipStream_t s) {
  const unsigned grid = (unsigned)((a.M + block / a.waves - 1) / (block / a.waves));
  if constexpr (CH < 8) if (a.weight != nullptr) return k_fp8_rows<T, true, CH><<<grid, 64 * block, 0, s>>>(a);
  k_fp8_rows<T, false, CH><<<grid, 64 * block, 0, s>>>(a);
}
template <typename T> void launch_rows(RowsArgs a, hipStream_t s) {
  int ch = 1;
  const auto waves = [&](int n) { return (a.nb * 16 + 64 * n - 1) / (64 * n); };
  const int most = a.weight != nullptr ? 4 : 8;      // (the norm of 8 runs would not fit the registers)
  while (ch < most && (waves(ch) > 16 || (long)a.M * waves(ch) > 8192)) ch *= 2;
  a.waves = waves(ch);
  const int block = (long)a.M * a.waves > 2048 ? 16 / a.waves * a.waves : a.waves;
  if (ch == 1) launch_rows<T, 1>(a, block, s); else if (ch == 2) launch_rows<T, 2>(a, block, s); else if (ch == 4) launch_rows<T, 4>(a, block, s); else launch_rows<T, 8>(a, block, s);
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
  const RowsArgs a{x, residual, weight, sum, static_cast<uint8_t*>(data), static_cast<uint8_t*>(exps), x_row_stride, residual_row_stride, padded_rows, M, K, (K + BLOCK - 1) / BLOCK, 1, tile_step, tile_first, eps, whole};
  if (type == 0) launch_rows<__bf16>(a, (hipStream_t)stream);
  else if (type == 1) launch_rows<_Float16>(a, (hipStream_t)stream);
  else launch_rows<float>(a, (hipStream_t)stream);
  return gaac::launch_status("gaac_fp8_rows");
}

extern "C" int gaac_fp8_values(const void* data, const void* exps, long padded_rows, int tile_step, int tile_first, int M, int K, void* out, long out_row_stride, void* stream) {
  GAAC_REQUIRE(data != nullptr && exps != nullptr && out != nullptr, "gaac_fp8_values: null pointer");
  GAAC_REQUIRE(M > 0 && M <= 1 << 24 && K > 0 && K <= MAX_K, "gaac_fp8_values: bad sizes (%d rows of %d, up to 2^24 of %d)", M, K, MAX_K);
  GAAC_REQUIRE(tile_step >= 1 && tile_first >= 0 && tile_first < tile_step && padded_rows >= 16l * ((M + 15) / 16) * tile_step, "gaac_fp8_values: bad sizes (%d rows in every %dth of tiles of %ld rows)", M, tile_step, padded_rows);
  GAAC_REQUIRE(address(data) % 16 == 0 && address(exps) % 4 == 0, "gaac_fp8_values: data must be 16-byte aligned, exponents 4-byte");
  const int nb = (K + BLOCK - 1) / BLOCK;
  const bool whole = address(out) % 16 == 0 && out_row_stride % 8 == 0;
  k_fp8_values<<<(unsigned)((M + 15) / 16) * nb, 256, 0, (hipStream_t)stream>>>(static_cast<const uint8_t*>(data), static_cast<const uint8_t*>(exps), padded_rows, tile_step, tile_first, M, K, nb, static_cast<__bf16*>(out), out_row_stride, whole);
  return gaac::launch_status("gaac_fp8_values");
}

extern "C" int gaac_fp8_product(const void* x, const void* x_exps, const void* w, const void* w_exps, int M, int N, int K, int gated, int out_type, void* out, long out_row_stride, void* stream) {
  GAAC_REQUIRE(x != nullptr && x_exps != nullptr && w != nullptr && w_exps != nullptr && out != nullptr, "gaac_fp8_product: null pointer");
  GAAC_REQUIRE(out_type >= 0 && out_type <= 2, "gaac_fp8_product: type must be 0 (bf16), 1 (fp16) or 2 (fp32)");
  GAAC_REQUIRE(M > 0 && M <= 1 << 20 && K > 0 && K <= MAX_K && N > 0 && N <= 1 << 22, "gaac_fp8_product: bad sizes (%d rows of %d by %d)", M, K, N);
  GAAC_REQUIRE((address(x) | address(w)) % 16 == 0 && (address(x_exps) | address(w_exps)) % 4 == 0, "gaac_fp8_product: data must be 16-byte aligned, exponents 4-byte");
  const int size = out_type == 2 ? 4 : 2, tiles = (N + 15) / 16 * (gated ? 2 : 1);
  const bool whole = address(out) % (4 * size) == 0 && out_row_stride % 4 == 0;
  const ProductArgs a{x, static_cast<const unsigned*>(x_exps), static_cast<const uint8_t*>(w), static_cast<const unsigned*>(w_exps), out, 0, 16l * ((M + 15) / 16), 16l * tiles, out_row_stride, M, N, K, (K + BLOCK - 1) / BLOCK, tiles, whole};
  if (out_type == 0) launch_product<__bf16>(a, gated != 0, (hipStream_t)stream);
  else if (out_type == 1) launch_product<_Float16>(a, gated != 0, (hipStream_t)stream);
  else launch_product<float>(a, gated != 0, (hipStream_t)stream);
  return gaac::launch_status("gaac_fp8_product");
}
