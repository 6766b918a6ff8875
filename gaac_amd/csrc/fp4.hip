// The 4-bit cache: its tiles, their encoder (prompt, appended token), decoder, and decode attention over them.
//
// Format (OCP MXFP4): 32 consecutive channels of one token and head are a block.  A block has one power of two 2^E, E the smallest integer with
// amax < 7 * 2^E, from -125 to 125, held as the byte E + 127 (255: the block held a NaN or an infinity and reads as NaN), and 4-bit codes: sign, and the nearest of
// 0 .5 1 1.5 2 3 4 6 to |x| * 2^-E, ties to the even code, at most 6.  With amax < 7 * 2^E no element is off by more than half of the grid's last step, and
// the exponent needs one addition to amax's bits.  Rounding is by a power of two, so a code is exact whatever type it is computed in; every value is a
// normal number of bf16 (2^-126 to 6 * 2^125) or zero, so expanding a code rounds nothing.  gfx950 converts both ways in one instruction for two elements, scale included.
//
// A tile is 32 tokens of one cache head, K and V, 4352 bytes in a row.  Its unit is a dword: 8 consecutive channels of one token, so that appending a
// token writes whole dwords.  They lie in the order of the operands of the matrix instructions, a lane's 16 bytes next to each other, lane l = 16 g + m:
//   K, token 16 s + m, channels 32 g + 8 i ..:  byte 1024 s + 16 l + 4 i.      A block a lane: the operand of the scaled 16x16x128 product, as it is.
//   V, token 16 s + 4 g + i, channels 8 m ..:   byte 2048 + 1024 s + 16 l + 4 i.      Expanded and transposed in registers: V^T of the 16x16x32 product.
//   K's exponent byte of token 16 s + m, block g: 4096 + 2 l + s.  V's of token 16 s + 4 g + i, block b: 4224 + 32 b + 8 g + 4 s + i.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <limits.h>
#include "gaac_capi.h"
#include "../../include/gaac_hip.h"

namespace {

constexpr int NW = 8;      // waves of an attention block: two blocks on a CU (and dwords of a lane's part of a query)
constexpr int DIM = 128, TT = 32, TILE = 4352, V_AT = 2048, KS_AT = 4096, VS_AT = 4224;

typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i8 __attribute__((ext_vector_type(8)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ unsigned pk_max(unsigned a, unsigned b) {
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(us2, a), __builtin_bit_cast(us2, b)));
}
// Largest magnitude (bf16 bits) of a unit's 8 elements, two candidates packed.
__device__ __forceinline__ unsigned unit_max(u4 x) {
  return pk_max(pk_max(x[0] & 0x7fff7fffu, x[1] & 0x7fff7fffu), pk_max(x[2] & 0x7fff7fffu, x[3] & 0x7fff7fffu));
}
// Exponent byte from the packed magnitudes of a block.  amax = m 2^e < 7 * 2^E = 1.75 * 2^(E+2): one more where the mantissa is 1.75 or above.
__device__ __forceinline__ unsigned exponent_byte(unsigned packed) {
  const unsigned a = max(packed & 0xffffu, packed >> 16);
  return a >= 0x7f80u ? 255u : (unsigned)min(max((int)((a + 0x20u) >> 7) - 2, 2), 252);
}
// The conversions look at the exponent field only: bits above and below the byte, which stands at bit `at` of x, may be anything.
__device__ __forceinline__ float scale_of(unsigned x, int at = 0) { return __builtin_bit_cast(float, at <= 23 ? x << (23 - at) : x >> (at - 23)); }
__device__ __forceinline__ bf2 pair(unsigned x) { return __builtin_bit_cast(bf2, x); }      // (a bit cast of a vector's element takes the first one)
__device__ __forceinline__ unsigned encode_unit(u4 x, float scale) {
  unsigned w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, pair(x[0]), scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, pair(x[1]), scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, pair(x[2]), scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, pair(x[3]), scale, 3);
  return w;
}
__device__ __forceinline__ u4 decode_unit(unsigned w, float scale) {
  u4 x;
  x[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
  x[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
  x[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
  x[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
  return x;
}

// ---------------------------------------------------------------------------------------------------- prompt
// A wave encodes K (blockIdx.z = 0) or V of one tile; four tiles a block.  Bound by HBM: 8 KB read and 2.1 KB written per tile and kind.  A lane
// loads 64 bytes in a row of two tokens (K) or 16 of eight (V: whole 256-byte rows by 16 lanes); a store is 1 KB in a row.  All 8 loads of a lane are in flight
// before the first is used.  32768 tokens x 8 heads: 36.8 us, 4.6 TB/s read and written, a large copy's rate (K's rows loaded whole by 16 lanes and turned through LDS:
// 36.3); 777 x 8: 3.4, a launch being 1.6.  Rows of the last tile behind the prompt become zero bytes.
__global__ __launch_bounds__(256) void k_fp4_store(const uint16_t* k, const uint16_t* v, long k_hs, long k_rs, long v_hs, long v_rs, int L, int tiles, uint8_t* cache, int* len) {
  if (len != nullptr && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) *len = L;
  const int tile = blockIdx.x * 4 + (threadIdx.x >> 6), l = threadIdx.x & 63, m = l & 15, g = l >> 4, head = blockIdx.y;
  if (tile * TT >= L) return;
  uint8_t* out = cache + ((long)head * tiles + tile) * TILE;
  if (blockIdx.z == 0) {
    const uint16_t* src = k + head * k_hs + 32 * g;
    u4 x[2][4];
    for (int s = 0; s < 2; ++s) {
      const int t = tile * TT + 16 * s + m;
      for (int i = 0; i < 4; ++i) x[s][i] = t < L ? *reinterpret_cast<const u4*>(src + t * k_rs + 8 * i) : u4{0, 0, 0, 0};
    }
    unsigned exps = 0;
    for (int s = 0; s < 2; ++s) {      // a block of K is a lane's
      const unsigned e = exponent_byte(pk_max(pk_max(unit_max(x[s][0]), unit_max(x[s][1])), pk_max(unit_max(x[s][2]), unit_max(x[s][3]))));
      u4 w;
      for (int i = 0; i < 4; ++i) w[i] = encode_unit(x[s][i], scale_of(e));
      if (tile * TT + 16 * s + m < L) exps |= e << 8 * s;
      *reinterpret_cast<u4*>(out + 1024 * s + 16 * l) = w;
    }
    *reinterpret_cast<uint16_t*>(out + KS_AT + 2 * l) = (uint16_t)exps;
  } else {
    const uint16_t* src = v + head * v_hs + 8 * m;
    u4 x[2][4];
    for (int s = 0; s < 2; ++s)
      for (int i = 0; i < 4; ++i) {
        const int t = tile * TT + 16 * s + 4 * g + i;
        x[s][i] = t < L ? *reinterpret_cast<const u4*>(src + t * v_rs) : u4{0, 0, 0, 0};
      }
    u2 exps = {0, 0};
    for (int s = 0; s < 2; ++s) {
      u4 w;
      for (int i = 0; i < 4; ++i) {      // a block of V is four lanes next to each other
        unsigned a = unit_max(x[s][i]);
        a = pk_max(a, __shfl_xor(a, 1));
        a = pk_max(a, __shfl_xor(a, 2));
        const unsigned e = exponent_byte(a);
        w[i] = encode_unit(x[s][i], scale_of(e));
        if (tile * TT + 16 * s + 4 * g + i < L) exps[s] |= e << 8 * i;
      }
      *reinterpret_cast<u4*>(out + V_AT + 1024 * s + 16 * l) = w;
    }
    if ((m & 3) == 0) *reinterpret_cast<u2*>(out + VS_AT + 8 * m + 8 * g) = exps;      // block m / 4
  }
}

// The way back, by the same waves.  Bound by HBM: 2.1 KB read and 8 KB written per tile and kind, rows of 256 bytes written by 16 lanes (32768 tokens x 8 heads:
// 36.1 us, 4.7 TB/s; K with 64 bytes of a row a lane, as the encoder reads it: 48.5).
__global__ __launch_bounds__(256) void k_fp4_load(const uint8_t* cache, int L, int tiles, uint16_t* k, uint16_t* v, long k_hs, long k_rs, long v_hs, long v_rs) {
  const int tile = blockIdx.x * 4 + (threadIdx.x >> 6), l = threadIdx.x & 63, m = l & 15, g = l >> 4, head = blockIdx.y;
  if (tile * TT >= L) return;
  const uint8_t* in = cache + ((long)head * tiles + tile) * TILE;
  if (blockIdx.z == 0) {
    // (not in the order that a lane's 16 bytes have: a token's row is written as a whole by 16 lanes, and the dwords come out of the same lines)
    unsigned w[8], e[8];
    for (int i = 0; i < 8; ++i) {      // token 4 i + g, unit m
      const int t = 4 * i + g, lane = 16 * (m >> 2) + (t & 15);
      w[i] = *reinterpret_cast<const unsigned*>(in + 1024 * (t >> 4) + 16 * lane + 4 * (m & 3));
      e[i] = in[KS_AT + 2 * lane + (t >> 4)];
    }
    for (int i = 0; i < 8; ++i) {
      const int t = tile * TT + 4 * i + g;
      if (t < L) *reinterpret_cast<u4*>(k + head * k_hs + t * k_rs + 8 * m) = decode_unit(w[i], scale_of(e[i]));
    }
  } else {
    const u2 exps = *reinterpret_cast<const u2*>(in + VS_AT + 32 * (m >> 2) + 8 * g);
    for (int s = 0; s < 2; ++s) {
      const u4 w = *reinterpret_cast<const u4*>(in + V_AT + 1024 * s + 16 * l);
      for (int i = 0; i < 4; ++i) {
        const int t = tile * TT + 16 * s + 4 * g + i;
        if (t < L) *reinterpret_cast<u4*>(v + head * v_hs + t * v_rs + 8 * m) = decode_unit(w[i], scale_of(exps[s] >> 8 * i & 255));
      }
    }
  }
}

// A slot's length for the host, as the other kernels read it: the word is the caller's to write, and below 0 means "not there yet" to the host's wait.
__global__ void k_fp4_length(const int* len, int cap, int* host) { __hip_atomic_store(host, max(min(*len, cap), 0), __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM); }

// ---------------------------------------------------------------------------------------------------- one token
// A block per batch row, a thread per unit (K or V, head, 8 channels); a block of channels is four threads next to each other.  The row's length is
// raised once all of the block have read it.  Bound by the launch and one load after the other (slot, length, element): 2.6 us from 4 rows x 8 heads to 32, of which
// an empty launch takes 1.6.
__global__ __launch_bounds__(256) void k_fp4_append(const int* slots, int n_slots, int n_kv, const uint16_t* k, const uint16_t* v, long k_bs, long k_hs, long v_bs, long v_hs, int* lens,
                                                    int tiles, int cap, uint8_t* cache, int* errors) {
  const int b = blockIdx.x, slot = slots[b];
  if (slot < 0) return;
  bool again = false;      // a slot that an earlier row of the batch names: two tokens for one place
  for (int i = threadIdx.x; i < b; i += 256) again |= slots[i] == slot;
  const int len = slot < n_slots ? lens[slot] : 0;
  const bool full = (unsigned)len >= (unsigned)cap;      // (or below 0)
  const bool twice = __syncthreads_or(again);
  if (twice || slot >= n_slots || full) {      // (of a slot named twice the length may be raised by now: what is reported does not go by it)
    if (threadIdx.x == 0) atomicOr(errors, slot >= n_slots ? 4 : twice ? 2 : 1);
    return;
  }
  const int t = len & (TT - 1), s = t >> 4, m = t & 15, g = (t >> 2) & 3, i = t & 3;
  for (int at = threadIdx.x; at < n_kv * 32; at += 256) {
    const int u = at & 15, kind = at >> 4 & 1, head = at >> 5;
    const u4 x = *reinterpret_cast<const u4*>((kind ? v + b * v_bs + head * v_hs : k + b * k_bs + head * k_hs) + 8 * u);
    unsigned a = unit_max(x);
    a = pk_max(a, __shfl_xor(a, 1));
    a = pk_max(a, __shfl_xor(a, 2));
    const unsigned e = exponent_byte(a), w = encode_unit(x, scale_of(e));
    uint8_t* tile = cache + (((long)slot * n_kv + head) * tiles + len / TT) * TILE;
    *reinterpret_cast<unsigned*>(tile + 1024 * s + (kind ? V_AT + 16 * (16 * g + u) + 4 * i : 16 * (16 * (u >> 2) + m) + 4 * (u & 3))) = w;
    if ((u & 3) == 0) tile[kind ? VS_AT + 32 * (u >> 2) + 8 * g + 4 * s + i : KS_AT + 2 * (16 * (u >> 2) + m) + s] = (uint8_t)e;
  }
  if (threadIdx.x == 0) lens[slot] = len + 1;
}

// ---------------------------------------------------------------------------------------------------- attention
// How the rows' tiles are shared out: split p of a kv head takes tiles [first, end) of row `row`.  Every row is cut into splits of `size` tiles, size being
// the smallest that needs no more than P splits in all, so that long rows get many splits and short ones a single one.  All of it is computed by each wave
// from the lengths on the device.
struct Share { int row, len, slot, first, end, index, count; };      // row < 0: nothing for this split

__device__ __forceinline__ int row_len(const int* lens, int n_slots, int cap, int slot) { return slot >= 0 && slot < n_slots ? max(min(lens[slot], cap), 0) : 0; }      // (lens is the caller's to write)
// Sums over the wave in the vector unit (rows of 16 by shifts, then across rows), not through LDS: a lane exchange there takes ten times as long.
template <int CTRL, int ROWS> __device__ __forceinline__ int moved(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int wave_scan(int x) {      // inclusive
  x += moved<0x111, 0xf>(x); x += moved<0x112, 0xf>(x); x += moved<0x114, 0xf>(x); x += moved<0x118, 0xf>(x);      // row_shr 1, 2, 4, 8
  x += moved<0x142, 0xa>(x); x += moved<0x143, 0xc>(x);                                                            // row_bcast 15, 31
  return x;
}
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }
__device__ __forceinline__ int splits_of(int tiles, int size) { return (tiles + size - 1) / size; }

__device__ __forceinline__ int split_size(const int* slots, const int* lens, int n_slots, int cap, int B, int P) {
  const int l = threadIdx.x & 63;
  int total = 0, mine = 0;
  for (int b = l; b < B; b += 64) total += mine = (row_len(lens, n_slots, cap, slots[b]) + TT - 1) / TT;
  if (B == 1) return max((__builtin_amdgcn_readfirstlane(total) + P - 1) / P, 1);
  total = wave_sum(total);
  int lo = max((total + P - 1) / P, 1), hi = P > B ? max((total + P - B - 1) / (P - B), lo) : max(total, 1);
  if (B > 64) return hi;      // sum of ceil(t / hi) < total / hi + B <= P
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (wave_sum(splits_of(mine, mid)) <= P) hi = mid; else lo = mid + 1;
  }
  return hi;
}

__device__ __forceinline__ Share share_of(const int* slots, const int* lens, int n_slots, int cap, int B, int size, int p) {
  const int l = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    const int b = b0 + l, slot = b < B ? slots[b] : -1, len = row_len(lens, n_slots, cap, slot), n = splits_of((len + TT - 1) / TT, size);
    const int run = wave_scan(n);
    const unsigned long long here = __ballot(n > 0 && p >= before + run - n && p < before + run);
    if (here) {
      const int src = __builtin_ctzll(here);
      const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, src); };
      Share s;
      s.row = b0 + src; s.len = of(len); s.slot = of(slot); s.count = of(n); s.index = p - (before + of(run) - s.count);
      s.first = s.index * size; s.end = min(s.first + size, (s.len + TT - 1) / TT);
      return s;
    }
    before += __builtin_amdgcn_readlane(run, 63);
  }
  return Share{-1, 0, 0, 0, 0, 0, 0};
}

// The output of a row without tokens is 0, of one whose slot the cache does not have NaN.
__device__ __forceinline__ void empty_row(const int* slots, int n_slots, int row, int kvh, int n_kv, int G, uint16_t* out) {
  for (int i = threadIdx.x; i < G * DIM; i += 64 * NW) out[((long)row * n_kv + kvh) * G * DIM + i] = slots[row] >= n_slots ? 0x7fc0 : 0;
}

__device__ __forceinline__ float bits(unsigned x) { return __builtin_bit_cast(float, x); }

struct Tile { u4 k[2], v[2]; unsigned ks; u2 vs; };

__device__ __forceinline__ Tile load_tile(const uint8_t* t, unsigned l) {
  unsigned ks = KS_AT + 2 * l, vs = VS_AT + 32 * ((l & 15) >> 2) + 8 * (l >> 4), at = 16 * l;
  asm("" : "+v"(ks), "+v"(vs), "+v"(at));      // 32-bit offsets from the wave's address, here and not as 64-bit ones that live through the loop
  Tile x;
  x.ks = __builtin_nontemporal_load(reinterpret_cast<const uint16_t*>(t + ks));
  x.vs = __builtin_nontemporal_load(reinterpret_cast<const u2*>(t + vs));
  for (int s = 0; s < 2; ++s) x.k[s] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(t + at + 1024 * s));
  for (int s = 0; s < 2; ++s) x.v[s] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(t + at + V_AT + 1024 * s));
  return x;
}

// A query head as two operands of the scaled product, in the 8-bit type with 4 bits of mantissa: q = 2^E (hi + lo / 16), |hi| in [0, 256].  q has 8 bits: hi
// takes 4 of them and lo the other 4, exactly; what is smaller than 2^-13 of the head's maximum keeps 2^-21 of that at least.  Lane 16 g + n has channels 16 g ..
// and 64 + 16 g .. of head n (the operand's order); hi_exp and lo_exp are exponent bytes, 255 (NaN) where q is not finite.
struct Query { i8 hi, lo; unsigned hi_exp, lo_exp; };

// The maximum needs all of a head's channels, the conversion of the lane's eight dwords is shared out over the block's eight waves, one each (`halves`: in LDS; one barrier): by each wave
// for itself it took more instructions than two tiles (1000 tokens x 8 heads 7.3 us, so 6.5; 32 rows of 300..6000 24.1, 23.2; 65536 x 8 18.0,
// 17.2; all with weights of one bf16 number).
struct RawQuery { u4 x[4]; u2 own; };
__device__ __forceinline__ RawQuery load_query(const uint16_t* q, bool there, int g, int w) {
  RawQuery r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.x[i] = there ? *reinterpret_cast<const u4*>(q + 64 * (i >> 1) + 16 * g + 8 * (i & 1)) : u4{0, 0, 0, 0};
  r.own = there ? *reinterpret_cast<const u2*>(q + 64 * (w >> 2) + 16 * g + 4 * (w & 3)) : u2{0, 0};
  return r;
}
__device__ __forceinline__ Query convert_query(const RawQuery& raw, int w, bool negative, u2 (*halves)[64]) {
  const int l = threadIdx.x & 63;
  const u4 (&x)[4] = raw.x;
  const u2 own = raw.own;
  unsigned a = pk_max(pk_max(unit_max(x[0]), unit_max(x[1])), pk_max(unit_max(x[2]), unit_max(x[3])));
  a = pk_max(a, __shfl_xor(a, 16));
  a = pk_max(a, __shfl_xor(a, 32));
  a = max(a & 0xffffu, a >> 16);
  const unsigned e = (unsigned)max((int)(a >> 7) - 7, 5);
  const float down = bits((254 - e) << 23) * (negative ? -1.f : 1.f);      // +-2^-E
  int hi = 0, lo = 0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float a0 = bits(own[k] << 16) * down, a1 = bits(own[k] & 0xffff0000u) * down;
    const int h = __builtin_amdgcn_cvt_pk_fp8_f32(a0, a1, 0, false);
    const float l0 = (a0 - __builtin_amdgcn_cvt_f32_fp8(h, 0)) * 16.f, l1 = (a1 - __builtin_amdgcn_cvt_f32_fp8(h, 1)) * 16.f;
    const int o = __builtin_amdgcn_cvt_pk_fp8_f32(l0, l1, 0, false);
    hi |= (h & 0xffff) << 16 * k; lo |= (o & 0xffff) << 16 * k;
  }
  halves[w][l] = u2{(unsigned)hi, (unsigned)lo};
  __syncthreads();
  Query r;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const u2 v = halves[c][l];
    r.hi[c] = (int)v[0]; r.lo[c] = (int)v[1];
  }
  r.hi_exp = a >= 0x7f80u ? 255 : e; r.lo_exp = a >= 0x7f80u ? 255 : e - 4;
  return r;
}

// Online softmax of a wave: lane 16 g + n holds query head n.  max2 is in units of log2 and common to the four lanes of a head; sum is the lane's own tokens'.
struct Running { float max2, sum; f4 o[8]; };      // o[j][r]: channel 32 g + 8 r + j

// Channels 8 m + 2 c and 8 m + 2 c + 1 of the lane's eight tokens: pairs of channels of one token become pairs of tokens of one channel.  Weights: p + rest.
template <int C> __device__ __forceinline__ void attend_pair(Running& r, const u4 (&v)[2], const float (&sc)[8], bf8 p, bf8 rest) {
  unsigned x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v[i >> 2][i & 3], sc[i], C));
  u4 a, b;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x05040100u);
    b[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x07060302u);
  }
  r.o[2 * C] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), rest, r.o[2 * C], 0, 0, 0);
  r.o[2 * C + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, b), rest, r.o[2 * C + 1], 0, 0, 0);
  r.o[2 * C] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), p, r.o[2 * C], 0, 0, 0);
  r.o[2 * C + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, b), p, r.o[2 * C + 1], 0, 0, 0);
}

// Scores: C = K Q^T, 16 tokens x 16 heads, all 128 channels in one scaled product for each half of Q; K goes in as it lies in the cache.  C's rows 4 g + r are the
// lane's tokens, which is the order that V's units have along the contraction of O = V^T P^T: the weights go from one product into the other in registers.
// A weight goes as two numbers of bf16, its rounding and what that leaves (2^-16 of it is lost): as one, off by up to 2^-8, it would show where values cancel.  The second
// products cost little (1000 tokens x 8 heads 6.55 -> 7.06 us, 32 rows of 300..6000 23.4 -> 24.1, 65536 x 8 and 16 rows of 4096..65536 the same), since a dot product of pairs takes what is left in
// one instruction.  The sum of the weights and the output are held in 32 bits.  The maximum is only raised where a score exceeds it by 2^8, so that the accumulators are rarely scaled.
template <bool LAST> __device__ __forceinline__ void attend_tile(Running& r, const Tile& t, const Query& q, float scale2, int valid, int g) {
  f4 s[2];
  const i8 k0 = {(int)t.k[0][0], (int)t.k[0][1], (int)t.k[0][2], (int)t.k[0][3], 0, 0, 0, 0}, k1 = {(int)t.k[1][0], (int)t.k[1][1], (int)t.k[1][2], (int)t.k[1][3], 0, 0, 0, 0};
  s[0] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k0, q.lo, f4{0, 0, 0, 0}, 4, 0, 0, t.ks, 0, q.lo_exp);      // 4: E2M1, 0: E4M3; byte 0 of ks
  s[1] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k1, q.lo, f4{0, 0, 0, 0}, 4, 0, 1, t.ks, 0, q.lo_exp);      // byte 1
  s[0] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k0, q.hi, s[0], 4, 0, 0, t.ks, 0, q.hi_exp);
  s[1] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k1, q.hi, s[1], 4, 0, 1, t.ks, 0, q.hi_exp);
  float d[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) d[i] = __builtin_fmaf(s[i >> 2][i & 3], scale2, -r.max2);
  u4 v[2] = {t.v[0], t.v[1]};
  u2 vs = t.vs;
  unsigned dead = 0;
  if constexpr (LAST) {      // tokens behind the end: no weight, and nothing that an earlier sequence left in their place (it may be NaN)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (16 * (i >> 2) + 4 * g + (i & 3) >= valid) {
        d[i] = -__builtin_inff(); dead |= 1u << i;
        v[i >> 2][i & 3] = 0; vs[i >> 2] &= ~(255u << 8 * (i & 3));
      }
  }
  float top = d[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) top = fmaxf(top, d[i]);
  if (__ballot(top > 8.f)) {
    float x = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < 8; ++i) x = fmaxf(x, dead >> i & 1 ? -__builtin_inff() : s[i >> 2][i & 3] * scale2);
    x = fmaxf(x, __shfl_xor(x, 16));
    x = fmaxf(fmaxf(x, __shfl_xor(x, 32)), r.max2);
    const float a = __builtin_amdgcn_exp2f(r.max2 - x);
    r.max2 = x; r.sum *= a;
#pragma unroll
    for (int j = 0; j < 8; ++j) r.o[j] *= a;
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = dead >> i & 1 ? -__builtin_inff() : __builtin_fmaf(s[i >> 2][i & 3], scale2, -x);
  }
  bf8 p, rest;
  unsigned minus_low = 0xbf80u, minus_high = 0xbf800000u;      // (-1, 0) and (0, -1)
  asm("" : "+s"(minus_low), "+s"(minus_high));      // (as an inline constant of this instruction the first would be the second)
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float w0 = __builtin_amdgcn_exp2f(d[i]), w1 = __builtin_amdgcn_exp2f(d[i + 1]);
    r.sum += w0; r.sum += w1;
    const bf2 both = {(__bf16)w0, (__bf16)w1};
    p[i] = both[0]; p[i + 1] = both[1];
    rest[i] = (__bf16)__builtin_amdgcn_fdot2_f32_bf16(both, pair(minus_low), w0, false); rest[i + 1] = (__bf16)__builtin_amdgcn_fdot2_f32_bf16(both, pair(minus_high), w1, false);
  }
  float sc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sc[i] = scale_of(vs[i >> 2], 8 * (i & 3));
  attend_pair<0>(r, v, sc, p, rest); attend_pair<1>(r, v, sc, p, rest); attend_pair<2>(r, v, sc, p, rest); attend_pair<3>(r, v, sc, p, rest);
}

constexpr int OROW = DIM + 4;      // LDS row of a head's accumulators

// Partials of split p, kv head and head of its G (`at` = (p * n_kv + kvh) * G + head): maximum and sum as one 64-bit word, and behind all of these DIM accumulators
// each.  They go to another block, maybe on another XCD: stored past the caches (agent scope), waited for, and read past them, which costs no write-back of a whole
// L2 as a release does (measured: 0.05 us a block, one after the other).
typedef unsigned long long u64;
template <typename T> __device__ __forceinline__ void put(T* p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename T> __device__ __forceinline__ T get(const T* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ float lane(float x, int i) { return bits(__builtin_amdgcn_readlane(__builtin_bit_cast(int, x), i)); }

constexpr int LINE = 32;      // tickets are a cache line apart: all blocks draw theirs at about the same time

// Adds up the `count` splits from p0 on of the G heads of a (row, kv head), in their order, by the whole block: two waves a head, a lane a channel.  All loads of the
// first 32 splits are in flight together (64K tokens x 8 heads, 32 splits: 2.3 us, against 3.8 in three dependent rounds).
__device__ void merge(const float* part, long acc_at, int p0, int count, int n_kv, int kvh, int G, uint16_t* out) {
  constexpr int AHEAD = 32, STEP = 8;
  const int l = threadIdx.x & 63;
#pragma unroll 1
  for (int h = __builtin_amdgcn_readfirstlane(threadIdx.x / DIM); h < G; h += 64 * NW / DIM) {
    const int ch = threadIdx.x % DIM;
    const long at = ((long)p0 * n_kv + kvh) * G + h, step = (long)n_kv * G;
    float top = -__builtin_inff(), sum = 0, o = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < count; i0 += AHEAD) {
      const int n = min(count - i0, AHEAD);
      const float* acc = part + acc_at + (at + i0 * step) * DIM + ch;
      float x[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; j += STEP)
        if (j < n) {
#pragma unroll
          for (int i = j; i < j + STEP; ++i) x[i] = get(acc + (unsigned)min(i, n - 1) * (unsigned)step * DIM);
        }
      const u64 ms = l < n ? get(reinterpret_cast<const u64*>(part) + at + (i0 + l) * step) : 0xff800000ull;
      float m = bits((unsigned)ms), t = m;
      for (int d = 32; d > 0; d >>= 1) t = fmaxf(t, __shfl_xor(t, d));
      t = fmaxf(t, top);
      const float before = i0 == 0 ? 0.f : __builtin_amdgcn_exp2f(top - t), w = __builtin_amdgcn_exp2f(m - t);
      top = t;
      float s = l < n ? w * bits((unsigned)(ms >> 32)) : 0.f;
      for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
      sum = sum * before + s;
      o *= before;
#pragma unroll
      for (int j = 0; j < AHEAD; j += STEP) {
        __builtin_amdgcn_sched_barrier(0);      // (weights in scalar registers: eight at a time)
        if (j < n) {
#pragma unroll
          for (int i = j; i < j + STEP; ++i) if (i < n) o += lane(w, i) * x[i];
        }
      }
    }
    out[h * DIM + ch] = __builtin_bit_cast(uint16_t, (__bf16)(o / sum));
  }
}

// Decode attention.  Bound by the read of the cache where rows are long: 16 rows of 4096..65536 tokens x 8 heads 101 us, 606 MB, 6.0 TB/s, the rate of a plain read of
// that size being 6.1; by the launch, the plan and the merge where the cache is short: 1 row of 65536 x 8 heads, 17.1 us, has its 71 MB after about 14 (2 to 2.6 of
// them launch and plan), leaves the partials within 1.5 and adds them up in 2.3; by instructions on few CUs (1000 x 8 heads, four tiles a wave, 7.1 us).  A wave has whole tiles, so what it needs comes in 6 loads
// of whole lines and no lane waits for another; one tile is in flight while another is worked on: 16 waves a CU, 68 KB of loads in flight on each.  Two tiles in
// flight by 8 waves a CU take the same 101 us there, but 1 us more on shorter rows, whose first tiles wait for the second ones.  Four waves a SIMD need 128 registers at most: it has 123.
// One block = eight waves = one split of one (row, kv head).  One split a row (P == B): the output is written here; otherwise a row with several splits leaves
// partials, and the block that draws the last of the (row, kv head)'s tickets adds them up and puts the tickets back (tickets NULL: k_fp4_merge does it).
__global__ __launch_bounds__(64 * NW, 4) void k_fp4_attn(const uint8_t* cache, const int* lens, const int* slots, int n_slots, int tiles, int cap, const uint16_t* q, int B, int n_kv, int G,
                                                         float scale, int P, float* part, unsigned* tickets, uint16_t* out) {
  extern __shared__ __attribute__((aligned(16))) float lds[];      // [NW][G][OROW] accumulators, [NW][16] maxima, [NW][16] sums
  const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = l & 15, g = l >> 4, kvh = blockIdx.x % n_kv, p = blockIdx.x / n_kv;
  Share sh;
  if (P == B) {
    sh.row = p; sh.slot = slots[p]; sh.len = row_len(lens, n_slots, cap, sh.slot); sh.first = 0; sh.end = (sh.len + TT - 1) / TT; sh.index = 0; sh.count = 1;
    if (sh.len == 0) {
      empty_row(slots, n_slots, p, kvh, n_kv, G, out);
      return;
    }
  } else {
    if (p < B && row_len(lens, n_slots, cap, slots[p]) == 0) empty_row(slots, n_slots, p, kvh, n_kv, G, out);
    sh = share_of(slots, lens, n_slots, cap, B, split_size(slots, lens, n_slots, cap, B, P), p);
    if (sh.row < 0) return;
  }
  const int row = __builtin_amdgcn_readfirstlane(sh.row), slot = __builtin_amdgcn_readfirstlane(sh.slot), len = __builtin_amdgcn_readfirstlane(sh.len);
  const int first = __builtin_amdgcn_readfirstlane(sh.first), end = __builtin_amdgcn_readfirstlane(sh.end), count = __builtin_amdgcn_readfirstlane(sh.count);
  const int p0 = p - __builtin_amdgcn_readfirstlane(sh.index);
  const uint8_t* base = cache + ((long)slot * n_kv + kvh) * tiles * TILE;
  const long q0 = ((long)row * n_kv + kvh) * G * DIM;
  // one tile in flight while another is worked on; behind the end the last one is read again and left alone
  const auto tile = [&](int t) { return load_tile(base + (long)min(t, end - 1) * TILE, l); };
  int t = first + w;
  const RawQuery raw = load_query(q + q0 + n * DIM, n < G, g, w);
  asm volatile("" ::: "memory");      // (the query first: the tile is still on its way while it is converted)
  Tile x = tile(t);
  __shared__ u2 halves[NW][64];
  const Query qr = convert_query(raw, w, scale < 0, halves);
  const float scale2 = fabsf(scale) * 1.44269504f;
  Running r;
  r.max2 = -__builtin_inff(); r.sum = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) r.o[j] = f4{0, 0, 0, 0};
  const int full = min(len / TT, end);      // a tile with tokens behind the row's end comes last
  while (t < full) {
    const Tile y = tile(t + NW);
    attend_tile<false>(r, x, qr, scale2, TT, g);
    t += NW;
    if (t >= full) { x = y; break; }
    x = tile(t + NW);
    attend_tile<false>(r, y, qr, scale2, TT, g);
    t += NW;
  }
  if (t < end) attend_tile<true>(r, x, qr, scale2, len - t * TT, g);
  r.sum += __shfl_xor(r.sum, 16);
  r.sum += __shfl_xor(r.sum, 32);
  float *acc = lds, *mx = lds + NW * G * OROW, *sm = mx + NW * 16;
  if (n < G) {
#pragma unroll
    for (int rr = 0; rr < 4; ++rr)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<f4*>(acc + (w * G + n) * OROW + 32 * g + 8 * rr + 4 * h) = f4{r.o[4 * h][rr], r.o[4 * h + 1][rr], r.o[4 * h + 2][rr], r.o[4 * h + 3][rr]};
    if (g == 0) { mx[w * 16 + n] = r.max2; sm[w * 16 + n] = r.sum; }
  }
  __syncthreads();
  const long acc_at = 2l * P * n_kv * G;
  #pragma unroll 1
  for (int i = threadIdx.x; i < G * DIM; i += 64 * NW) {
    const int h = i / DIM, ch = i % DIM;
    float top = mx[h];
    for (int k = 1; k < NW; ++k) top = fmaxf(top, mx[k * 16 + h]);
    float o = 0, sum = 0;
    for (int k = 0; k < NW; ++k) {
      const float f = __builtin_amdgcn_exp2f(mx[k * 16 + h] - top);
      o += f * acc[(k * G + h) * OROW + ch]; sum += f * sm[k * 16 + h];
    }
    if (count == 1) out[q0 + i] = __builtin_bit_cast(uint16_t, (__bf16)(o / sum));
    else {
      const long at = ((long)p * n_kv + kvh) * G + h;
      put(part + acc_at + at * DIM + ch, o);
      if (ch == 0) put(reinterpret_cast<u64*>(part) + at, (u64)__builtin_bit_cast(unsigned, sum) << 32 | __builtin_bit_cast(unsigned, top));
    }
  }
  if (count == 1 || tickets == nullptr) return;
  unsigned* ticket = tickets + ((long)row * n_kv + kvh) * LINE;
  __shared__ int last;
  stores_done();
  __syncthreads();
  if (threadIdx.x == 0) {
    last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)count - 1;
    if (last) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (last) merge(part, acc_at, p0, count, n_kv, kvh, G, out + q0);
}

// The same merge as a launch of its own: a block per (row, kv head); rows without or with a single split are done already.
__global__ __launch_bounds__(64 * NW) void k_fp4_merge(const float* part, const int* lens, const int* slots, int n_slots, int cap, int B, int n_kv, int G, int P, uint16_t* out) {
  const int row = blockIdx.x / n_kv, kvh = blockIdx.x % n_kv, l = threadIdx.x & 63;
  const int len = row_len(lens, n_slots, cap, slots[row]), size = split_size(slots, lens, n_slots, cap, B, P), count = splits_of((len + TT - 1) / TT, size);
  if (count <= 1) return;
  int first = 0;
  for (int b = l; b < row; b += 64) first += splits_of((row_len(lens, n_slots, cap, slots[b]) + TT - 1) / TT, size);
  merge(part, 2l * P * n_kv * G, wave_sum(first), count, n_kv, kvh, G, out + (long)blockIdx.x * G * DIM);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

extern "C" {

int gaac_fp4_store(const void* k, const void* v, long k_head_stride, long k_row_stride, long v_head_stride, long v_row_stride, int L, int n_kv, int tiles, uint8_t* cache, int* len, void* stream) {
  GAAC_REQUIRE(cache != nullptr && len != nullptr && (L == 0 || (k != nullptr && v != nullptr)), "gaac_fp4_store: null pointer");
  GAAC_REQUIRE(n_kv > 0 && n_kv <= 65535 && tiles > 0 && L >= 0 && L <= (long)tiles * TT, "gaac_fp4_store: bad sizes (n_kv %d, %d tokens, %d tiles of %d)", n_kv, L, tiles, TT);
  GAAC_REQUIRE(aligned16(k) && aligned16(v) && aligned16(cache) && (k_head_stride | k_row_stride | v_head_stride | v_row_stride) % 8 == 0, "gaac_fp4_store: rows must be 16-byte aligned");
  k_fp4_store<<<dim3(L > 0 ? (L + 4 * TT - 1) / (4 * TT) : 1, n_kv, 2), 256, 0, (hipStream_t)stream>>>((const uint16_t*)k, (const uint16_t*)v, k_head_stride, k_row_stride, v_head_stride, v_row_stride, L, tiles,
                                                                                                    cache, len);
  return gaac::launch_status("gaac_fp4_store");
}

int gaac_fp4_load(const uint8_t* cache, int L, int n_kv, int tiles, void* k, void* v, long k_head_stride, long k_row_stride, long v_head_stride, long v_row_stride, void* stream) {
  GAAC_REQUIRE(cache != nullptr && k != nullptr && v != nullptr, "gaac_fp4_load: null pointer");
  GAAC_REQUIRE(n_kv > 0 && n_kv <= 65535 && tiles > 0 && L > 0 && L <= (long)tiles * TT, "gaac_fp4_load: bad sizes (n_kv %d, %d tokens, %d tiles of %d)", n_kv, L, tiles, TT);
  GAAC_REQUIRE(aligned16(k) && aligned16(v) && aligned16(cache) && (k_head_stride | k_row_stride | v_head_stride | v_row_stride) % 8 == 0, "gaac_fp4_load: rows must be 16-byte aligned");
  k_fp4_load<<<dim3((L + 4 * TT - 1) / (4 * TT), n_kv, 2), 256, 0, (hipStream_t)stream>>>(cache, L, tiles, (uint16_t*)k, (uint16_t*)v, k_head_stride, k_row_stride, v_head_stride, v_row_stride);
  return gaac::launch_status("gaac_fp4_load");
}

int gaac_fp4_length(const int* len, int tiles, int* host, void* stream) {
  GAAC_REQUIRE(len != nullptr && host != nullptr && tiles > 0 && tiles <= INT_MAX / TT, "gaac_fp4_length: bad arguments (%d tiles)", tiles);
  __atomic_store_n(host, -1, __ATOMIC_RELAXED);      // not there yet
  k_fp4_length<<<1, 1, 0, (hipStream_t)stream>>>(len, tiles * TT, host);
  return gaac::launch_status("gaac_fp4_length");
}

int gaac_fp4_append(const int* slots, int B, int n_slots, int n_kv, const void* k, const void* v, long k_batch_stride, long k_head_stride, long v_batch_stride, long v_head_stride, int* lens, int tiles, int cap,
                    uint8_t* cache, int* errors, void* stream) {
  GAAC_REQUIRE(slots != nullptr && k != nullptr && v != nullptr && lens != nullptr && cache != nullptr && errors != nullptr, "gaac_fp4_append: null pointer");
  GAAC_REQUIRE(B > 0 && B < 1 << 24 && n_slots > 0 && n_kv > 0 && n_kv < 1 << 24 && tiles > 0 && cap > 0 && cap <= (long)tiles * TT, "gaac_fp4_append: bad sizes (B %d, n_slots %d, n_kv %d, capacity %d in %d tiles)", B, n_slots,
               n_kv, cap, tiles);
  GAAC_REQUIRE(aligned16(k) && aligned16(v) && aligned16(cache) && (k_batch_stride | k_head_stride | v_batch_stride | v_head_stride) % 8 == 0, "gaac_fp4_append: rows must be 16-byte aligned");
  k_fp4_append<<<B, 256, 0, (hipStream_t)stream>>>(slots, n_slots, n_kv, (const uint16_t*)k, (const uint16_t*)v, k_batch_stride, k_head_stride, v_batch_stride, v_head_stride, lens, tiles, cap, cache, errors);
  return gaac::launch_status("gaac_fp4_append");
}

int gaac_fp4_attn(const uint8_t* cache, const int* lens, const int* slots, int n_slots, int tiles, int cap, const void* q, int B, int n_q, int n_kv, float scale, int nsplit, float* partials, unsigned* tickets, void* out,
                  void* stream) {
  GAAC_REQUIRE(cache != nullptr && lens != nullptr && slots != nullptr && q != nullptr && out != nullptr, "gaac_fp4_attn: null pointer");
  GAAC_REQUIRE(B > 0 && n_slots > 0 && n_kv > 0 && n_kv <= 65535 && n_q >= n_kv && n_q % n_kv == 0 && n_q / n_kv <= 16, "gaac_fp4_attn: GQA group size must be 1..16 (n_q %d, n_kv %d)", n_q, n_kv);
  GAAC_REQUIRE(tiles > 0 && cap > 0 && cap <= (long)tiles * TT && nsplit > 0 && (long)B * nsplit * n_kv < (1l << 32) / (64 * NW) && (long)B * n_q < 1l << 31, "gaac_fp4_attn: bad sizes (B %d, capacity %d in %d tiles, %d splits)", B,
               cap, tiles, nsplit);
  GAAC_REQUIRE(nsplit == 1 || (partials != nullptr && reinterpret_cast<uintptr_t>(partials) % 8 == 0), "gaac_fp4_attn: more than one split needs partials, 8-byte aligned");
  GAAC_REQUIRE(aligned16(q) && aligned16(cache), "gaac_fp4_attn: q must be 16-byte aligned");
  // The plan adds up the rows' tiles in 32 bits; a batch whose rows could come to more has blocks enough without splits.
  const bool splits = nsplit > 1 && (long)B * tiles + (long)B * nsplit < 1l << 30;
  const int G = n_q / n_kv, P = splits ? B * nsplit : B;
  const int lds = 4 * (NW * G * OROW + 2 * NW * 16);
  if (lds > 60 * 1024) {      // (with the 4 KB that the kernel has by itself more than the 64 that need no asking)
    const hipError_t e = hipFuncSetAttribute((const void*)k_fp4_attn, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) { gaac::fail("gaac_fp4_attn: %s", hipGetErrorString(e)); return (int)e; }
  }
  k_fp4_attn<<<P * n_kv, 64 * NW, lds, (hipStream_t)stream>>>(cache, lens, slots, n_slots, tiles, cap, (const uint16_t*)q, B, n_kv, G, scale, P, partials, tickets, (uint16_t*)out);
  const int rc = gaac::launch_status("gaac_fp4_attn");
  if (rc != 0 || P == B || tickets != nullptr) return rc;
  k_fp4_merge<<<B * n_kv, 64 * NW, 0, (hipStream_t)stream>>>(partials, lens, slots, n_slots, cap, B, n_kv, G, P, (uint16_t*)out);
  return gaac::launch_status("gaac_fp4_attn (merge)");
}

}  // extern "C"
