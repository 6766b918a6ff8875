// Norms of queries and keys for each head and their rotation, in one pass over both.
//   y = x * rsqrt(mean(x^2) + eps) * w over the head's D channels (no weights: y = x), then for each pair p < R/2 of the first R channels
//   (y1 cos - y2 sin, y2 cos + y1 sin), the pair being (p, p + R/2), or (2p, 2p + 1) if interleaved; cos and sin are row `position` of tables.
// Bound by HBM for a prompt (each element read once and written once: 16384 tokens x 40 heads of 128 channels in bf16, 344 MB, 67 us, 5.1 TB/s, where a large copy
// makes 4.7), by the launch for a decode step (4 tokens x 40 heads: 3.3 us, of which an empty launch takes 1.6; 777 x 28: 5.3).  A lane holds 16 channels of a head, two runs of 8 that
// make whole pairs, so nothing but the sum of squares goes between lanes: D / 16 lanes a head, 16-byte loads.  A wave keeps to one token and goes through
// its heads, the lane's cos and sin staying in registers.  Arithmetic in 32 bits, one rounding at the end; products are not fused into the sums of the
// rotation, so that without weights a result is bit for bit what separate multiplications and additions in 32 bits give.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "gaac_capi.h"
#include "../../include/gaac_hip.h"

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

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

struct Args {
  const void *q, *k, *wq, *wk, *pos;
  void *qo, *ko;
  const float *cos, *sin;
  long q_ts, q_hs, k_ts, k_hs, wq_hs, wk_hs, N;
  int n_q, n_k, R, max_pos, parts, pos64;
  float eps;
};

// A wave: one token, heads part * HPW + h, then steps of parts * HPW.
template <typename T, int D, bool INTERLEAVED, bool NORM>
__global__ __launch_bounds__(256) void k_norm_rope(Args a) {
#pragma clang fp contract(off)
  constexpr int LPH = D / 16, HPW = 64 / LPH;
  const long wave = (long)blockIdx.x * 4 + (threadIdx.x >> 6), token = wave / a.parts;
  if (token >= a.N) return;
  const int part = wave % a.parts, l = threadIdx.x & 63, j = l % LPH, half = a.R / 2, heads = a.n_q + a.n_k;
  const long pos = a.pos64 ? static_cast<const long*>(a.pos)[token] : static_cast<const int*>(a.pos)[token];
  const bool rotated = j < a.R / 16, inside = pos >= 0 && pos < a.max_pos;
  const int c0 = rotated ? 8 * j : a.R + 16 * (j - a.R / 16), c1 = rotated ? c0 + half : c0 + 8;      // first channels of the lane's two runs
  float cs[8], sn[8];
  if (rotated && inside) {      // 8 pairs: of both runs together, or the first run's four and the second's
    const float *c = a.cos + pos * half, *s = a.sin + pos * half;
    if constexpr (INTERLEAVED) {
      const f4 ca = *reinterpret_cast<const f4*>(c + c0 / 2), cb = *reinterpret_cast<const f4*>(c + c1 / 2), sa = *reinterpret_cast<const f4*>(s + c0 / 2), sb = *reinterpret_cast<const f4*>(s + c1 / 2);
      for (int i = 0; i < 4; ++i) { cs[i] = ca[i]; cs[4 + i] = cb[i]; sn[i] = sa[i]; sn[4 + i] = sb[i]; }
    } else {
      load8(c + c0, cs);
      load8(s + c0, sn);
    }
  } else {      // a position that the tables do not have: NaN
    const float one = inside ? 1.f : __builtin_nanf("");
    for (int i = 0; i < 8; ++i) { cs[i] = one; sn[i] = 0.f; }
  }
  for (int h = part * HPW + l / LPH; h < heads; h += a.parts * HPW) {
    const bool is_q = h < a.n_q;
    const int hh = is_q ? h : h - a.n_q;
    const T* src = is_q ? static_cast<const T*>(a.q) + token * a.q_ts + hh * a.q_hs : static_cast<const T*>(a.k) + token * a.k_ts + hh * a.k_hs;
    T* dst = is_q ? static_cast<T*>(a.qo) + (token * a.n_q + hh) * D : static_cast<T*>(a.ko) + (token * a.n_k + hh) * D;
    float x[8], y[8];
    load8(src + c0, x);
    load8(src + c1, y);
    if constexpr (NORM) {
      const T* w = is_q ? static_cast<const T*>(a.wq) + hh * a.wq_hs : static_cast<const T*>(a.wk) + hh * a.wk_hs;
      float wx[8], wy[8], sum = 0;
      load8(w + c0, wx);
      load8(w + c1, wy);
      for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(x[i], x[i], __builtin_fmaf(y[i], y[i], sum));
      for (int o = LPH / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
      const float r = 1.f / __builtin_sqrtf(sum * (1.f / D) + a.eps);
      for (int i = 0; i < 8; ++i) { x[i] = x[i] * r * wx[i]; y[i] = y[i] * r * wy[i]; }
    }
    if (rotated) {
      if constexpr (INTERLEAVED) {
        for (int i = 0; i < 4; ++i) {
          const float x0 = x[2 * i], x1 = x[2 * i + 1], y0 = y[2 * i], y1 = y[2 * i + 1];
          x[2 * i] = x0 * cs[i] - x1 * sn[i]; x[2 * i + 1] = x1 * cs[i] + x0 * sn[i];
          y[2 * i] = y0 * cs[4 + i] - y1 * sn[4 + i]; y[2 * i + 1] = y1 * cs[4 + i] + y0 * sn[4 + i];
        }
      } else {
        for (int i = 0; i < 8; ++i) {
          const float x0 = x[i], y0 = y[i];
          x[i] = x0 * cs[i] - y0 * sn[i]; y[i] = y0 * cs[i] + x0 * sn[i];
        }
      }
    } else if (!inside) {
      for (int i = 0; i < 8; ++i) { x[i] = cs[i]; y[i] = cs[i]; }
    }
    store8(dst + c0, x);
    store8(dst + c1, y);
  }
}

template <typename T, int D> void launch(const Args& a, bool interleaved, bool norm, hipStream_t stream) {
  const unsigned grid = (unsigned)((a.N * a.parts + 3) / 4);
  if (norm) {
    if (interleaved) k_norm_rope<T, D, true, true><<<grid, 256, 0, stream>>>(a); else k_norm_rope<T, D, false, true><<<grid, 256, 0, stream>>>(a);
  } else {
    if (interleaved) k_norm_rope<T, D, true, false><<<grid, 256, 0, stream>>>(a); else k_norm_rope<T, D, false, false><<<grid, 256, 0, stream>>>(a);
  }
}
template <typename T> void launch(const Args& a, int D, bool interleaved, bool norm, hipStream_t stream) {
  if (D == 64) launch<T, 64>(a, interleaved, norm, stream);
  else if (D == 128) launch<T, 128>(a, interleaved, norm, stream);
  else launch<T, 256>(a, interleaved, norm, stream);
}

}  // namespace

extern "C" int gaac_qk_norm_rope(int type, const void* q, const void* k, long q_token_stride, long q_head_stride, long k_token_stride, long k_head_stride, long N, int n_q, int n_k, int D, int R, const void* q_weight,
                                 const void* k_weight, long q_weight_stride, long k_weight_stride, float eps, const void* positions, int positions64, const float* cos, const float* sin, int max_pos,
                                 int interleaved, void* q_out, void* k_out, void* stream) {
  GAAC_REQUIRE(q != nullptr && k != nullptr && positions != nullptr && cos != nullptr && sin != nullptr && q_out != nullptr && k_out != nullptr, "gaac_qk_norm_rope: null pointer");
  GAAC_REQUIRE(type >= 0 && type <= 2, "gaac_qk_norm_rope: type must be 0 (bf16), 1 (fp16) or 2 (fp32)");
  GAAC_REQUIRE((D == 64 || D == 128 || D == 256) && R > 0 && R <= D && R % 16 == 0, "gaac_qk_norm_rope: head_dim must be 64, 128 or 256, and a multiple of 16 channels of it rotated (%d of %d)", R, D);
  GAAC_REQUIRE(N > 0 && n_q > 0 && n_k > 0 && max_pos > 0 && n_q < 1 << 20 && n_k < 1 << 20 && N < 1l << 26, "gaac_qk_norm_rope: bad sizes (%ld tokens, %d + %d heads, %d positions)", N, n_q, n_k, max_pos);
  GAAC_REQUIRE((q_weight == nullptr) == (k_weight == nullptr), "gaac_qk_norm_rope: weights for both or for neither");
  const uintptr_t all = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(cos) |
                        reinterpret_cast<uintptr_t>(sin) | reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight);
  GAAC_REQUIRE(all % 16 == 0 && (q_token_stride | q_head_stride | k_token_stride | k_head_stride | q_weight_stride | k_weight_stride) % (type == 2 ? 4 : 8) == 0, "gaac_qk_norm_rope: rows must be 16-byte aligned");
  const int groups = (n_q + n_k + 1024 / D - 1) / (1024 / D);      // of the 64 / (D/16) heads that a wave takes at a time
  Args a{q, k, q_weight, k_weight, positions, q_out, k_out, cos, sin, q_token_stride, q_head_stride, k_token_stride, k_head_stride, q_weight_stride, k_weight_stride, N, n_q, n_k, R, max_pos, groups, positions64 != 0, eps};
  // A wave for each group of heads until the chip is full twice over, then one that goes through a token's groups and reads cos and sin once (40 heads of 128 channels, us,
  // split / not: 4 tokens 2.8 / 5.2, 777 5.6 / 7.8, 2400 11.2 / 11.5, 4096 16.1 / 15.6, 16384 67.1 / 65.5).
  if (N * groups > 16384) a.parts = 1;
  const bool norm = q_weight != nullptr;
  if (type == 0) launch<__bf16>(a, D, interleaved != 0, norm, (hipStream_t)stream);
  else if (type == 1) launch<_Float16>(a, D, interleaved != 0, norm, (hipStream_t)stream);
  else launch<float>(a, D, interleaved != 0, norm, (hipStream_t)stream);
  return gaac::launch_status("gaac_qk_norm_rope");
}
