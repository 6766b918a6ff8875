// Python calls of the library's entry points (include/gaac_hip.h): gaac_amd._binding.<entry point>(arguments), raising RuntimeError with the
// library's message where an entry point returns non-zero.  Tensors are handed over as they are; a host tensor raises.  A function in the place of
// an address (the stream) is called for it once the arguments before it have been looked at: without a GPU, a host tensor is what the error names.
// What it is for: a launch has up to 47 arguments, half of them tensors.  Through ctypes, with is_cuda and data_ptr() called from Python for each
// tensor, attention() costs the host 14 us, more than the kernel takes over a short context, and a step of append and attention 24; with the
// arguments converted here 9 and 15, made here as a whole (below) 7 and 12.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <algorithm>
#include <exception>
#include <tuple>
#include <type_traits>
#include <utility>
#include "../../include/gaac_hip.h"

namespace {

const char* (*g_last_error)() = nullptr;

// One argument; false with a Python error set.  Numbers convert as ctypes converts them: anything with __index__, cut to the type's bits.
bool convert(PyObject* o, void*& v) {
  if (o == Py_None) { v = nullptr; return true; }
  if (THPVariable_Check(o)) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) {
      PyErr_SetString(PyExc_RuntimeError, "gaac_amd kernels need device tensors (got a CPU tensor): there is no CPU path");
      return false;
    }
    v = t.data_ptr();
    return true;
  }
  if (PyCallable_Check(o)) {
    PyObject* r = PyObject_CallNoArgs(o);
    const bool ok = r != nullptr && PyLong_Check(r) && convert(r, v);
    if (r != nullptr && !PyLong_Check(r)) PyErr_SetString(PyExc_TypeError, "expected a function that returns an address");
    Py_XDECREF(r);
    return ok;
  }
  if (!PyLong_Check(o)) { PyErr_Format(PyExc_TypeError, "expected a tensor, an address or None, got %s", Py_TYPE(o)->tp_name); return false; }
  v = reinterpret_cast<void*>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLongMask(o)));
  return !PyErr_Occurred();
}
bool convert(PyObject* o, long& v) {
  if (PyFloat_Check(o)) { PyErr_SetString(PyExc_TypeError, "expected an integer, got float"); return false; }
  v = static_cast<long>(PyLong_AsUnsignedLongMask(o));
  return v != -1 || !PyErr_Occurred();
}
bool convert(PyObject* o, int& v) {
  long l;
  if (!convert(o, l)) return false;
  v = static_cast<int>(l);
  return true;
}
bool convert(PyObject* o, float& v) {
  const double d = PyFloat_AsDouble(o);
  v = static_cast<float>(d);
  return d != -1.0 || !PyErr_Occurred();
}

template <typename A> using Held = std::conditional_t<std::is_pointer_v<A>, void*, A>;      // what an argument is converted to
template <typename A> A passed(Held<A> v) { if constexpr (std::is_pointer_v<A>) return static_cast<A>(v); else return v; }

template <typename... A, size_t... I>
PyObject* invoke(const char* name, int (*fn)(A...), PyObject* const* args, std::index_sequence<I...>) {
  std::tuple<Held<A>...> held;
  try {
    if (!(convert(args[I], std::get<I>(held)) && ...)) return nullptr;
  } catch (const std::exception& e) {      // a tensor without memory
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(passed<A>(std::get<I>(held))...);
  Py_END_ALLOW_THREADS
  if (rc != 0) {
    PyErr_Format(PyExc_RuntimeError, "%s failed (%d): %s", name, rc, g_last_error());
    return nullptr;
  }
  Py_RETURN_NONE;
}
template <typename... A>
PyObject* invoke(const char* name, int (*fn)(A...), PyObject* const* args, Py_ssize_t n) {
  if (fn == nullptr) { PyErr_SetString(PyExc_RuntimeError, "gaac_amd._binding.bind has not been called"); return nullptr; }
  if (n != static_cast<Py_ssize_t>(sizeof...(A))) {
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (%zd given)", name, static_cast<Py_ssize_t>(sizeof...(A)), n);
    return nullptr;
  }
  return invoke(name, fn, args, std::index_sequence_for<A...>{});
}

#define GAAC_ENTRY_POINTS(X)                                                                                                              \
  X(gaac_wait_words) X(gaac_page_finish) X(gaac_cache_check)                                                                              \
  X(gaac_exponent_hist) X(gaac_bases_from_hist) X(gaac_encode_tiles) X(gaac_compact) X(gaac_tile_scan) X(gaac_page_pack)                  \
  X(gaac_row_offsets) X(gaac_decode_tiles) X(gaac_prompt_store) X(gaac_cache_prefill) X(gaac_attn_split) X(gaac_attn_combine)             \
  X(gaac_cache_append)                                                                                                                    \
  X(gaac_paged_store) X(gaac_paged_free) X(gaac_paged_release) X(gaac_paged_decode) X(gaac_paged_attn) X(gaac_bf16_attn)                  \
  X(gaac_attn_fused) X(gaac_attn_fused_static) X(gaac_static_init) X(gaac_static_reset) X(gaac_static_flags) X(gaac_attn_launch)    \
  X(gaac_fp4_store) X(gaac_fp4_load) X(gaac_fp4_length) X(gaac_fp4_append) X(gaac_fp4_attn) X(gaac_qk_norm_rope) X(gaac_sample) \
  X(gaac_fp8_rows) X(gaac_fp8_values) X(gaac_fp8_product) X(gaac_fp8_product_form) X(gaac_logprobs)
#define X(name)                                            \
  decltype(&::name) p_##name = nullptr;                    \
  PyObject* py_##name(PyObject*, PyObject* const* args, Py_ssize_t n) { return invoke(#name, p_##name, args, n); }
GAAC_ENTRY_POINTS(X)
#undef X

// ---------------------------------------------------------------------------------------------------- whole calls
// What CompressedKVCache, Codec and attention() do on each call, where the arguments are what a program usually has: plain tensors on the device, in the
// layout that the kernels read.  None where they are not, before anything is launched: the Python code of the call, which has the checks and messages,
// takes over, as it does where there is no binding.  Host us a call, Python / here: attention 9.0 / 7.2, over the slot cache 8.5 / 6.9, append 6.2 / 4.8 (a launch
// alone takes 3), a page's decoder 5.4 / 4.3; 4096 tokens x 8 heads encoded and expanded again 37.9 / 30.2, a prompt of 777 tokens 21.7 / 18.4.
struct Otherwise {};      // thrown: not such arguments

struct Refs {             // objects that are held until the call has been made (another thread may replace an attribute meanwhile)
  PyObject* r[64];
  int n = 0;
  ~Refs() { while (n > 0) Py_DECREF(r[--n]); }
  PyObject* operator()(PyObject* o, PyObject* name) {
    PyObject* p = PyObject_GetAttr(o, name);
    if (p == nullptr) throw Otherwise{};
    return r[n++] = p;
  }
};
#define GAAC_NAMES(X)                                                                                                                        \
  X(k) X(v) X(sm) X(codes) X(flags) X(tile_off) X(ovf) X(head_start) X(ovf_head_start) X(base3) X(base4) X(tail) X(ovf_used) X(ovf_cap)     \
  X(n_kv) X(cap) X(S) X(H) X(kind) X(tail_len) X(overflow) X(n_slots) X(per_sequence_bases) X(_scan) X(pm) X(pl) X(pa) X(epoch) X(rows) X(nslot)                            \
  X(data) X(lens) X(tiles)
#define X(name) PyObject* n_##name = nullptr;
GAAC_NAMES(X)
#undef X

constexpr long DIM = 128, TILE = 16, CODE_BYTES = 48, TILE_ESCAPES = 1280, HIST_BYTES = 256 * 64 * 4 + 32;

const at::Tensor& tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) throw Otherwise{};
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda()) throw Otherwise{};
  return t;
}
template <typename P> P* address(PyObject* o) { return static_cast<P*>(tensor(o).data_ptr()); }
long number(PyObject* o) {
  if (!PyLong_CheckExact(o)) throw Otherwise{};
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw Otherwise{};
  return v;
}
void* stream_of(PyObject* o) {
  void* v = nullptr;
  if (!convert(o, v)) throw Otherwise{};
  return v;
}
bool is_rows(const at::Tensor& t, int dims) { return t.dim() == dims && t.scalar_type() == at::kBFloat16 && t.size(dims - 1) == DIM; }
// rows_in_place: whether the encoder can read the rows where they lie
bool in_place(const at::Tensor& t, int head_dim, int row_dim, long& hs, long& rs) {
  hs = t.size(head_dim) > 1 ? t.stride(head_dim) : 0;
  rs = t.size(row_dim) > 1 ? t.stride(row_dim) : DIM;
  return t.stride(2) == 1 && rs >= DIM && rs % 8 == 0 && hs % 8 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
at::Tensor bytes(const at::Tensor& like, at::IntArrayRef shape, at::ScalarType type = at::kByte) { return at::empty(shape, at::TensorOptions().dtype(type).device(like.device())); }
at::Tensor host_words(long n) { return at::empty({n}, at::TensorOptions().dtype(at::kInt).pinned_memory(true)); }

struct Failed { const char* name; int rc; };      // thrown: an entry point's refusal, with the GIL held
void must(const char* name, int rc) { if (rc != 0) throw Failed{name, rc}; }
template <typename F> PyObject* whole_call(Py_ssize_t given, Py_ssize_t n, F body) {
  if (given != n) { PyErr_Format(PyExc_TypeError, "expected %zd arguments (%zd given)", n, given); return nullptr; }
  if (p_gaac_wait_words == nullptr) { PyErr_SetString(PyExc_RuntimeError, "gaac_amd._binding.bind has not been called"); return nullptr; }
  try {
    return body();
  } catch (const Otherwise&) {
  } catch (const Failed& f) {
    PyErr_Format(PyExc_RuntimeError, "%s failed (%d): %s", f.name, f.rc, g_last_error());
    return nullptr;
  } catch (const std::exception&) {      // no memory, a tensor without any: Python meets the same and raises its own type (nothing is stored until a call's last launch)
  }
  PyErr_Clear();
  Py_RETURN_NONE;
}
struct NoGil {      // (taken back also where an exception leaves: a tensor without an address of its own, as in vmap)
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};
template <typename F> int without_gil(F f) {
  const NoGil released;
  return f();
}
PyObject* numbers(const at::Tensor& words) {
  const long n = words.numel();
  const int* w = static_cast<const int*>(words.data_ptr());
  PyObject* l = PyList_New(n);
  for (long i = 0; l != nullptr && i < n; ++i) {
    PyObject* o = PyLong_FromLong(w[i]);
    if (o == nullptr) { Py_DECREF(l); return nullptr; }
    PyList_SET_ITEM(l, i, o);
  }
  return l;
}

// attend(K, V, n_kv, ws, q, slots or None, SL or None, S_pad, scale, nsplit, tail_len or None, S_all, stream) -> out like q [B, n_q, 128]
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 13, [&]() -> PyObject* {
    Refs get;
    const at::Tensor& q = tensor(a[4]);
    const long n_kv = number(a[2]), S_pad = number(a[7]), nsplit = number(a[9]), S_all = number(a[11]);
    if (!is_rows(q, 3) || !q.is_contiguous() || n_kv <= 0 || q.size(1) % n_kv != 0 || q.size(1) < n_kv || q.size(1) / n_kv > 16 || !PyFloat_CheckExact(a[8])) throw Otherwise{};
    const long B = q.size(0), n_q = q.size(1);
    const bool tail = a[10] != Py_None;
    const int* slots = nullptr;
    if (a[5] != Py_None) {
      const at::Tensor& s = tensor(a[5]);
      if (s.dim() != 1 || s.size(0) != B || s.scalar_type() != at::kInt || !s.is_contiguous()) throw Otherwise{};
      slots = static_cast<const int*>(s.data_ptr());
    }
    if (number(get(a[3], n_rows)) != B * n_q || number(get(a[3], n_nslot)) != nsplit || B == 0) throw Otherwise{};
    struct Store { uint8_t *sm, *cd; int *fl, *to; uint8_t* ov; int* hs; uint8_t *b3, *b4; void* tail; long nb; } st[2];
    for (int i = 0; i < 2; ++i) {
      PyObject* o = a[i];
      Store& s = st[i];
      s.sm = address<uint8_t>(get(o, n_sm)); s.cd = address<uint8_t>(get(o, n_codes)); s.fl = address<int>(get(o, n_flags)); s.to = address<int>(get(o, n_tile_off));
      s.ov = address<uint8_t>(get(o, n_ovf)); s.hs = address<int>(get(o, tail ? n_head_start : n_ovf_head_start));
      PyObject* b3 = get(o, n_base3);
      s.nb = tensor(b3).size(0); s.b3 = address<uint8_t>(b3); s.b4 = address<uint8_t>(get(o, n_base4));
      s.tail = tail ? address<void>(get(o, n_tail)) : nullptr;
    }
    const int* SL = a[6] == Py_None ? nullptr : address<int>(a[6]);
    const int* TL = tail ? address<int>(a[10]) : nullptr;
    auto *pm = address<unsigned long long>(get(a[3], n_pm)), *pl = address<unsigned long long>(get(a[3], n_pl)), *pa = address<unsigned long long>(get(a[3], n_pa));
    unsigned* epoch = address<unsigned>(get(a[3], n_epoch));
    const float scale = static_cast<float>(PyFloat_AS_DOUBLE(a[8]));
    void* stream = stream_of(a[12]);
    at::Tensor out = bytes(q, {B, n_q, DIM}, at::kBFloat16);
    must("gaac_attn_fused", without_gil([&] {
      return p_gaac_attn_fused(st[0].sm, st[0].cd, st[0].fl, st[0].to, st[0].ov, st[0].hs, st[0].b3, st[0].b4, st[1].sm, st[1].cd, st[1].fl, st[1].to, st[1].ov, st[1].hs,
                               st[1].b3, st[1].b4, q.data_ptr(), slots, static_cast<int>(B), static_cast<int>(n_q), static_cast<int>(n_kv), SL, static_cast<int>(S_pad), scale,
                               static_cast<int>(nsplit), static_cast<int>(st[0].nb), st[0].tail, st[1].tail, TL, tail ? static_cast<int>(TILE) : 0, static_cast<int>(S_all), pm, pl, pa,
                               epoch, out.data_ptr(), stream);
    }));
    return THPVariable_Wrap(out);
  });
}

struct CacheStore { void* tail; uint8_t *b3, *b4, *sm, *cd; int* fl; uint8_t* ov; int *to, *used; };
CacheStore cache_store(Refs& get, PyObject* o) {
  return {address<void>(get(o, n_tail)), address<uint8_t>(get(o, n_base3)), address<uint8_t>(get(o, n_base4)), address<uint8_t>(get(o, n_sm)), address<uint8_t>(get(o, n_codes)),
          address<int>(get(o, n_flags)), address<uint8_t>(get(o, n_ovf)), address<int>(get(o, n_tile_off)), address<int>(get(o, n_ovf_used))};
}

// token_append(cache, slots, k, v, stream) -> True
PyObject* token_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 5, [&]() -> PyObject* {
    Refs get;
    const at::Tensor &slots = tensor(a[1]), &k = tensor(a[2]), &v = tensor(a[3]);
    const long n_kv = number(get(a[0], n_n_kv)), cap = number(get(a[0], n_cap));
    if (!is_rows(k, 3) || !is_rows(v, 3) || k.sizes() != v.sizes() || k.size(1) != n_kv || !k.is_contiguous() || !v.is_contiguous()) throw Otherwise{};
    if (slots.scalar_type() != at::kInt || slots.numel() != k.size(0) || !slots.is_contiguous() || k.size(0) == 0) throw Otherwise{};
    PyObject *ko = get(a[0], n_k), *vo = get(a[0], n_v);
    const CacheStore K = cache_store(get, ko), V = cache_store(get, vo);
    int *tail_len = address<int>(get(a[0], n_tail_len)), *S = address<int>(get(a[0], n_S)), *overflow = address<int>(get(a[0], n_overflow));
    const long ovf_cap = number(get(ko, n_ovf_cap)), nb = tensor(get(ko, n_base3)).size(0);
    void* stream = stream_of(a[4]);
    must("gaac_cache_append", without_gil([&] {
      return p_gaac_cache_append(static_cast<int*>(slots.data_ptr()), static_cast<int>(k.size(0)), static_cast<int>(n_kv), k.data_ptr(), v.data_ptr(), tail_len, S, static_cast<int>(cap),
                                 static_cast<int>(ovf_cap), static_cast<int>(nb), K.tail, K.b3, K.b4, K.sm, K.cd, K.fl, K.ov, K.to, K.used, V.tail, V.b3, V.b4, V.sm, V.cd, V.fl, V.ov,
                                 V.to, V.used, overflow, stream);
    }));
    Py_RETURN_TRUE;
  });
}

// prompt_store(cache, slot, k, v, stream) -> the heads' escape totals, of K and then of V
PyObject* prompt_store(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 5, [&]() -> PyObject* {
    Refs get;
    const at::Tensor &k = tensor(a[2]), &v = tensor(a[3]);
    const long slot = number(a[1]), n_kv = number(get(a[0], n_n_kv)), cap = number(get(a[0], n_cap)), n_slots = number(get(a[0], n_n_slots));
    if (!is_rows(k, 3) || !is_rows(v, 3) || k.sizes() != v.sizes() || k.size(1) != n_kv || k.size(0) < TILE || k.size(0) > cap || slot < 0 || slot >= n_slots) throw Otherwise{};
    long k_hs, k_rs, v_hs, v_rs;
    if (!in_place(k, 1, 0, k_hs, k_rs) || !in_place(v, 1, 0, v_hs, v_rs)) throw Otherwise{};
    const long L = k.size(0), nt = 2 * n_kv * (L / TILE);
    PyObject *ko = get(a[0], n_k), *vo = get(a[0], n_v);
    const int calibrate = PyObject_IsTrue(get(a[0], n_per_sequence_bases));
    if (calibrate < 0) throw Otherwise{};
    const CacheStore K = cache_store(get, ko), V = cache_store(get, vo);
    int *tail_len = address<int>(get(a[0], n_tail_len)), *S = address<int>(get(a[0], n_S)), *head_start = address<int>(get(ko, n_head_start));
    const long ovf_cap = number(get(ko, n_ovf_cap)), nb = tensor(get(ko, n_base3)).size(0);
    const at::Tensor& scan = tensor(get(a[0], n__scan));
    const long scan_row = scan.size(2);
    void* stream = stream_of(a[4]);
    // scratch: escape slots | exponent counts (hist_bytes in kv_cache.py) | tile sizes | head sizes
    const long tables = 2 * n_kv * std::max(std::min((L + 255) / 256, std::max(std::min(256 / (2 * n_kv), 64l), 1l)), (L + 65534) / 65535);
    const long at_hist = nt * TILE_ESCAPES, at_sizes = at_hist + (calibrate ? tables * HIST_BYTES : 0);
    at::Tensor scratch = bytes(k, {at_sizes + 4 * (nt + 2 * n_kv)}), totals = host_words(2 * n_kv);
    uint8_t* base = static_cast<uint8_t*>(scratch.data_ptr());
    int* words = static_cast<int*>(totals.data_ptr());
    must("gaac_prompt_store", without_gil([&] {
      return p_gaac_prompt_store(k.data_ptr(), v.data_ptr(), k_hs, k_rs, v_hs, v_rs, static_cast<int>(L), static_cast<int>(n_kv), static_cast<int>(slot * n_kv), static_cast<int>(cap),
                                 static_cast<int>(ovf_cap), static_cast<int>(nb), calibrate, tail_len, S, head_start, K.tail, K.b3, K.b4, K.sm, K.cd, K.fl, K.ov, K.to, K.used,
                                 V.tail, V.b3, V.b4, V.sm, V.cd, V.fl, V.ov, V.to, V.used, base + at_hist, at_sizes - at_hist, base,
                                 reinterpret_cast<int*>(base + at_sizes), reinterpret_cast<int*>(base + at_sizes + 4 * nt),
                                 static_cast<unsigned long long*>(scan.data_ptr()) + slot * n_kv * scan_row, scan.stride(0), static_cast<int>(scan_row), 0, words, stream);
    }));
    must("gaac_wait_words", without_gil([&] { return p_gaac_wait_words(words, static_cast<int>(2 * n_kv), stream); }));
    return numbers(totals);
  });
}

// page_encode(x, kind, base3, base4, n_kv, bytes of room a row, stream)
//   -> (sm, codes, flags, ovf_off, ovf or None where the room was too small, head_start, tile_off, the heads' totals, slots | sizes of the tiles | of the heads)
PyObject* page_encode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 7, [&]() -> PyObject* {
    const at::Tensor &x = tensor(a[0]), &b3 = tensor(a[2]), &b4 = tensor(a[3]);
    const long kind = number(a[1]), n_kv = number(a[4]), row_room = number(a[5]);
    long hs, rs;
    if (x.dim() != 3 || x.size(2) != DIM || x.itemsize() != 2 || x.size(0) == 0 || x.size(1) == 0 || !in_place(x, 0, 1, hs, rs)) throw Otherwise{};
    const long H = x.size(0), S = x.size(1), tiles = (S + TILE - 1) / TILE, S_pad = tiles * TILE, nt = H * tiles, room = row_room * H * S + 8;
    const int Hi = static_cast<int>(H), Si = static_cast<int>(S), Pi = static_cast<int>(S_pad);
    if (S_pad >= 1l << 31 || H >= 1l << 31) throw Otherwise{};
    void* stream = stream_of(a[6]);
    // each buffer is made when the next launch needs it
    at::Tensor sm = bytes(x, {H, S_pad * DIM}), cd = bytes(x, {H, S_pad * CODE_BYTES}), fl = bytes(x, {H, S_pad}, at::kInt), slots = bytes(x, {nt * TILE_ESCAPES + 4 * (nt + H)});
    uint8_t* slot = static_cast<uint8_t*>(slots.data_ptr());
    int *sizes = reinterpret_cast<int*>(slot + nt * TILE_ESCAPES), *heads = sizes + nt;
    must("gaac_encode_tiles", without_gil([&] {
      return p_gaac_encode_tiles(static_cast<int>(kind), x.data_ptr(), hs, rs, Hi, Si, Pi, static_cast<uint8_t*>(b3.data_ptr()), static_cast<uint8_t*>(b4.data_ptr()), static_cast<int>(n_kv),
                                 nullptr, static_cast<uint8_t*>(sm.data_ptr()), static_cast<uint8_t*>(cd.data_ptr()), static_cast<int*>(fl.data_ptr()), slot, sizes, stream);
    }));
    at::Tensor totals = host_words(H), off = bytes(x, {H, tiles}, at::kInt), ovf_off = bytes(x, {H, S}, at::kInt), start = bytes(x, {H + 1}, at::kInt), ovf = bytes(x, {room});
    int* words = static_cast<int*>(totals.data_ptr());
    must("gaac_page_finish", without_gil([&] {
      return p_gaac_page_finish(slot, sizes, static_cast<int*>(fl.data_ptr()), Hi, Si, Pi, static_cast<int*>(off.data_ptr()), heads, words, static_cast<int*>(start.data_ptr()),
                                static_cast<uint8_t*>(ovf.data_ptr()), room, static_cast<int*>(ovf_off.data_ptr()), stream);
    }));
    must("gaac_wait_words", without_gil([&] { return p_gaac_wait_words(words, Hi, stream); }));
    long total = 0;
    for (long h = 0; h < H; ++h) total += words[h];
    const bool fits = total + 8 <= room && total < (1l << 31) - 1;
    PyObject* list = numbers(totals);
    if (list == nullptr) return nullptr;
    PyObject* stream_view = fits ? THPVariable_Wrap(ovf.narrow(0, 0, total + 8)) : Py_NewRef(Py_None);
    return Py_BuildValue("(NNNNNNNNN)", THPVariable_Wrap(sm), THPVariable_Wrap(cd), THPVariable_Wrap(fl), THPVariable_Wrap(ovf_off), stream_view, THPVariable_Wrap(start),
                         THPVariable_Wrap(off), list, THPVariable_Wrap(slots));
  });
}

// page_decode(page, stream) -> bf16 [H, S, 128]
PyObject* page_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 2, [&]() -> PyObject* {
    Refs get;
    const long H = number(get(a[0], n_H)), S = number(get(a[0], n_S)), n_kv = number(get(a[0], n_n_kv));
    PyObject* kind = get(a[0], n_kind);
    if (!PyUnicode_CheckExact(kind) || H <= 0 || S <= 0) throw Otherwise{};
    const at::Tensor& sm = tensor(get(a[0], n_sm));
    if (sm.dim() != 2) throw Otherwise{};
    const auto at = [&](PyObject* name) { return tensor(get(a[0], name)).data_ptr(); };
    auto *cd = at(n_codes), *fl = at(n_flags), *off = at(n_tile_off), *ovf = at(n_ovf), *start = at(n_ovf_head_start), *b3 = at(n_base3), *b4 = at(n_base4);
    void* stream = stream_of(a[1]);
    at::Tensor out = bytes(sm, {H, S, DIM}, at::kBFloat16);
    must("gaac_decode_tiles", without_gil([&] {
      return p_gaac_decode_tiles(PyUnicode_CompareWithASCIIString(kind, "k") == 0 ? 0 : 1, static_cast<uint8_t*>(sm.data_ptr()), static_cast<uint8_t*>(cd), static_cast<int*>(fl),
                                 static_cast<int*>(off), static_cast<uint8_t*>(ovf), static_cast<int*>(start), static_cast<uint8_t*>(b3), static_cast<uint8_t*>(b4),
                                 static_cast<int>(n_kv), nullptr, static_cast<int>(H), static_cast<int>(S), static_cast<int>(sm.size(1) / DIM), out.data_ptr(), S * DIM, DIM, stream);
    }));
    return THPVariable_Wrap(out);
  });
}
// The calls of the 4-bit cache, of qk_norm_rope and of sample, the same way.  Their tensors have to be on the current device.  Host us a call, Python / here: prefill
// 9.9 / 3.3, append 8.8 / 3.6, attention 8.2 / 4.9 (with splits 11.1 / 7.1), qk_norm_rope 16.9 / 5.5, sample 9.0 / 4.7 (of three launches 14.0 / 9.8).
const at::Tensor& here(PyObject* o) {
  const at::Tensor& t = tensor(o);
  if (t.device() != c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getDevice()) throw Otherwise{};
  return t;
}
bool loses_gradient(const at::Tensor& t) { return (c10::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined(); }
// rows [n, heads, d] that a kernel reads through strides of whole 16 bytes
void strides_of(const at::Tensor& t, long& row, long& head) {
  const long per = 16 / t.itemsize();
  row = t.size(0) > 1 ? t.stride(0) : 0;
  head = t.size(1) > 1 ? t.stride(1) : 0;
  if (t.stride(2) != 1 || row % per != 0 || head % per != 0 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) throw Otherwise{};
}
bool is_slots(const at::Tensor& t, long B) { return t.dim() == 1 && t.size(0) == B && t.scalar_type() == at::kInt && t.is_contiguous(); }
struct Fp4Cache {
  uint8_t* data;
  int* lens;
  long n_slots, n_kv, tiles;
  Fp4Cache(Refs& get, PyObject* o) : data(static_cast<uint8_t*>(here(get(o, n_data)).data_ptr())), lens(address<int>(get(o, n_lens))), n_slots(number(get(o, n_n_slots))), n_kv(number(get(o, n_n_kv))),
                                     tiles(number(get(o, n_tiles))) {}
  uint8_t* slot(long i) const { return data + i * n_kv * tiles * 4352; }
};

// fp4_prefill(cache, slot, k, v, stream) -> True
PyObject* fp4_prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 5, [&]() -> PyObject* {
    Refs get;
    const Fp4Cache c(get, a[0]);
    const long slot = number(a[1]);
    const at::Tensor &k = here(a[2]), &v = here(a[3]);
    if (loses_gradient(k) || loses_gradient(v)) throw Otherwise{};
    if (!is_rows(k, 3) || !is_rows(v, 3) || k.sizes() != v.sizes() || k.size(1) != c.n_kv || k.size(0) == 0 || k.size(0) > c.tiles * 32 || slot < 0 || slot >= c.n_slots) throw Otherwise{};
    long k_rs, k_hs, v_rs, v_hs;
    strides_of(k, k_rs, k_hs);
    strides_of(v, v_rs, v_hs);
    void* stream = stream_of(a[4]);
    must("gaac_fp4_store", without_gil([&] {
      return p_gaac_fp4_store(k.data_ptr(), v.data_ptr(), k_hs, k_rs, v_hs, v_rs, static_cast<int>(k.size(0)), static_cast<int>(c.n_kv), static_cast<int>(c.tiles), c.slot(slot), c.lens + slot, stream);
    }));
    Py_RETURN_TRUE;
  });
}

// fp4_append(cache, slots, k, v, stream) -> True
PyObject* fp4_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 5, [&]() -> PyObject* {
    Refs get;
    const Fp4Cache c(get, a[0]);
    const at::Tensor &slots = here(a[1]), &k = here(a[2]), &v = here(a[3]);
    if (loses_gradient(k) || loses_gradient(v)) throw Otherwise{};
    if (!is_rows(k, 3) || !is_rows(v, 3) || k.sizes() != v.sizes() || k.size(1) != c.n_kv || k.size(0) == 0 || !is_slots(slots, k.size(0))) throw Otherwise{};
    long k_rs, k_hs, v_rs, v_hs;
    strides_of(k, k_rs, k_hs);
    strides_of(v, v_rs, v_hs);
    int* overflow = address<int>(get(a[0], n_overflow));
    const long cap = number(get(a[0], n_cap));
    void* stream = stream_of(a[4]);
    must("gaac_fp4_append", without_gil([&] {
      return p_gaac_fp4_append(static_cast<int*>(slots.data_ptr()), static_cast<int>(k.size(0)), static_cast<int>(c.n_slots), static_cast<int>(c.n_kv), k.data_ptr(), v.data_ptr(), k_rs, k_hs, v_rs, v_hs, c.lens,
                               static_cast<int>(c.tiles), static_cast<int>(cap), c.data, overflow, stream);
    }));
    Py_RETURN_TRUE;
  });
}

// fp4_attend(cache, q, slots, scale, nsplit, tickets or None, stream) -> out like q [B, n_q, 128]
PyObject* fp4_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 7, [&]() -> PyObject* {
    Refs get;
    const Fp4Cache c(get, a[0]);
    const at::Tensor &q = here(a[1]), &slots = here(a[2]);
    if (loses_gradient(q)) throw Otherwise{};
    const long nsplit = number(a[4]), cap = number(get(a[0], n_cap));
    if (!is_rows(q, 3) || !q.is_contiguous() || reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 != 0 || q.size(0) == 0 || !is_slots(slots, q.size(0)) || nsplit < 1 || nsplit > 1 << 20) throw Otherwise{};
    const long B = q.size(0), n_q = q.size(1);
    if (n_q < c.n_kv || n_q % c.n_kv != 0 || n_q / c.n_kv > 16 || !PyFloat_CheckExact(a[3])) throw Otherwise{};
    unsigned* tickets = a[5] == Py_None ? nullptr : address<unsigned>(a[5]);
    const float scale = static_cast<float>(PyFloat_AS_DOUBLE(a[3]));
    void* stream = stream_of(a[6]);
    at::Tensor out = bytes(q, {B, n_q, DIM}, at::kBFloat16), partials;
    if (nsplit > 1) partials = bytes(q, {B * nsplit * n_q * (DIM + 2)}, at::kFloat);
    float* part = nsplit > 1 ? static_cast<float*>(partials.data_ptr()) : nullptr;
    must("gaac_fp4_attn", without_gil([&] {
      return p_gaac_fp4_attn(c.data, c.lens, static_cast<int*>(slots.data_ptr()), static_cast<int>(c.n_slots), static_cast<int>(c.tiles), static_cast<int>(cap), q.data_ptr(), static_cast<int>(B), static_cast<int>(n_q),
                             static_cast<int>(c.n_kv), scale, static_cast<int>(nsplit), part, tickets, out.data_ptr(), stream);
    }));
    return THPVariable_Wrap(out);
  });
}

// fp4_read(cache, slot, stream) -> (K, V) bf16 [tokens, n_kv, 128]; waits for the slot's length
PyObject* fp4_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 3, [&]() -> PyObject* {
    Refs get;
    const Fp4Cache c(get, a[0]);
    const long slot = number(a[1]);
    if (slot < 0 || slot >= c.n_slots) throw Otherwise{};
    void* stream = stream_of(a[2]);
    at::Tensor word = host_words(1);
    int* len = static_cast<int*>(word.data_ptr());
    must("gaac_fp4_length", without_gil([&] { return p_gaac_fp4_length(c.lens + slot, static_cast<int>(c.tiles), len, stream); }));
    must("gaac_wait_words", without_gil([&] { return p_gaac_wait_words(len, 1, stream); }));
    const long L = *len, row = c.n_kv * DIM;
    const at::Tensor& like = tensor(get(a[0], n_data));
    at::Tensor k = bytes(like, {L, c.n_kv, DIM}, at::kBFloat16), v = bytes(like, {L, c.n_kv, DIM}, at::kBFloat16);
    if (L > 0)
      must("gaac_fp4_load", without_gil([&] {
        return p_gaac_fp4_load(c.slot(slot), static_cast<int>(L), static_cast<int>(c.n_kv), static_cast<int>(c.tiles), k.data_ptr(), v.data_ptr(), DIM, row, DIM, row, stream);
      }));
    return Py_BuildValue("(NN)", THPVariable_Wrap(k), THPVariable_Wrap(v));
  });
}

int float_type(const at::Tensor& t) {      // the number of the type in the C interface
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: throw Otherwise{};
  }
}

// norm_rope(q, k, positions, cos, sin, q_weight or None, k_weight or None, eps, interleaved, stream) -> (q, k)
PyObject* norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 10, [&]() -> PyObject* {
    const at::Tensor &q = here(a[0]), &k = here(a[1]), &pos = here(a[2]), &cos = here(a[3]), &sin = here(a[4]);
    const int type = float_type(q);
    if (loses_gradient(q) || loses_gradient(k) || loses_gradient(cos) || loses_gradient(sin) || (a[5] != Py_None && loses_gradient(tensor(a[5]))) || (a[6] != Py_None && loses_gradient(tensor(a[6])))) throw Otherwise{};
    if (q.dim() != 3 || k.dim() != 3 || q.scalar_type() != k.scalar_type() || q.size(0) != k.size(0) || q.size(2) != k.size(2) || q.size(0) == 0 || q.size(1) == 0 || k.size(1) == 0) throw Otherwise{};
    const long N = q.size(0), n_q = q.size(1), n_k = k.size(1), D = q.size(2);
    if ((D != 64 && D != 128 && D != 256) || N >= 1l << 26 || n_q >= 1 << 20 || n_k >= 1 << 20) throw Otherwise{};
    if (pos.dim() != 1 || pos.size(0) != N || !pos.is_contiguous() || (pos.scalar_type() != at::kLong && pos.scalar_type() != at::kInt)) throw Otherwise{};
    if (cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat || cos.dim() != 2 || cos.sizes() != sin.sizes() || cos.size(0) < 1 || cos.size(0) >= 1l << 31 || !cos.is_contiguous() || !sin.is_contiguous()) throw Otherwise{};
    const long R = 2 * cos.size(1);
    if (R < 16 || R > D || R % 16 != 0 || !PyFloat_CheckExact(a[7])) throw Otherwise{};
    long q_ts, q_hs, k_ts, k_hs, w_hs[2] = {0, 0};
    strides_of(q, q_ts, q_hs);
    strides_of(k, k_ts, k_hs);
    void* w[2] = {nullptr, nullptr};
    uintptr_t all = reinterpret_cast<uintptr_t>(cos.data_ptr()) | reinterpret_cast<uintptr_t>(sin.data_ptr());
    if ((a[5] == Py_None) != (a[6] == Py_None)) throw Otherwise{};
    for (int i = 0; i < 2 && a[5] != Py_None; ++i) {
      const at::Tensor& t = here(a[5 + i]);
      const long heads = i == 0 ? n_q : n_k;
      if (t.scalar_type() != q.scalar_type() || !t.is_contiguous() || !((t.dim() == 1 && t.size(0) == D) || (t.dim() == 2 && t.size(0) == heads && t.size(1) == D))) throw Otherwise{};
      w[i] = t.data_ptr(); w_hs[i] = t.dim() == 2 ? D : 0;
      all |= reinterpret_cast<uintptr_t>(w[i]);
    }
    const int interleaved = PyObject_IsTrue(a[8]);
    if (all % 16 != 0 || interleaved < 0) throw Otherwise{};
    void* stream = stream_of(a[9]);
    at::Tensor qo = bytes(q, {N, n_q, D}, q.scalar_type()), ko = bytes(k, {N, n_k, D}, q.scalar_type());
    must("gaac_qk_norm_rope", without_gil([&] {
      return p_gaac_qk_norm_rope(type, q.data_ptr(), k.data_ptr(), q_ts, q_hs, k_ts, k_hs, N, static_cast<int>(n_q), static_cast<int>(n_k), static_cast<int>(D), static_cast<int>(R), w[0], w[1], w_hs[0], w_hs[1],
                                 static_cast<float>(PyFloat_AS_DOUBLE(a[7])), pos.data_ptr(), pos.scalar_type() == at::kLong, static_cast<float*>(cos.data_ptr()), static_cast<float*>(sin.data_ptr()),
                                 static_cast<int>(cos.size(0)), interleaved, qo.data_ptr(), ko.data_ptr(), stream);
    }));
    return Py_BuildValue("(NN)", THPVariable_Wrap(qo), THPVariable_Wrap(ko));
  });
}

// draw(logits, u, temperature, top_k, top_p, min_p, stream) -> tokens int64 [B]; each setting a number or a tensor [B]
PyObject* draw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 7, [&]() -> PyObject* {
    const at::Tensor &x = here(a[0]), &u = here(a[1]);
    const int type = float_type(x);
    if (x.dim() != 2 || x.size(0) == 0 || x.size(0) >= 1l << 31 || x.size(1) == 0 || x.size(1) > (1l << 20) - 16 || (x.size(1) > 1 && x.stride(1) != 1)) throw Otherwise{};
    const long B = x.size(0), V = x.size(1);
    if (u.dim() != 1 || u.size(0) != B || u.scalar_type() != at::kFloat || !u.is_contiguous()) throw Otherwise{};
    const auto rows = [&](PyObject* o, at::ScalarType t) -> void* {
      if (!THPVariable_CheckExact(o)) return nullptr;
      const at::Tensor& r = here(o);
      if (r.dim() != 1 || r.size(0) != B || r.scalar_type() != t || !r.is_contiguous()) throw Otherwise{};
      return r.data_ptr();
    };
    const auto real = [&](PyObject* o) -> float {
      if (PyFloat_CheckExact(o)) return static_cast<float>(PyFloat_AS_DOUBLE(o));
      if (THPVariable_CheckExact(o)) return 0.f;
      return static_cast<float>(number(o));
    };
    float *t = static_cast<float*>(rows(a[2], at::kFloat)), *p = static_cast<float*>(rows(a[4], at::kFloat)), *m = static_cast<float*>(rows(a[5], at::kFloat));
    int* k = static_cast<int*>(rows(a[3], at::kInt));
    const long top_k = THPVariable_CheckExact(a[3]) ? 0 : std::max(0l, std::min(number(a[3]), V));
    const float temperature = real(a[2]), top_p = real(a[4]), min_p = real(a[5]);
    void* stream = stream_of(a[6]);
    const long segments = (V + 7 + 4095) / 4096, work_bytes = segments == 1 ? 0 : std::min(B, 1024l) * (16 * segments + 90128);      // work_bytes in sampling.py
    at::Tensor out = bytes(x, {B}, at::kLong), work = bytes(x, {work_bytes});
    must("gaac_sample", without_gil([&] {
      return p_gaac_sample(type, x.data_ptr(), B > 1 ? x.stride(0) : 0, static_cast<int>(B), static_cast<int>(V), static_cast<float*>(u.data_ptr()), t, temperature, k, static_cast<int>(top_k), p, top_p, m, min_p,
                           work.data_ptr(), work_bytes, static_cast<int64_t*>(out.data_ptr()), stream);
    }));
    return THPVariable_Wrap(out);
  });
}
// Rows in 8 bits, their products, and log probabilities, the same way.  Host us a call, Python / here: quantize_fp8 11.2 / 6.1, rms_norm_fp8 with a residual 14.6 / 7.0, dequantize 7.8 / 5.0, a product of rows in
// 8 bits 8.5 / 5.2 and of a tensor 21.1 / 9.5 (two launches; its 8 bits in two allocations instead of one: 10.2), token_logprobs 15.7 / 6.5, with alternatives 19.5 / 8.2.
long blocks_of(long K) { return (K + 127) / 128; }
long padded(long rows) { return (rows + 15) / 16 * 16; }
at::ScalarType type_of(long code) {
  if (code < 0 || code > 2) throw Otherwise{};
  return code == 0 ? at::kBFloat16 : code == 1 ? at::kHalf : at::kFloat;
}
// [M, K] with elements next to each other -> its row stride
long rows_of(const at::Tensor& t, long most) {
  if (t.dim() != 2 || t.size(0) == 0 || t.size(0) > 1l << 24 || t.size(1) == 0 || t.size(1) > most || (t.size(1) > 1 && t.stride(1) != 1)) throw Otherwise{};
  return t.size(0) > 1 ? t.stride(0) : 0;
}
struct Rows8 {
  at::Tensor data, exps;
  Rows8(const at::Tensor& like, long M, long K) : data(bytes(like, {padded(M) * blocks_of(K) * 128})), exps(bytes(like, {(blocks_of(K) + 3) / 4 * padded(M) * 4})) {}
};

// fp8_rows(x, weight or None, eps, residual or None, stream) -> (data, exps) or (data, exps, sum)
PyObject* fp8_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 5, [&]() -> PyObject* {
    const at::Tensor& x = here(a[0]);
    const int type = float_type(x);
    const bool norm = a[1] != Py_None, add = a[3] != Py_None;
    const long x_rs = rows_of(x, norm ? 32768 : 65536), M = x.size(0), K = x.size(1);
    if (loses_gradient(x)) throw Otherwise{};
    void *w = nullptr, *r = nullptr, *h = nullptr;
    long r_rs = 0;
    float eps = 0;
    at::Tensor sum;
    if (norm) {
      const at::Tensor& t = here(a[1]);
      if (t.scalar_type() != x.scalar_type() || t.dim() != 1 || t.size(0) != K || !t.is_contiguous() || loses_gradient(t) || !PyFloat_CheckExact(a[2])) throw Otherwise{};
      w = t.data_ptr(); eps = static_cast<float>(PyFloat_AS_DOUBLE(a[2]));
    }
    if (add) {
      const at::Tensor& t = here(a[3]);
      if (!norm || t.scalar_type() != x.scalar_type() || t.sizes() != x.sizes() || loses_gradient(t)) throw Otherwise{};
      r_rs = rows_of(t, 32768); r = t.data_ptr();
      sum = bytes(x, {M, K}, x.scalar_type()); h = sum.data_ptr();
    }
    void* stream = stream_of(a[4]);
    const Rows8 out(x, M, K);
    must("gaac_fp8_rows", without_gil([&] {
      return p_gaac_fp8_rows(type, x.data_ptr(), x_rs, r, r_rs, w, eps, static_cast<int>(M), static_cast<int>(K), h, out.data.data_ptr(), out.exps.data_ptr(), padded(M), 1, 0, stream);
    }));
    if (add) return Py_BuildValue("(NNN)", THPVariable_Wrap(out.data), THPVariable_Wrap(out.exps), THPVariable_Wrap(sum));
    return Py_BuildValue("(NN)", THPVariable_Wrap(out.data), THPVariable_Wrap(out.exps));
  });
}

// fp8_multiply(x [M, K], or data of M rows; exps or None, M, weight's data, exps, N, K, gated, type, stream) -> [M, N]
PyObject* fp8_multiply(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 10, [&]() -> PyObject* {
    const at::Tensor &x = here(a[0]), &w = here(a[3]), &we = here(a[4]);
    const long M = number(a[2]), N = number(a[5]), K = number(a[6]), type = number(a[8]);
    const bool rows = a[1] != Py_None;
    if (M <= 0 || M > 1 << 20) throw Otherwise{};
    const int gated = PyObject_IsTrue(a[7]);
    const at::ScalarType out_type = type_of(type);
    long x_rs = 0;
    if (!rows) {
      x_rs = rows_of(x, 65536);
      if (x.size(0) != M || x.size(1) != K || loses_gradient(x)) throw Otherwise{};
    }
    const int x_type = rows ? 0 : float_type(x);
    void* stream = stream_of(a[9]);
    const void *data = nullptr, *exps = nullptr;
    at::Tensor made;      // both in one piece
    if (rows) { data = x.data_ptr(); exps = here(a[1]).data_ptr(); }
    else {
      const long codes = padded(M) * blocks_of(K) * 128;
      made = bytes(x, {codes + (blocks_of(K) + 3) / 4 * padded(M) * 4});
      void *to = made.data_ptr(), *to_exps = static_cast<uint8_t*>(to) + codes;
      must("gaac_fp8_rows", without_gil([&] {
        return p_gaac_fp8_rows(x_type, x.data_ptr(), x_rs, nullptr, 0, nullptr, 0.f, static_cast<int>(M), static_cast<int>(K), nullptr, to, to_exps, padded(M), 1, 0, stream);
      }));
      data = to; exps = to_exps;
    }
    at::Tensor out = bytes(x, {M, N}, out_type);
    must("gaac_fp8_product", without_gil([&] {
      return p_gaac_fp8_product(data, exps, w.data_ptr(), we.data_ptr(), static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), gated, static_cast<int>(type), out.data_ptr(), N, stream);
    }));
    return THPVariable_Wrap(out);
  });
}

// fp8_values(data, exps, M, K, tile step, first tile, stream) -> bf16 [M, K]
PyObject* fp8_values(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 7, [&]() -> PyObject* {
    const at::Tensor &data = here(a[0]), &exps = here(a[1]);
    const long M = number(a[2]), K = number(a[3]), step = number(a[4]), first = number(a[5]);
    if (M <= 0) throw Otherwise{};
    void* stream = stream_of(a[6]);
    at::Tensor out = bytes(data, {M, K}, at::kBFloat16);
    must("gaac_fp8_values", without_gil([&] {
      return p_gaac_fp8_values(data.data_ptr(), exps.data_ptr(), padded(M) * step, static_cast<int>(step), static_cast<int>(first), static_cast<int>(M), static_cast<int>(K), out.data_ptr(), K, stream);
    }));
    return THPVariable_Wrap(out);
  });
}

// logprobs(logits, tokens, top, stream) -> (logprob, rank, entropy, top_logprobs or None, top_tokens or None)
PyObject* logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return whole_call(n, 4, [&]() -> PyObject* {
    const at::Tensor &x = here(a[0]), &t = here(a[1]);
    const int type = float_type(x);
    const long top = number(a[2]);
    if (x.dim() != 2 || x.size(0) == 0 || x.size(1) == 0 || x.size(1) > (1l << 20) - 16 || x.size(0) > (1l << 22) / ((x.size(1) + 8191) / 8192) || (x.size(1) > 1 && x.stride(1) != 1) || loses_gradient(x)) throw Otherwise{};
    const long B = x.size(0), V = x.size(1);
    if (t.dim() != 1 || t.size(0) != B || t.scalar_type() != at::kLong || !t.is_contiguous() || top < 0 || top > std::min(64l, V)) throw Otherwise{};
    void* stream = stream_of(a[3]);
    const long segments = (V + 8191) / 8192, work_bytes = segments == 1 ? 0 : B * segments * (16 + 8 * top);      // logprobs_work_bytes in sampling.py
    at::Tensor work, value = bytes(x, {B}, at::kFloat), rank = bytes(x, {B}, at::kLong), entropy = bytes(x, {B}, at::kFloat), top_values, top_tokens;
    if (work_bytes > 0) work = bytes(x, {work_bytes});
    if (top > 0) { top_values = bytes(x, {B, top}, at::kFloat); top_tokens = bytes(x, {B, top}, at::kLong); }
    must("gaac_logprobs", without_gil([&] {
      return p_gaac_logprobs(type, x.data_ptr(), B > 1 ? x.stride(0) : 0, static_cast<int>(B), static_cast<int>(V), static_cast<int64_t*>(t.data_ptr()), static_cast<int>(top), work_bytes > 0 ? work.data_ptr() : nullptr, work_bytes,
                             static_cast<float*>(value.data_ptr()), static_cast<int64_t*>(rank.data_ptr()), static_cast<float*>(entropy.data_ptr()), top > 0 ? static_cast<float*>(top_values.data_ptr()) : nullptr,
                             top > 0 ? static_cast<int64_t*>(top_tokens.data_ptr()) : nullptr, stream);
    }));
    return Py_BuildValue("(NNNNN)", THPVariable_Wrap(value), THPVariable_Wrap(rank), THPVariable_Wrap(entropy), top > 0 ? THPVariable_Wrap(top_values) : Py_NewRef(Py_None),
                         top > 0 ? THPVariable_Wrap(top_tokens) : Py_NewRef(Py_None));
  });
}
#define GAAC_WHOLE_CALLS(X) X(attend) X(token_append) X(prompt_store) X(page_encode) X(page_decode) X(fp4_prefill) X(fp4_append) X(fp4_attend) X(fp4_read) X(norm_rope) X(draw) X(fp8_rows) X(fp8_multiply) X(fp8_values) X(logprobs)

// bind(path): the entry points of the library at path (the product or one of its measurement builds); AttributeError names a missing one
PyObject* bind(PyObject*, PyObject* path) {
  const char* file = PyUnicode_AsUTF8(path);
  if (file == nullptr) return nullptr;
  void* lib = dlopen(file, RTLD_NOW | RTLD_LOCAL);
  if (lib == nullptr) { PyErr_SetString(PyExc_RuntimeError, dlerror()); return nullptr; }
  const auto find = [&](const char* name) {
    void* p = dlsym(lib, name);
    if (p == nullptr && !PyErr_Occurred()) PyErr_Format(PyExc_AttributeError, "%s: undefined symbol: %s", file, name);
    return p;
  };
#define X(name) p_##name = reinterpret_cast<decltype(p_##name)>(find(#name));
  GAAC_ENTRY_POINTS(X)
#undef X
  g_last_error = reinterpret_cast<const char* (*)()>(find("gaac_last_error"));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

#define X(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr},
#define Y(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr},
PyMethodDef methods[] = {GAAC_ENTRY_POINTS(X) GAAC_WHOLE_CALLS(Y){"bind", bind, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
#undef X
#undef Y
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() {
#define X(name) if ((n_##name = PyUnicode_InternFromString(#name)) == nullptr) return nullptr;
  GAAC_NAMES(X)
#undef X
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", GAAC_TORCH_VERSION) != 0) { Py_DECREF(m); return nullptr; }      // whose headers these are
  return m;
}
