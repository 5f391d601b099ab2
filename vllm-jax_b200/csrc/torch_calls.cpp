// The quantised cache's operators as Python calls: argument checks, outputs and
// scratch, current stream, C entry. Behind vllm_b200/kernels/quantized_cache.py,
// which documents them.
//
// Compiled because the calls are short: an eager decode of one sequence is 5 us
// on the GPU, and the same checks in Python with a ctypes call took 15 us of
// host time.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContextLight.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/sub.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "../../include/vjattn.h"

namespace {

// ---- what bind() is given: the C entries, and Python's side of the package
decltype(&vj_kv_store_quantized) store_entry;
decltype(&vj_paged_decode_quantized) decode_entry;
decltype(&vj_paged_decode_quantized_workspace_size) workspace_entry;
decltype(&vj_kv_read_quantized) read_entry;
decltype(&vj_paged_prefill_split) prefill_entry, prefill_part_entry;
decltype(&vj_paged_prefill_split_workspace_size) prefill_workspace_entry;
decltype(&vj_paged_prefill_quantized) direct_entry;
decltype(&vj_paged_prefill_quantized_workspace_size) direct_workspace_entry;
PyObject *native;             // module: check(status), launch_count
PyObject *error_flag_of;      // (device index) -> address
PyObject *rope_table_of;      // (device, theta) -> tensor

struct Raised {};             // a Python error is set

[[noreturn]] void fail(const char *format, ...) {
  va_list args;
  va_start(args, format);
  PyErr_FormatV(PyExc_ValueError, format, args);
  va_end(args);
  throw Raised{};
}
template <typename T>
T raise_if_null(T p) {
  if (p == nullptr) throw Raised{};
  return p;
}

// A new reference, dropped at the end of its scope.
struct Owned {
  PyObject *p;
  explicit Owned(PyObject *p) : p(raise_if_null(p)) {}
  Owned(const Owned &) = delete;
  ~Owned() { Py_DECREF(p); }
};

// A tensor argument: the Python object and what it holds, or nothing (None).
struct Arg {
  PyObject *o = nullptr;
  const at::Tensor *t = nullptr;
  explicit operator bool() const { return t != nullptr; }
  const at::Tensor *operator->() const { return t; }
  void *ptr() const { return t ? t->data_ptr() : nullptr; }
};
Arg tensor(PyObject *o, const char *name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "`%s` must be a tensor, not %s", name, Py_TYPE(o)->tp_name);
    throw Raised{};
  }
  return {o, &THPVariable_Unpack(o)};
}
Arg maybe(PyObject *o, const char *name) { return o == Py_None ? Arg{} : tensor(o, name); }

bool truth(PyObject *o) {
  const int r = PyObject_IsTrue(o);
  if (r < 0) throw Raised{};
  return r != 0;
}
double number(PyObject *o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw Raised{};
  return x;
}
int64_t integer(PyObject *o) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) throw Raised{};
  return x;
}
int32_t i32(int64_t x, const char *name) {
  if (x < INT32_MIN || x > INT32_MAX) fail("%s does not fit 32 bits: %lld", name, (long long)x);
  return static_cast<int32_t>(x);
}

[[noreturn]] void fail_dtype(const Arg &a, const char *name, const char *must_be) {
  const Owned got(PyObject_GetAttrString(a.o, "dtype"));
  fail("The dtype of `%s` must be %s. Got %S", name, must_be, got.p);
}
void require_dtype(const Arg &a, at::ScalarType type, const char *name, const char *must_be) {
  if (a->scalar_type() != type) fail_dtype(a, name, must_be);
}
void require_bf16(const Arg &a, const char *name) {
  require_dtype(a, at::kBFloat16, name, "torch.bfloat16");
}

// The CUDA device all tensors are on.
int device_of(std::initializer_list<const Arg *> args) {
  int index = -1;
  for (const Arg *a : args) {
    if (!*a) continue;
    if (!(*a)->is_cuda()) {
      const Owned device(PyObject_GetAttrString(a->o, "device"));
      fail("vllm_b200 kernels run on CUDA tensors only (no CPU fallback); got a tensor on %S",
           device.p);
    }
    const int i = (*a)->get_device();
    if (index >= 0 && i != index) fail("tensors on different devices: cuda:%d and cuda:%d", index, i);
    index = i;
  }
  return index;
}

// The device's error word (kept for good by its owner, so its address is too).
int32_t *error_flag(int index) {
  static int32_t *flags[64];
  if (index < 64 && flags[index]) return flags[index];
  const Owned address(PyObject_CallFunction(error_flag_of, "i", index));
  int32_t *p = reinterpret_cast<int32_t *>(integer(address.p));
  if (index < 64) flags[index] = p;
  return p;
}

// A C entry without the interpreter's lock; counts the launches of its longest form (as
// _native.call does), raises its errors.
template <typename F>
void enter(int launches, F &&entry) {
  int status;
  Py_BEGIN_ALLOW_THREADS;
  status = entry();
  Py_END_ALLOW_THREADS;
  if (status != VJ_OK) {
    const Owned raised(PyObject_CallMethod(native, "check", "i", status));
    fail("status %d", status);        // check() raises
  }
  const Owned count(PyObject_GetAttrString(native, "launch_count"));
  const Owned more(PyLong_FromLongLong(integer(count.p) + launches));
  if (PyObject_SetAttrString(native, "launch_count", more.p) < 0) throw Raised{};
}

struct Pool {
  Arg data, scales;
  uint8_t *k, *v, *ks, *vs;
  int32_t code, hkv, D, bs;
  int64_t nb, sb, st, sh, cb, ch;
};
Pool pool_tensors(PyObject *cache) {
  if (!PyTuple_Check(cache) || PyTuple_GET_SIZE(cache) != 2) {
    PyErr_Format(PyExc_TypeError, "`cache` must be a QuantizedKVCache, not %s",
                 Py_TYPE(cache)->tp_name);
    throw Raised{};
  }
  Pool p;
  p.data = tensor(PyTuple_GET_ITEM(cache, 0), "cache.data");
  p.scales = tensor(PyTuple_GET_ITEM(cache, 1), "cache.scales");
  return p;
}
void check_pool(Pool &p) {
  const auto shape = p.data->sizes();
  if (shape.size() != 5 || shape[0] != 2) {
    const Owned got(PyObject_GetAttrString(p.data.o, "shape"));
    fail("cache.data must have shape (2, num_blocks, block_size, Hkv, D); got %S", got.p);
  }
  const auto type = p.data->scalar_type();
  p.code = type == at::kFloat8_e4m3fn ? VJ_CACHE_E4M3 : type == at::kChar ? VJ_CACHE_INT8 : 0;
  if (!p.code) fail_dtype(p.data, "cache.data", "float8_e4m3fn or int8");
  require_dtype(p.scales, at::kByte, "cache.scales", "torch.uint8");
  p.nb = shape[1];
  p.bs = i32(shape[2], "block_size");
  p.hkv = i32(shape[3], "Hkv");
  p.D = i32(shape[4], "head_dim");
  const auto s = p.scales->sizes();
  if (s.size() != 4 || s[0] != 2 || s[1] != p.nb || s[2] != p.hkv || s[3] != p.bs) {
    const Owned got(PyObject_GetAttrString(p.scales.o, "shape"));
    fail("cache.scales must have shape (2, num_blocks, Hkv, block_size) = (2, %lld, %d, %d); got %S",
         (long long)p.nb, p.hkv, p.bs, got.p);
  }
  const auto d = p.data->strides(), c = p.scales->strides();
  if (d[4] != 1 || c[3] != 1) {
    fail("cache.data's head_dim and cache.scales' block_size must be contiguous");
  }
  p.sb = d[1], p.st = d[2], p.sh = d[3], p.cb = c[1], p.ch = c[2];
  p.k = static_cast<uint8_t *>(p.data->data_ptr());
  p.ks = static_cast<uint8_t *>(p.scales->data_ptr());
  p.v = p.k + d[0];
  p.vs = p.ks + c[0];
}

// A [T, H, D] tensor with packed heads.
struct Rows {
  int64_t heads = 0, stride = 0;
  void *ptr = nullptr;
};
Rows rows(const Arg &a, const char *name, int64_t T, int64_t D) {
  require_bf16(a, name);
  const auto s = a->sizes(), st = a->strides();
  if (s.size() != 3 || s[0] != T || s[2] != D || st[2] != 1 || (st[1] != D && s[1] != 1)) {
    fail("`%s` must be a [num_tokens, H, head_dim] tensor with packed heads", name);
  }
  // (a stride of 0 would mean packed rows to the C entries)
  if (T > 1 && st[0] < s[1] * D) fail("rows of `%s` must not overlap", name);
  return {s[1], T > 1 ? st[0] : s[1] * D, a.ptr()};
}
const int32_t *indices(const Arg &a, const char *name, int64_t T) {
  require_dtype(a, at::kInt, name, "torch.int32");
  if (a->dim() != 1 || a->size(0) != T || !a->is_contiguous()) {
    const Owned got(PyObject_GetAttrString(a.o, "shape"));
    fail("%s must be a contiguous [%lld] tensor; got shape %S", name, (long long)T, got.p);
  }
  return static_cast<const int32_t *>(a.ptr());
}
const void *weight(const Arg &a, const char *name, int64_t D) {
  require_bf16(a, name);
  if (a->dim() != 1 || a->size(0) != D || !a->is_contiguous()) {
    fail("%s must be a contiguous [head_dim] tensor", name);
  }
  return a.ptr();
}
// Packed [n, Hq, D] rows of q.
void check_q(const Arg &q, const char *shape) {
  require_bf16(q, "q");
  if (q->dim() != 3 || !q->is_contiguous()) fail("q must be a contiguous [%s, Hq, head_dim] tensor", shape);
}
void check_heads(const Arg &q, const Pool &p) {
  if (q->size(2) != p.D || p.hkv == 0 || q->size(1) % p.hkv) {
    fail("q heads/head_dim do not match the cache");
  }
}
at::Tensor output(const Arg &out, const Arg &q) {
  if (!out) return at::empty(q->sizes(), q->options());
  if (out->sizes() != q->sizes() || out->scalar_type() != q->scalar_type() || !out->is_contiguous()) {
    fail("out must be a contiguous bf16 tensor of q's shape");
  }
  return *out.t;
}

struct Tables {
  const int32_t *ptr, *lens;
  int32_t width, stride;
};
Tables tables(const Arg &bt, const Arg &lens, int64_t B) {
  require_dtype(bt, at::kInt, "block_tables", "torch.int32");
  if (bt->dim() != 2 || bt->size(0) != B) fail("`block_tables` must have one row per sequence");
  Tables t;
  t.width = i32(bt->size(1), "the width of block_tables");
  if (B > 0 && t.width > 1 && bt->stride(1) != 1) fail("block_tables rows must be contiguous");
  int64_t stride = bt->stride(0);
  if (B == 0 || stride < t.width) {
    if (B > 1) fail("block_tables rows must not overlap");
    stride = t.width;
  }
  t.stride = i32(stride, "the stride of block_tables");
  t.ptr = static_cast<const int32_t *>(bt.ptr());
  t.lens = indices(lens, "context_lens", B);
  return t;
}

int num_sms() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }
cudaStream_t stream_of(int index) { return c10::cuda::getCurrentCUDAStream(index).stream(); }

// (q, k, v, cache, slot_mapping, positions, q_norm_weight, k_norm_weight, eps,
//  rope_theta, norm, rope, q_out, table)
PyObject *kv_store(PyObject *const *args) {
  const Arg q = maybe(args[0], "q"), k = tensor(args[1], "k"), v = tensor(args[2], "v");
  Pool p = pool_tensors(args[3]);
  const Arg slots = tensor(args[4], "slot_mapping"), positions = maybe(args[5], "positions");
  const Arg qw = maybe(args[6], "q_norm_weight"), kw = maybe(args[7], "k_norm_weight");
  const Arg given = maybe(args[12], "q_out");
  Arg table = maybe(args[13], "table");
  const int dev = device_of({&k, &v, &p.data, &p.scales, &slots, &q, &positions, &qw, &kw, &given,
                             &table});
  check_pool(p);
  if (v->sizes() != k->sizes()) {
    const Owned a(PyObject_GetAttrString(k.o, "shape")), b(PyObject_GetAttrString(v.o, "shape"));
    fail("k and v must have the same shape. Got %S and %S", a.p, b.p);
  }
  const int64_t T = k->dim() > 0 ? k->size(0) : 0;
  const Rows rk = rows(k, "k", T, p.D), rv = rows(v, "v", T, p.D);
  if (rk.heads != p.hkv) fail("cache heads/head_dim do not match k");
  const int32_t *slot_ptr = indices(slots, "slot_mapping", T);
  const bool norm = truth(args[10]), rope = truth(args[11]);
  Rows rq, ro;
  if (q) rq = rows(q, "q", T, p.D);
  if (given) {
    if (!q) fail("q_out needs q");
    ro = rows(given, "q_out", T, p.D);
    if (ro.heads != rq.heads) fail("q_out must have q's shape");
  }
  const void *qw_ptr = nullptr, *kw_ptr = nullptr, *table_ptr = nullptr;
  int32_t flags = 0, table_len = 0;
  if (norm) {
    flags |= VJ_KV_NORM;
    if (!kw || (q && !qw)) fail("norm=True needs q_norm_weight and k_norm_weight");
    kw_ptr = weight(kw, "k_norm_weight", p.D);
    if (q) qw_ptr = weight(qw, "q_norm_weight", p.D);
  }
  const double theta = number(args[9]);
  const int32_t *pos_ptr = nullptr;
  PyObject *made = nullptr;
  if (rope) {
    flags |= VJ_KV_ROPE;
    if (!positions) fail("rope=True needs positions");
    pos_ptr = indices(positions, "positions", T);
    if (!table) {
      const Owned device(PyObject_GetAttrString(k.o, "device"));
      made = raise_if_null(PyObject_CallFunction(rope_table_of, "Od", device.p, theta));
      Py_DECREF(made);               // the package keeps its tables
      table = tensor(made, "table");
    }
    require_dtype(table, at::kInt, "table", "torch.int32");
    if (!table->is_contiguous()) fail("table must be contiguous");
    table_len = i32(table->numel() / 64, "table");
    if (table_len) table_ptr = table.ptr();
  }
  const double eps = number(args[8]);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  at::Tensor q_out;
  if (given) {
    q_out = *given.t;
  } else if (q) {
    q_out = at::empty({T, rq.heads, p.D}, k->options());
    ro = {rq.heads, rq.heads * p.D, q_out.data_ptr()};
  }
  int32_t *const err = error_flag(dev);
  const cudaStream_t stream = stream_of(dev);
  const int32_t hq = i32(rq.heads, "Hq");
  enter(1, [&] {
    return store_entry(rq.ptr, rk.ptr, rv.ptr, qw_ptr, kw_ptr, pos_ptr, slot_ptr, ro.ptr, p.k, p.v,
                       p.ks, p.vs, p.code, T, hq, p.hkv, p.D, p.nb, p.bs, p.sb, p.st, p.sh, p.cb,
                       p.ch, rq.stride, rk.stride, rv.stride, ro.stride, table_ptr, table_len, eps,
                       static_cast<float>(theta), flags, err, stream);
  });
  if (!q) Py_RETURN_NONE;
  if (given) return Py_NewRef(given.o);
  return THPVariable_Wrap(std::move(q_out));
}

// (q, cache, block_tables, context_lens, scale, out, workspace)
PyObject *paged_decode(PyObject *const *args) {
  const Arg q = tensor(args[0], "q");
  Pool p = pool_tensors(args[1]);
  const Arg bt = tensor(args[2], "block_tables"), lens = tensor(args[3], "context_lens");
  const Arg given = maybe(args[5], "out"), scratch = maybe(args[6], "workspace");
  const int dev = device_of({&q, &p.data, &p.scales, &bt, &lens, &given, &scratch});
  check_pool(p);
  check_q(q, "batch");
  check_heads(q, p);
  const int32_t B = i32(q->size(0), "batch"), hq = i32(q->size(1), "Hq");
  const Tables t = tables(bt, lens, B);
  const float scale = static_cast<float>(args[4] == Py_None ? 1.0 / std::sqrt(p.D) : number(args[4]));
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  at::Tensor out = output(given, q);
  const size_t need = workspace_entry(B, hq, p.hkv, p.D, t.width, p.bs);
  at::Tensor ws;
  if (!scratch) {
    ws = at::empty({static_cast<int64_t>(need)}, q->options().dtype(at::kByte));
  } else {
    ws = *scratch.t;
    if (ws.scalar_type() != at::kByte || static_cast<size_t>(ws.numel()) < need || !ws.is_contiguous()) {
      fail("decode workspace must be contiguous uint8 with >= %zu bytes", need);
    }
  }
  const void *q_ptr = q.ptr();
  void *out_ptr = out.data_ptr(), *ws_ptr = ws.data_ptr();
  const size_t ws_bytes = ws.numel();
  int32_t *const err = error_flag(dev);
  const cudaStream_t stream = stream_of(dev);
  enter(2, [&] {
    return decode_entry(q_ptr, p.k, p.v, p.ks, p.vs, p.code, t.ptr, t.lens, out_ptr, B, hq, p.hkv,
                        p.D, p.nb, p.bs, t.width, t.stride, p.sb, p.st, p.sh, p.cb, p.ch, scale,
                        ws_ptr, ws_bytes, err, stream);
  });
  return given ? Py_NewRef(given.o) : THPVariable_Wrap(std::move(out));
}

// Rows of n sequences, from the first of t's, into packed K, then V, at `out`.
void read_back(const Pool &p, const Tables &t, void *out, int32_t n, int32_t len, int32_t zero_to,
               cudaStream_t stream) {
  uint8_t *const k_out = static_cast<uint8_t *>(out);
  uint8_t *const v_out = k_out + static_cast<int64_t>(n) * len * p.hkv * p.D * 2;
  enter(1, [&] {
    return read_entry(p.k, p.v, p.ks, p.vs, p.code, t.ptr, t.lens, k_out, v_out, n, len, zero_to,
                      p.hkv, p.D, p.nb, p.bs, t.width, t.stride, p.sb, p.st, p.sh, p.cb, p.ch,
                      stream);
  });
}

// (cache, block_tables, context_lens, max_context_len, out)
PyObject *read_kv_cache(PyObject *const *args) {
  Pool p = pool_tensors(args[0]);
  const Arg bt = tensor(args[1], "block_tables"), lens = tensor(args[2], "context_lens");
  const Arg given = maybe(args[4], "out");
  const int dev = device_of({&p.data, &p.scales, &bt, &lens, &given});
  check_pool(p);
  const int32_t B = i32(bt->dim() > 0 ? bt->size(0) : 0, "batch");
  const Tables t = tables(bt, lens, B);
  const int64_t most = integer(args[3]);
  if (most < 0) fail("max_context_len must not be negative");
  const int32_t len = i32(most ? most : static_cast<int64_t>(t.width) * p.bs, "max_context_len");
  const std::initializer_list<int64_t> shape = {2, B, len, p.hkv, p.D};
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  at::Tensor out;
  if (!given) {
    out = at::empty(shape, p.data->options().dtype(at::kBFloat16));
  } else {
    out = *given.t;
    if (out.sizes() != at::IntArrayRef(shape) || out.scalar_type() != at::kBFloat16 ||
        !out.is_contiguous()) {
      fail("out must be a contiguous bf16 tensor of shape (2, %d, %d, %d, %d)", B, len, p.hkv, p.D);
    }
  }
  read_back(p, t, out.data_ptr(), B, len, 0, stream_of(dev));
  return given ? Py_NewRef(given.o) : THPVariable_Wrap(std::move(out));
}

// Whether to take the pages in directly instead of reading the contexts back first, by
// what each way takes in us, fitted to 40 shapes of 1 to 2000 new tokens after 0 to 13854
// (B200). A wave of CTAs costs its start and so much per key tile; direct, a CTA has one
// row tile of 128 rows and converts its keys; read back, it has two and takes them
// ready, after a launch that writes them. Both join what a split over keys leaves.
// Measured read back / direct, 32 / 8 heads: 1 token after 1421 15.5 / 11.9; 32 after
// 11129 35.6 / 22.3; 2 x 256 after 347 22 / 16.6; 300 after 2774 36 / 51; 2 x 600 after
// 1420 66 / 82.
bool direct_prefill(int64_t S, int64_t T, int64_t hq, const Pool &p, int64_t longest, int64_t len,
                    size_t direct_bytes, size_t back_bytes) {
  const int64_t g = hq / p.hkv;
  if (S == 0 || T == 0) return true;
  if (g == 0 || 128 % g != 0) return false;            // the other way refuses it
  const int64_t part_bytes = std::min(T, S * longest) * hq * (p.D + 2) * 4, keys = (len + 127) / 128;
  auto cost = [&](int64_t rows, size_t bytes, double start, double tile) {
    const int64_t tt = rows / g, tiles = std::min((longest + tt - 1) / tt * S, T / tt + S);
    const int64_t parts = std::max<int64_t>(1, bytes / part_bytes);
    const int64_t waves = (tiles * p.hkv * parts + num_sms() - 1) / num_sms();
    return waves * (start + tile * ((keys + parts - 1) / parts)) +
           (parts > 1 ? 2.5 + 2.0 * bytes / 6e6 : 0.0);
  };
  const double read_back = S * len * p.hkv * 770.0 / 6e6;            // both ways through HBM
  return 2.0 + cost(128, direct_bytes, 5.5, 1.8) <= 5.0 + cost(256, back_bytes, 5.0, 1.45) + read_back;
}

// (q, cache, block_tables, cu_seqlens_q, context_lens, max_seqlen_q, scale, out,
//  max_context_len, scratch_rows)
PyObject *paged_prefill(PyObject *const *args) {
  constexpr int32_t kPage = 16, kKeyTile = 128;      // keys a prefill tile reads at once
  const Arg q = tensor(args[0], "q");
  Pool p = pool_tensors(args[1]);
  const Arg bt = tensor(args[2], "block_tables"), cu = tensor(args[3], "cu_seqlens_q");
  Arg lens = maybe(args[4], "context_lens");
  const Arg given = maybe(args[7], "out");
  const int dev = device_of({&q, &p.data, &p.scales, &bt, &cu, &lens, &given});
  check_pool(p);
  require_dtype(cu, at::kInt, "cu_seqlens_q", "torch.int32");
  check_q(q, "num_tokens");
  if (cu->dim() != 1 || cu->size(0) < 1 || !cu->is_contiguous()) {
    fail("cu_seqlens_q must be a contiguous [num_seqs + 1] tensor");
  }
  check_heads(q, p);
  const int32_t S = i32(cu->size(0) - 1, "num_seqs"), hq = i32(q->size(1), "Hq");
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  at::Tensor new_tokens;
  if (!lens) {
    new_tokens = at::sub(cu->slice(0, 1, S + 1), cu->slice(0, 0, S));
    lens = {cu.o, &new_tokens};
  }
  const Tables t = tables(bt, lens, S);
  const int32_t max_new = i32(integer(args[5]), "max_seqlen_q");
  const int64_t bound = integer(args[8]), capacity = static_cast<int64_t>(t.width) * p.bs;
  if (bound < 0) fail("max_context_len must not be negative");
  const int64_t most = std::min(bound ? bound : capacity, capacity);
  // whole key tiles: a tile's keys behind a context are zeros of its own, not another's rows
  const int32_t len =
      i32(std::max<int64_t>((most + kKeyTile - 1) / kKeyTile, 1) * kKeyTile, "max_context_len");
  const float scale = static_cast<float>(args[6] == Py_None ? 1.0 / std::sqrt(p.D) : number(args[6]));
  at::Tensor out = output(given, q);
  const int64_t T = q->size(0);
  const void *q_ptr = q.ptr();
  void *const out_ptr = out.data_ptr();
  const int32_t *const cu_ptr = static_cast<const int32_t *>(cu.ptr());
  int32_t *const err = error_flag(dev);
  const cudaStream_t stream = stream_of(dev);
  const size_t need = direct_workspace_entry(T, S, hq, p.hkv, p.D, max_new, len);
  if (direct_prefill(S, T, hq, p, max_new > 0 ? max_new : T, len, need,
                     prefill_workspace_entry(T, S, hq, p.hkv, p.D, max_new, len))) {
    at::Tensor ws;
    if (need) ws = at::empty({static_cast<int64_t>(need)}, q->options().dtype(at::kByte));
    void *const ws_ptr = need ? ws.data_ptr() : nullptr;
    enter(need ? 2 : 1, [&] {
      return direct_entry(q_ptr, p.k, p.v, p.ks, p.vs, p.code, t.ptr, cu_ptr, t.lens, out_ptr, T, S,
                          hq, p.hkv, p.D, p.nb, p.bs, t.width, t.stride, p.sb, p.st, p.sh, p.cb,
                          p.ch, max_new, len, scale, ws_ptr, need, err, stream);
    });
    return given ? Py_NewRef(given.o) : THPVariable_Wrap(std::move(out));
  }
  // the scratch: K and V, where page i of a group's sequence b is block b * per_seq
  // + i, then what a split over keys needs
  const int64_t row = static_cast<int64_t>(p.hkv) * p.D;
  const int64_t most_seqs = std::max<int64_t>(
      1, std::min<int64_t>(S, integer(args[9]) / (static_cast<int64_t>(len) * p.hkv)));
  // groups of the same size, or one sequence less
  const int64_t groups = S ? (S + most_seqs - 1) / most_seqs : 1, group = (S + groups - 1) / groups;
  const int32_t per_seq = len / kPage;
  size_t split_bytes = 0;               // (a smaller group may be split further)
  for (int64_t n = group; n >= std::max<int64_t>(group - 1, 0); --n) {
    split_bytes = std::max(split_bytes, prefill_workspace_entry(T, static_cast<int32_t>(n), hq, p.hkv,
                                                                p.D, max_new, len));
  }
  const at::Tensor scratch = at::empty(
      {2 * group * len * row + static_cast<int64_t>(split_bytes / 2)}, q->options());
  void *const k_ptr = scratch.data_ptr();
  void *const ws = static_cast<uint8_t *>(k_ptr) + 4 * group * len * row;
  for (int64_t i = 0; i < groups; ++i) {
    const int64_t s = S * i / groups;
    const int32_t n = static_cast<int32_t>(S * (i + 1) / groups - s);
    const Tables part = {t.ptr + s * t.stride, t.lens + s, t.width, t.stride};
    read_back(p, part, k_ptr, n, len, kKeyTile, stream);
    const size_t part_need = prefill_workspace_entry(T, n, hq, p.hkv, p.D, max_new, len);
    // the rows behind the last sequence are zeroed once, when all queries are read: out may be q
    const auto attend = s + n < S ? prefill_part_entry : prefill_entry;
    enter(part_need > 0 ? 2 : 1, [&] {
      return attend(q_ptr, k_ptr, static_cast<uint8_t *>(k_ptr) + n * len * row * 2, nullptr,
                    cu_ptr + s, part.lens, out_ptr, T, n, hq, p.hkv, p.D,
                    static_cast<int64_t>(std::max(n, 1)) * per_seq, kPage, per_seq, per_seq,
                    kPage * row, row, p.D, max_new, len, scale, ws, part_need, err, stream);
    });
  }
  return given ? Py_NewRef(given.o) : THPVariable_Wrap(std::move(out));
}

// (addresses of the nine entries in the order above, then the three objects)
PyObject *bind(PyObject *const *args) {
  store_entry = reinterpret_cast<decltype(store_entry)>(integer(args[0]));
  decode_entry = reinterpret_cast<decltype(decode_entry)>(integer(args[1]));
  workspace_entry = reinterpret_cast<decltype(workspace_entry)>(integer(args[2]));
  read_entry = reinterpret_cast<decltype(read_entry)>(integer(args[3]));
  prefill_entry = reinterpret_cast<decltype(prefill_entry)>(integer(args[4]));
  prefill_part_entry = reinterpret_cast<decltype(prefill_part_entry)>(integer(args[5]));
  prefill_workspace_entry = reinterpret_cast<decltype(prefill_workspace_entry)>(integer(args[6]));
  direct_entry = reinterpret_cast<decltype(direct_entry)>(integer(args[7]));
  direct_workspace_entry = reinterpret_cast<decltype(direct_workspace_entry)>(integer(args[8]));
  native = Py_NewRef(args[9]);
  error_flag_of = Py_NewRef(args[10]);
  rope_table_of = Py_NewRef(args[11]);
  Py_RETURN_NONE;
}

template <PyObject *(*kCall)(PyObject *const *), int kArgs>
PyObject *method(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != kArgs) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", kArgs, n);
    return nullptr;
  }
  try {
    return kCall(args);
  } catch (const Raised &) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

template <PyObject *(*kCall)(PyObject *const *), int kArgs>
PyMethodDef entry(const char *name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&method<kCall, kArgs>)),
          METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {entry<kv_store, 14>("kv_store"), entry<paged_decode, 7>("paged_decode"),
                         entry<read_kv_cache, 5>("read_kv_cache"),
                         entry<paged_prefill, 10>("paged_prefill"), entry<bind, 12>("bind"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_calls", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__torch_calls() {
  PyObject *const m = PyModule_Create(&module);
  // read from the file before it is loaded, too
  if (m && PyModule_AddStringConstant(m, "target", VJ_CALLS_TARGET) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
