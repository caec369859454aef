// The kv8 operators' way from torch tensors to libsdv: a Python extension module whose functions take
// the plain case of an operator's arguments -- tensors as the library takes them -- straight to the C
// ABI.  Anything else returns None, and the caller's general path copies what may be copied and says
// what is wrong with the rest.
//
// An engine calls these operators once per layer and token, so their host time is part of every token:
// the checks of ten tensors' types, shapes, strides and devices, the stream, the workspace and a call
// with 25 arguments through ctypes took 7 to 10 us, of which this leaves about 1 beside the launch.
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <unordered_map>

#include "sdv.h"

namespace {

decltype(&sdv_kv8_append) g_append;
decltype(&sdv_kv8_gather) g_gather;
decltype(&sdv_kv8_attention_slot) g_attention;
decltype(&sdv_kv8_attention_workspace_size) g_workspace_size;
decltype(&sdv_rope) g_rope;
decltype(&sdv_kv8_rope_append) g_rope_append;
decltype(&sdv_copy_blocks) g_copy;
decltype(&sdv_kv8_keep) g_keep;
decltype(&sdv_kv8_shared_attention) g_shared;
decltype(&sdv_kv8_shared_attention_workspace_size) g_shared_size;
decltype(&sdv_kv8_shared_attention_tile_rows) g_shared_rows;

// A tensor of no subclass (whose data might not be where it says), or nullptr.
const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool whole(PyObject* o, int64_t& v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow == 0 && v >= 0 && v <= INT32_MAX;
}

struct Pages {
  c10::Device device = c10::Device(c10::kCPU);
  int32_t blocks, kv, d, format, batch, max_blocks;
  void *k, *v;
  float* s;
  const int32_t* table;
};

bool fits(const at::Tensor& t, c10::Device dev, at::ScalarType type) {
  return t.device() == dev && t.scalar_type() == type && t.is_contiguous();
}

bool pages(PyObject* const* o, Pages& p) {
  const at::Tensor *k = tensor(o[0]), *v = tensor(o[1]), *s = tensor(o[2]), *bt = tensor(o[3]);
  if (!k || !v || !s || !bt || !k->is_cuda()) return false;
  p.device = k->device();
  const at::ScalarType type = k->scalar_type();
  if (type == at::kFloat8_e4m3fn)
    p.format = SDV_KV8_FP8;
  else if (type == at::kChar)
    p.format = SDV_KV8_INT8;
  else
    return false;
  if (k->dim() != 6 || v->dim() != 4 || s->dim() != 4 || bt->dim() != 2 || !fits(*k, p.device, type) || !fits(*v, p.device, type) ||
      !fits(*s, p.device, at::kFloat) || !fits(*bt, p.device, at::kInt))
    return false;
  const int64_t nb = k->size(0), kv = k->size(1), dc = k->size(3);
  if (k->size(2) != 4 || k->size(4) != 4 || k->size(5) != 16 || v->size(0) != nb || v->size(1) != kv || v->size(2) != dc * 16 ||
      v->size(3) != 16 || s->size(0) != nb || s->size(1) != kv || s->size(2) != 2 || s->size(3) != 16)
    return false;
  if (nb > INT32_MAX || kv > INT32_MAX || dc > 64 || bt->size(0) > INT32_MAX || bt->size(1) > INT32_MAX) return false;
  p.blocks = (int32_t)nb;
  p.kv = (int32_t)kv;
  p.d = (int32_t)dc * 16;
  p.batch = (int32_t)bt->size(0);
  p.max_blocks = (int32_t)bt->size(1);
  p.k = k->data_ptr();
  p.v = v->data_ptr();
  p.s = static_cast<float*>(s->data_ptr());
  p.table = static_cast<const int32_t*>(bt->data_ptr());
  return true;
}

// Packed BF16 rows (total, heads, D) whose tokens lie `stride` elements apart.
const at::Tensor* rows_of(PyObject* o, c10::Device dev, int64_t d, int64_t heads, int64_t& stride) {
  const at::Tensor* t = tensor(o);
  if (!t || t->dim() != 3 || t->scalar_type() != at::kBFloat16 || t->device() != dev) return nullptr;
  const int64_t n = t->size(0), h = t->size(1);
  if (t->size(2) != d || (heads && h != heads) || n == 0 || n > INT32_MAX || h > INT32_MAX) return nullptr;
  stride = n == 1 ? h * d : t->stride(0);
  if (t->stride(2) != 1 || (t->stride(1) != d && h != 1) || stride < h * d || stride % 8 != 0 ||
      reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 != 0)
    return nullptr;
  return t;
}
const at::Tensor* rows(PyObject* o, const Pages& p, int64_t heads, int64_t& stride) { return rows_of(o, p.device, p.d, heads, stride); }

bool ints_of(PyObject* o, c10::Device dev, int64_t n, const int32_t*& at) {
  const at::Tensor* t = tensor(o);
  if (!t || t->dim() != 1 || t->size(0) != n || !fits(*t, dev, at::kInt)) return false;
  at = static_cast<const int32_t*>(t->data_ptr());
  return true;
}
bool ints(PyObject* o, const Pages& p, int64_t n, const int32_t*& at) { return ints_of(o, p.device, n, at); }

bool real(PyObject* o, double& v) {
  if (!PyFloat_CheckExact(o)) return false;
  v = PyFloat_AS_DOUBLE(o);
  return true;
}

bool truth(PyObject* o, int32_t& v) {
  v = o == Py_True;
  return v || o == Py_False;
}

// The rotated dimensions that fp64 frequencies stand for, or 0.
int32_t frequencies(PyObject* o, c10::Device dev, int64_t d, const double*& at) {
  const at::Tensor* t = tensor(o);
  if (!t || t->dim() != 1 || !fits(*t, dev, at::kDouble)) return 0;
  const int64_t n = 2 * t->size(0);
  if (n <= 0 || n > d || n % 16 != 0) return 0;
  at = static_cast<const double*>(t->data_ptr());
  return (int32_t)n;
}

bool lengths(PyObject* o, const Pages& p, const int32_t*& at) {
  at = nullptr;
  return o == Py_None || ints(o, p, p.batch, at);
}

// The current device, made the tensors' for the call, and its stream.
struct Launch {
  c10::OptionalDeviceGuard guard;
  hipStream_t stream;
  explicit Launch(c10::Device dev) : guard(dev), stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream()) {}
  explicit Launch(const Pages& p) : Launch(p.device) {}
};

// A BF16 tensor, without the dispatcher's way there: rope's two outputs cost its caller 0.6 us less (5.8 -> 5.2 a call).
at::Tensor bf16(at::IntArrayRef size, c10::Device dev) { return at::detail::empty_cuda(size, at::kBFloat16, dev, std::nullopt); }

// kv8_attention's workspace lives as long as the call (its memory is used again in the order of the stream),
// so that nothing of a graph's memory, or of another private pool that is current, outlives it.  What
// has to be zero between calls is a slot of the library's: one per device and stream for eager calls, which
// their stream orders, and one per recording and stream, so that no two graphs share one.  A slot that a
// recording has had is not given out again, as the graph may be replayed at any time.  Without a slot (-1:
// all given out, or a stream whose handle names another one in each thread) the workspace's own counts are
// zeroed, by a fill of 1.8 us where a short call takes 8.
constexpr int32_t kEagerSlots = 256;

int32_t count_slot(const Pages& p, hipStream_t stream) {
  struct Key {
    int device;
    hipStream_t stream;
    bool operator==(const Key& o) const { return device == o.device && stream == o.stream; }
  };
  struct Hash {
    size_t operator()(const Key& k) const { return std::hash<void*>()(k.stream) * 31 + k.device; }
  };
  struct Slots {
    int32_t eager = -1;
    unsigned long long recording = 0;  // the last, and its slot
    int32_t recorded = -1;
  };
  struct Given {
    int32_t eager = 0, recorded = kEagerSlots;
  };
  static auto* slots = new std::unordered_map<Key, Slots, Hash>();  // never freed: the runtime may end before them
  static auto* given = new std::unordered_map<int, Given>();        // by device
  if (stream == hipStreamPerThread) return -1;
  Slots& s = (*slots)[{p.device.index(), stream}];
  Given& g = (*given)[p.device.index()];
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) {
    if (s.eager < 0 && g.eager < kEagerSlots) s.eager = g.eager++;
    return s.eager;
  }
  hipStreamCaptureStatus capture;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo(stream, &capture, &id) != hipSuccess || capture != hipStreamCaptureStatusActive || id == 0) return -1;
  if (s.recording != id) {
    s.recording = id;
    s.recorded = g.recorded < SDV_KV8_SLOTS ? g.recorded++ : -1;
  }
  return s.recorded;
}

PyObject* status(int st) { return PyLong_FromLong(st); }

// append(k_new, v_new, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_seq_len) -> status
PyObject* append(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pages p;
  int64_t ks, vs, max_len;
  const int32_t *cu, *lens;
  if (!g_append || n != 9 || !pages(o + 2, p) || !whole(o[8], max_len)) Py_RETURN_NONE;
  const at::Tensor *k = rows(o[0], p, p.kv, ks), *v = rows(o[1], p, p.kv, vs);
  if (!k || !v || k->size(0) != v->size(0) || !ints(o[6], p, p.batch + 1, cu) || !lengths(o[7], p, lens) || (!lens && max_len == 0))
    Py_RETURN_NONE;
  Launch on(p);
  return status(g_append(k->data_ptr(), v->data_ptr(), ks, vs, (int32_t)k->size(0), p.k, p.v, p.s, p.blocks, p.format, p.table,
                         p.max_blocks, cu, lens, (int32_t)max_len, p.batch, p.kv, p.d, on.stream));
  END_HANDLE_TH_ERRORS
}

// gather(k_pages, v_pages, scales, block_table, cu_rows, starts, total_rows) -> (k, v) or status
PyObject* gather(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pages p;
  int64_t total;
  const int32_t *cu, *starts;
  if (!g_gather || n != 7 || !pages(o, p) || !whole(o[6], total) || total == 0 || !ints(o[4], p, p.batch + 1, cu) || !ints(o[5], p, p.batch, starts))
    Py_RETURN_NONE;
  Launch on(p);
  const auto options = at::TensorOptions().dtype(at::kBFloat16).device(p.device);
  at::Tensor k = at::empty({total, p.kv, p.d}, options), v = at::empty({total, p.kv, p.d}, options);
  const int64_t stride = (int64_t)p.kv * p.d;
  const int st = g_gather(p.k, p.v, p.s, p.blocks, p.format, p.table, p.max_blocks, cu, starts, p.batch, (int32_t)total, p.kv, p.d,
                          k.data_ptr(), v.data_ptr(), stride, stride, on.stream);
  if (st != SDV_OK) return status(st);
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(k)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(v)));
  return out;
  END_HANDLE_TH_ERRORS
}

// attention(q, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_q_len, max_seq_len, scale,
//           tree_mask, out = None) -> out or status.  The GIL is held from the workspace to the last launch:
// the launches of one call stand together on their stream, whichever threads call.
PyObject* attention(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pages p;
  int64_t q_row, out_row, max_q, max_len;
  const int32_t *cu, *lens;
  if (!g_attention || (n != 11 && n != 12) || !pages(o + 1, p) || !whole(o[7], max_q) || !whole(o[8], max_len)) Py_RETURN_NONE;
  const at::Tensor* q = rows(o[0], p, 0, q_row);
  if (!q || !ints(o[5], p, p.batch + 1, cu) || !lengths(o[6], p, lens)) Py_RETURN_NONE;
  const int64_t total = q->size(0), heads = q->size(1);
  double scale = 1.0 / std::sqrt((double)p.d);
  if (o[9] != Py_None) {
    if (!PyFloat_CheckExact(o[9])) Py_RETURN_NONE;
    scale = PyFloat_AS_DOUBLE(o[9]);
  }
  const uint64_t* tree = nullptr;
  if (o[10] != Py_None) {
    const at::Tensor* t = tensor(o[10]);
    if (!t || max_q > 64 || t->dim() != 1 || t->size(0) != total ||
        !fits(*t, p.device, t->scalar_type() == at::kUInt64 ? at::kUInt64 : at::kLong))
      Py_RETURN_NONE;
    tree = static_cast<const uint64_t*>(t->data_ptr());
  }
  const size_t bytes = g_workspace_size(p.batch, (int32_t)total, (int32_t)heads, p.kv, p.d, (int32_t)max_q, (int32_t)max_len);
  if (bytes == 0) Py_RETURN_NONE;  // sizes that the general path refuses
  const at::Tensor* given = nullptr;
  if (n == 12 && o[11] != Py_None) {
    given = rows(o[11], p, heads, out_row);
    if (!given || given->size(0) != total) Py_RETURN_NONE;
  }
  Launch on(p);
  at::Tensor out;
  if (!given) {
    out = at::empty({total, heads, p.d}, q->options());
    out_row = heads * p.d;
  }
  const int32_t slot = count_slot(p, on.stream);
  const c10::DataPtr ws = c10::hip::HIPCachingAllocator::get()->allocate(bytes);
  if (slot < 0)
    at::from_blob(ws.get(), {SDV_KV8_SYNC_BYTES}, at::TensorOptions().dtype(at::kByte).device(p.device)).zero_();
  const int st = g_attention(q->data_ptr(), q_row, p.k, p.v, p.s, p.blocks, p.format, p.table, p.max_blocks, cu, lens, tree, p.batch,
                             (int32_t)total, (int32_t)heads, p.kv, p.d, (int32_t)max_q, (int32_t)max_len, (float)scale, ws.get(),
                             bytes, slot, given ? given->data_ptr() : out.data_ptr(), out_row, on.stream);
  if (st != SDV_OK) return status(st);
  if (given) {
    Py_INCREF(o[11]);
    return o[11];
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// rope(q, k or None, positions, inv_freq, interleaved, scale, inverse) -> (q, k or None) or status
PyObject* rope(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t qs, ks = 0, heads = 0;
  double scale;
  int32_t interleaved, inverse;
  const int32_t* positions;
  const double* inv_freq;
  if (!g_rope || n != 7 || !truth(o[4], interleaved) || !real(o[5], scale) || !truth(o[6], inverse)) Py_RETURN_NONE;
  const at::Tensor* first = tensor(o[0]);
  if (!first || first->dim() != 3 || !first->is_cuda()) Py_RETURN_NONE;
  const c10::Device dev = first->device();
  const int64_t d = first->size(2);
  const at::Tensor *q = rows_of(o[0], dev, d, 0, qs), *k = nullptr;
  if (!q || (o[1] != Py_None && !(k = rows_of(o[1], dev, d, 0, ks))) || !ints_of(o[2], dev, q->size(0), positions)) Py_RETURN_NONE;
  if (k && k->size(0) != q->size(0)) Py_RETURN_NONE;
  if (c10::GradMode::is_enabled() && (q->requires_grad() || (k && k->requires_grad()))) Py_RETURN_NONE;
  const int32_t rotary = frequencies(o[3], dev, d, inv_freq);
  if (rotary == 0) Py_RETURN_NONE;
  Launch on(dev);
  at::Tensor q_out = bf16({q->size(0), q->size(1), d}, dev), k_out;
  if (k) {
    heads = k->size(1);
    k_out = bf16({k->size(0), heads, d}, dev);
  }
  const int st = g_rope(q->data_ptr(), qs, (int32_t)q->size(1), k ? k->data_ptr() : nullptr, ks, (int32_t)heads, positions, inv_freq, rotary,
                        interleaved, (float)scale, inverse, (int32_t)q->size(0), (int32_t)d, q_out.data_ptr(), q->size(1) * d,
                        k ? k_out.data_ptr() : nullptr, heads * d, on.stream);
  if (st != SDV_OK) return status(st);
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(q_out)));
  if (!k) Py_INCREF(Py_None);
  PyTuple_SET_ITEM(out, 1, k ? THPVariable_Wrap(std::move(k_out)) : Py_None);
  return out;
  END_HANDLE_TH_ERRORS
}

// rope_append(q, k_new, v_new, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_seq_len, inv_freq,
//             interleaved, scale, positions or None) -> q or status
PyObject* rope_append(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pages p;
  int64_t qs, ks, vs, max_len;
  double scale;
  int32_t interleaved;
  const int32_t *cu, *lens, *positions = nullptr;
  const double* inv_freq;
  if (!g_rope_append || n != 14 || !pages(o + 3, p) || !whole(o[9], max_len) || !truth(o[11], interleaved) || !real(o[12], scale)) Py_RETURN_NONE;
  const at::Tensor *q = rows(o[0], p, 0, qs), *k = rows(o[1], p, p.kv, ks), *v = rows(o[2], p, p.kv, vs);
  if (!q || !k || !v || q->size(0) != k->size(0) || v->size(0) != k->size(0) || !ints(o[7], p, p.batch + 1, cu) || !lengths(o[8], p, lens) ||
      (!lens && max_len == 0) || (o[13] != Py_None && !ints(o[13], p, q->size(0), positions)))
    Py_RETURN_NONE;
  const int32_t rotary = frequencies(o[10], p.device, p.d, inv_freq);
  if (rotary == 0) Py_RETURN_NONE;
  Launch on(p);
  const int64_t heads = q->size(1);
  at::Tensor out = bf16({q->size(0), heads, p.d}, p.device);
  const int st = g_rope_append(q->data_ptr(), qs, out.data_ptr(), heads * p.d, (int32_t)heads, k->data_ptr(), v->data_ptr(), ks, vs,
                               (int32_t)q->size(0), p.k, p.v, p.s, p.blocks, p.format, p.table, p.max_blocks, cu, lens, (int32_t)max_len,
                               p.batch, p.kv, p.d, positions, inv_freq, rotary, interleaved, (float)scale, on.stream);
  if (st != SDV_OK) return status(st);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// The blocks of a layer (or of layers): K, V and scale tensors whose first dimensions are [layers,] blocks, KV heads.
struct Blocks {
  const at::Tensor* t[3];
  int64_t layers, blocks, bytes[3];
};

bool blocks(PyObject* const* o, Blocks& b) {
  for (int i = 0; i < 3; ++i)
    if (!(b.t[i] = tensor(o[i])) || !b.t[i]->is_cuda() || !b.t[i]->is_contiguous() || b.t[i]->device() != b.t[0]->device()) return false;
  const int64_t dim = b.t[1]->dim();
  if ((dim != 4 && dim != 5) || b.t[2]->scalar_type() != at::kFloat) return false;
  const int lead = (int)dim - 4;
  b.layers = lead ? b.t[1]->size(0) : 1;
  b.blocks = b.t[1]->size(lead);
  if (b.layers <= 0 || b.blocks <= 0 || b.blocks > INT32_MAX || b.layers > INT32_MAX) return false;
  for (const at::Tensor* t : b.t) {
    if (t->dim() < lead + 3) return false;
    for (int i = 0; i < lead + 2; ++i)
      if (t->size(i) != b.t[1]->size(i)) return false;
  }
  for (int i = 0; i < 3; ++i) b.bytes[i] = b.t[i]->numel() / (b.layers * b.blocks) * (int64_t)b.t[i]->element_size();
  return true;
}

// copy_blocks(k, v, scales, src, dst, k_to, v_to, scales_to) -> status
PyObject* copy_blocks(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Blocks from, to;
  if (!g_copy || n != 8 || !blocks(o, from) || !blocks(o + 5, to) || to.t[0]->device() != from.t[0]->device() || to.layers != from.layers) Py_RETURN_NONE;
  for (int i = 0; i < 3; ++i) {
    if (to.t[i]->dim() != from.t[i]->dim() || to.t[i]->scalar_type() != from.t[i]->scalar_type()) Py_RETURN_NONE;
    const int64_t dim = from.t[1]->dim() - 4;
    for (int64_t j = dim + 1; j < to.t[i]->dim(); ++j)
      if (to.t[i]->size(j) != from.t[i]->size(j)) Py_RETURN_NONE;
  }
  const c10::Device dev = from.t[0]->device();
  const at::Tensor* ids = tensor(o[3]);
  const int32_t *src, *dst;
  if (!ids || ids->dim() != 1 || ids->size(0) > INT32_MAX || !ints_of(o[3], dev, ids->size(0), src) || !ints_of(o[4], dev, ids->size(0), dst)) Py_RETURN_NONE;
  if (ids->size(0) == 0) return status(SDV_OK);
  Launch on(dev);
  return status(g_copy(from.t[0]->data_ptr(), from.t[1]->data_ptr(), static_cast<const float*>(from.t[2]->data_ptr()), (int32_t)from.blocks,
                       to.t[0]->data_ptr(), to.t[1]->data_ptr(), static_cast<float*>(to.t[2]->data_ptr()), (int32_t)to.blocks, from.bytes[0],
                       from.bytes[1], from.bytes[2], (int32_t)from.layers, src, dst, (int32_t)ids->size(0), on.stream));
  END_HANDLE_TH_ERRORS
}

// keep(k_pages, v_pages, scales, block_table, cu_kept, kept, starts) -> status
PyObject* keep(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Blocks b;
  if (!g_keep || n != 7 || !blocks(o, b)) Py_RETURN_NONE;
  const at::Tensor &k = *b.t[0], &v = *b.t[1], &s = *b.t[2], *bt = tensor(o[3]), *ids = tensor(o[5]);
  const c10::Device dev = k.device();
  const int64_t lead = v.dim() - 4, kv = v.size(lead + 1), d = v.size(lead + 2);
  if (k.dim() != lead + 6 || s.dim() != lead + 4 || k.scalar_type() != v.scalar_type() ||
      (k.scalar_type() != at::kFloat8_e4m3fn && k.scalar_type() != at::kChar) || k.size(lead + 2) != 4 || k.size(lead + 3) * 16 != d ||
      k.size(lead + 4) != 4 || k.size(lead + 5) != 16 || v.size(lead + 3) != 16 || s.size(lead + 2) != 2 || s.size(lead + 3) != 16)
    Py_RETURN_NONE;
  if (!bt || bt->dim() != 2 || !fits(*bt, dev, at::kInt) || bt->size(0) > INT32_MAX || bt->size(1) > INT32_MAX || !ids || ids->dim() != 1 ||
      ids->size(0) > INT32_MAX || kv > INT32_MAX || d > INT32_MAX)
    Py_RETURN_NONE;
  const int32_t *cu, *kept, *starts;
  if (!ints_of(o[4], dev, bt->size(0) + 1, cu) || !ints_of(o[5], dev, ids->size(0), kept) || !ints_of(o[6], dev, bt->size(0), starts)) Py_RETURN_NONE;
  if (ids->size(0) == 0) return status(SDV_OK);
  Launch on(dev);
  return status(g_keep(k.data_ptr(), v.data_ptr(), static_cast<float*>(s.data_ptr()), (int32_t)b.blocks, k.numel() / b.layers,
                       v.numel() / b.layers, s.numel() / b.layers, (int32_t)b.layers, static_cast<const int32_t*>(bt->data_ptr()),
                       (int32_t)bt->size(1), cu, kept, (int32_t)ids->size(0), starts, (int32_t)bt->size(0), (int32_t)kv, (int32_t)d, on.stream));
  END_HANDLE_TH_ERRORS
}

// shared(q, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_q_len, max_seq_len, cu_groups, prefix_lens,
//        max_prefix_len, scale, tree_mask, tile_rows, out = None) -> out or status
PyObject* shared(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pages p;
  int64_t q_row, out_row, max_q, max_len, max_prefix, tile;
  const int32_t *cu, *lens, *groups, *prefix;
  if (!g_shared || (n != 15 && n != 16) || !pages(o + 1, p) || !whole(o[7], max_q) || !whole(o[8], max_len) || !whole(o[11], max_prefix) ||
      !whole(o[14], tile))
    Py_RETURN_NONE;
  const at::Tensor *q = rows(o[0], p, 0, q_row), *cg = tensor(o[9]);
  if (!q || !ints(o[5], p, p.batch + 1, cu) || !lengths(o[6], p, lens) || !cg || cg->dim() != 1 || cg->size(0) < 1 || cg->size(0) > p.batch + 1 ||
      !ints(o[9], p, cg->size(0), groups) || !ints(o[10], p, p.batch, prefix))
    Py_RETURN_NONE;
  const int64_t total = q->size(0), heads = q->size(1);
  double scale = 1.0 / std::sqrt((double)p.d);
  if (o[12] != Py_None && !real(o[12], scale)) Py_RETURN_NONE;
  const uint64_t* tree = nullptr;
  if (o[13] != Py_None) {
    const at::Tensor* t = tensor(o[13]);
    if (!t || max_q > 64 || t->dim() != 1 || t->size(0) != total ||
        !fits(*t, p.device, t->scalar_type() == at::kUInt64 ? at::kUInt64 : at::kLong))
      Py_RETURN_NONE;
    tree = static_cast<const uint64_t*>(t->data_ptr());
  }
  const int32_t ng = (int32_t)cg->size(0) - 1;
  if (tile == 0) {
    tile = g_shared_rows(p.batch, ng, (int32_t)total, (int32_t)heads, p.kv, p.d, (int32_t)max_q, (int32_t)max_len, (int32_t)max_prefix);
    if (tile == 0) {  // every sequence by itself
      if (max_prefix > (int64_t)p.max_blocks * 16) Py_RETURN_NONE;
      PyObject* const plain[12] = {o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[7], o[8], o[12], o[13], n == 16 ? o[15] : Py_None};
      return attention(nullptr, plain, 12);
    }
  }
  const size_t bytes = g_shared_size(p.batch, ng, (int32_t)total, (int32_t)heads, p.kv, p.d, (int32_t)max_q, (int32_t)max_len, (int32_t)max_prefix,
                                     (int32_t)tile);
  if (bytes == 0) Py_RETURN_NONE;  // sizes that the general path refuses
  const at::Tensor* given = nullptr;
  if (n == 16 && o[15] != Py_None) {
    given = rows(o[15], p, heads, out_row);
    if (!given || given->size(0) != total) Py_RETURN_NONE;
  }
  Launch on(p);
  at::Tensor out;
  if (!given) {
    out = at::empty({total, heads, p.d}, q->options());
    out_row = heads * p.d;
  }
  const c10::DataPtr ws = c10::hip::HIPCachingAllocator::get()->allocate(bytes);
  const int st = g_shared(q->data_ptr(), q_row, p.k, p.v, p.s, p.blocks, p.format, p.table, p.max_blocks, cu, lens, tree, groups, prefix,
                          p.batch, ng, (int32_t)total, (int32_t)heads, p.kv, p.d, (int32_t)max_q, (int32_t)max_len, (int32_t)max_prefix,
                          (int32_t)tile, (float)scale, ws.get(), bytes, given ? given->data_ptr() : out.data_ptr(), out_row, on.stream);
  if (st != SDV_OK) return status(st);
  if (given) {
    Py_INCREF(o[15]);
    return o[15];
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

bool addresses(PyObject* const* o, Py_ssize_t n, void** at) {
  for (Py_ssize_t i = 0; i < n; ++i) {
    at[i] = PyLong_AsVoidPtr(o[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a null address");
      return false;
    }
  }
  return true;
}

// bind_moves(rope, rope_append, copy_blocks, keep): the same for the operators that move and turn rows
PyObject* bind_moves(PyObject*, PyObject* const* o, Py_ssize_t n) {
  void* at[4];
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "bind_moves needs four addresses");
    return nullptr;
  }
  if (!addresses(o, n, at)) return nullptr;
  g_rope = reinterpret_cast<decltype(g_rope)>(at[0]);
  g_rope_append = reinterpret_cast<decltype(g_rope_append)>(at[1]);
  g_copy = reinterpret_cast<decltype(g_copy)>(at[2]);
  g_keep = reinterpret_cast<decltype(g_keep)>(at[3]);
  Py_RETURN_NONE;
}

// bind_shared(shared_attention, its workspace_size, its tile_rows)
PyObject* bind_shared(PyObject*, PyObject* const* o, Py_ssize_t n) {
  void* at[3];
  if (n != 3) {
    PyErr_SetString(PyExc_TypeError, "bind_shared needs three addresses");
    return nullptr;
  }
  if (!addresses(o, n, at)) return nullptr;
  g_shared = reinterpret_cast<decltype(g_shared)>(at[0]);
  g_shared_size = reinterpret_cast<decltype(g_shared_size)>(at[1]);
  g_shared_rows = reinterpret_cast<decltype(g_shared_rows)>(at[2]);
  Py_RETURN_NONE;
}

// bind(append, gather, attention, workspace_size): the addresses of the loaded library's entry points
PyObject* bind(PyObject*, PyObject* const* o, Py_ssize_t n) {
  void* at[4];
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "bind needs four addresses");
    return nullptr;
  }
  if (!addresses(o, n, at)) return nullptr;
  g_append = reinterpret_cast<decltype(g_append)>(at[0]);
  g_gather = reinterpret_cast<decltype(g_gather)>(at[1]);
  g_attention = reinterpret_cast<decltype(g_attention)>(at[2]);
  g_workspace_size = reinterpret_cast<decltype(g_workspace_size)>(at[3]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(append)), METH_FASTCALL, nullptr},
    {"gather", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(gather)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attention)), METH_FASTCALL, nullptr},
    {"rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(rope)), METH_FASTCALL, nullptr},
    {"rope_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(rope_append)), METH_FASTCALL, nullptr},
    {"copy_blocks", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(copy_blocks)), METH_FASTCALL, nullptr},
    {"keep", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(keep)), METH_FASTCALL, nullptr},
    {"bind_moves", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind_moves)), METH_FASTCALL, nullptr},
    {"shared", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(shared)), METH_FASTCALL, nullptr},
    {"bind_shared", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind_shared)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv8_binding", nullptr, -1, methods};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__kv8_binding() { return PyModule_Create(&module); }
