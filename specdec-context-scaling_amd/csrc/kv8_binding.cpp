// The kv8 operators' way from torch tensors to libsdv: a Python extension module whose functions take
// the plain case of an operator's arguments -- tensors as the library takes them -- straight to the C
// ABI.  Anything else returns None, and the caller's general path copies what may be copied and says
// what is wrong with the rest.
//
// An engine calls these operators once per layer and token, so their host time is part of every token:
// the checks of ten tensors' types, shapes, strides and devices, the stream, the workspace and a call
// with 25 arguments through ctypes took 7 to 10 us, of which this leaves about 1 beside the launch.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
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
const at::Tensor* rows(PyObject* o, const Pages& p, int64_t heads, int64_t& stride) {
  const at::Tensor* t = tensor(o);
  if (!t || t->dim() != 3 || t->scalar_type() != at::kBFloat16 || t->device() != p.device) return nullptr;
  const int64_t n = t->size(0), h = t->size(1);
  if (t->size(2) != p.d || (heads && h != heads) || n == 0 || n > INT32_MAX || h > INT32_MAX) return nullptr;
  stride = n == 1 ? h * p.d : t->stride(0);
  if (t->stride(2) != 1 || (t->stride(1) != p.d && h != 1) || stride < h * p.d || stride % 8 != 0 ||
      reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 != 0)
    return nullptr;
  return t;
}

bool ints(PyObject* o, const Pages& p, int64_t n, const int32_t*& at) {
  const at::Tensor* t = tensor(o);
  if (!t || t->dim() != 1 || t->size(0) != n || !fits(*t, p.device, at::kInt)) return false;
  at = static_cast<const int32_t*>(t->data_ptr());
  return true;
}

bool lengths(PyObject* o, const Pages& p, const int32_t*& at) {
  at = nullptr;
  return o == Py_None || ints(o, p, p.batch, at);
}

// The current device, made the tensors' for the call, and its stream.
struct Launch {
  c10::OptionalDeviceGuard guard;
  hipStream_t stream;
  explicit Launch(const Pages& p) : guard(p.device), stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(p.device.index()).stream()) {}
};

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

// bind(append, gather, attention, workspace_size): the addresses of the loaded library's entry points
PyObject* bind(PyObject*, PyObject* const* o, Py_ssize_t n) {
  void* at[4];
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "bind needs four addresses");
    return nullptr;
  }
  for (int i = 0; i < 4; ++i) {
    at[i] = PyLong_AsVoidPtr(o[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a null address");
      return nullptr;
    }
  }
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
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv8_binding", nullptr, -1, methods};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__kv8_binding() { return PyModule_Create(&module); }
