// The episode cache's entry points for torch tensors, called by episode_cache.py: the checks of a call, its
// output tensors, stream and workspace, and the call of the C ABI, in one step. A call on a few rows is over
// on the GPU in 4 to 9 us, and as Python statements over ctypes these things took 17 to 24 us.
//
// A function returns None for arguments that it does not accept: episode_cache.py, whose checks know what is
// wrong, then raises. A status other than 0 of the C ABI is returned as an int.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cmath>
#include <cstring>
#include <map>
#include <mutex>
#include <utility>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "mkx_cache.h"

namespace {

using at::Tensor;

// The C ABI, bound by address (bind): this file links to torch only, whichever build of the library is in use.
mkx_status (*plan_fn)(const mkx_plan_inputs*, int, cudaStream_t);
mkx_status (*store_fn)(const mkx_store_inputs*, int, cudaStream_t);
mkx_status (*attend_fn)(const mkx_attend_inputs*, size_t, int, cudaStream_t);
size_t (*workspace_fn)(const mkx_attend_inputs*, int);

constexpr long long MAX_ROWS = 1 << 30;  // of an episode

bool tensor(PyObject* o, Tensor& t) {
  if (!THPVariable_Check(o)) return false;
  t = THPVariable_Unpack(o);
  return true;
}
bool vector(const Tensor& t, int64_t n, at::ScalarType type, at::Device dev) {
  return t.scalar_type() == type && t.dim() == 1 && t.size(0) == n && t.device() == dev && t.is_contiguous();
}
// Whether autograd would expect this call in its graph: it records nothing.
bool recorded(const Tensor& t) { return t.defined() && t.requires_grad() && at::GradMode::is_enabled(); }
// A tensor that a call has written in place: what autograd saved of it before is out of date. (Inference tensors are
// not versioned.)
void written(const Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
bool page_size(int64_t n) { return n == 16 || n == 32 || n == 64 || n == 128 || n == 256; }
bool half_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
bool table_fits(const Tensor& t, int64_t b, int64_t page_rows, at::Device dev) {
  return t.dim() == 2 && t.size(0) == b && t.size(1) >= 1 && t.scalar_type() == at::kInt && t.device() == dev &&
         t.is_contiguous() && t.size(1) * page_rows <= MAX_ROWS;
}
// Strides of the leading dims; dims contiguous, everything else on 16-byte boundaries. A dim of size one has
// no stride of its own. Where rows lie apart no stride is zero: what is written to
// (several rows would share a place), and pages that a tensor map describes.
enum Use { SHARED, APART };
template <int N>
bool strides(const Tensor& t, long long (&out)[N], Use use) {
  if (t.size(N) > 1 && t.stride(N) != 1) return false;
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) return false;
  for (int i = 0; i < N; ++i) {
    out[i] = t.size(i) > 1 ? t.stride(i) : t.size(N);
    if (out[i] & 7 || (use == APART && out[i] == 0)) return false;
  }
  return true;
}
bool integer(PyObject* o, long long& v) {
  v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
PyObject* none() { Py_RETURN_NONE; }
cudaStream_t stream_of(at::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }
at::TensorOptions on(at::Device dev, at::ScalarType type) { return at::TensorOptions().device(dev).dtype(type); }

// A vector of n values at word `at` of a block of 32-bit words (`at` even for 64-bit values).
Tensor view(const Tensor& block, int64_t at, int64_t n, at::ScalarType type) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(block.storage()), block.key_set(),
                                                      c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_storage_offset(type == at::kLong ? at / 2 : at);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

// ---- placing: (length, new, table, free, marks, page_rows, rows, ticket) -> (start, slot, episode, position, length, marks)
PyObject* plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor length, fresh, table, ring, marks, ticket;
  long long page_rows, rows;
  if (n != 8 || !tensor(a[0], length) || !tensor(a[1], fresh) || !tensor(a[2], table) || !tensor(a[3], ring) ||
      !tensor(a[4], marks) || !integer(a[5], page_rows) || !integer(a[6], rows))
    return none();
  const bool in_place = a[7] != Py_None;
  const at::Device dev = length.device();
  const int64_t b = length.numel();
  if (!dev.is_cuda() || b < 1 || b > MKX_MAX_EPISODES || !page_size(page_rows) || rows < 0 || rows >= 1ll << 31 ||
      !vector(length, b, at::kInt, dev) || !vector(fresh, b, at::kInt, dev) || ring.numel() < 1 ||
      ring.numel() >= 1ll << 31 || !vector(ring, ring.numel(), at::kInt, dev) || !vector(marks, 3, at::kLong, dev) ||
      !table_fits(table, b, page_rows, dev))
    return none();
  if (in_place && (!tensor(a[7], ticket) || !vector(ticket, 1, at::kInt, dev))) return none();
  // one allocation: slot, episode, position, marks, each on a 16-byte boundary, then length and start
  const int64_t padded = (rows + 3) / 4 * 4;
  const Tensor block = at::empty({4 * padded + 8 + 2 * b + 1}, on(dev, at::kInt));
  Tensor slot = view(block, 0, rows, at::kLong), episode = view(block, 2 * padded, rows, at::kInt),
         position = view(block, 3 * padded, rows, at::kInt),
         marks_after = in_place ? marks : view(block, 4 * padded, 3, at::kLong),
         after = in_place ? length : view(block, 4 * padded + 8, b, at::kInt),
         start = view(block, 4 * padded + 8 + b, b + 1, at::kInt);
  mkx_plan_inputs p;
  std::memset(&p, 0, sizeof(p));
  p.length = static_cast<const int*>(length.data_ptr());
  p.new_rows = static_cast<const int*>(fresh.data_ptr());
  p.table = static_cast<int*>(table.data_ptr());
  p.ring = static_cast<const int*>(ring.data_ptr());
  p.marks = static_cast<const long long*>(marks.data_ptr());
  p.start = static_cast<int*>(start.data_ptr());
  p.slot = static_cast<long long*>(slot.data_ptr());
  p.episode = static_cast<int*>(episode.data_ptr());
  p.position = static_cast<int*>(position.data_ptr());
  p.length_out = static_cast<int*>(after.data_ptr());
  p.marks_out = static_cast<long long*>(marks_after.data_ptr());
  p.ticket = in_place ? static_cast<int*>(ticket.data_ptr()) : nullptr;
  p.B = (int)b;
  p.table_width = (int)table.size(1);
  p.ring_pages = (int)ring.numel();
  p.page_rows = (int)page_rows;
  p.rows = (int)rows;
  const mkx_status st = plan_fn(&p, dev.index(), stream_of(dev));
  if (st) return PyLong_FromLong(st);
  written(table);
  if (in_place)
    for (const Tensor* t : {&length, &marks, &ticket}) written(*t);
  PyObject* out = PyTuple_New(6);
  if (!out) return nullptr;
  const Tensor* all[6] = {&start, &slot, &episode, &position, &after, &marks_after};
  for (int i = 0; i < 6; ++i) PyTuple_SET_ITEM(out, i, THPVariable_Wrap(*all[i]));
  return out;
  END_HANDLE_TH_ERRORS
}

// ---- storing: (k, v, slot, k_pages, v_pages, q, positions, rotary bytes, out) -> out, or True without q
PyObject* store(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor k, v, slot, kp, vp, q, pos, out;
  if (n != 9 || !tensor(a[0], k) || !tensor(a[1], v) || !tensor(a[2], slot) || !tensor(a[3], kp) || !tensor(a[4], vp))
    return none();
  const at::Device dev = k.device();
  const auto type = k.scalar_type();
  if (!dev.is_cuda() || k.dim() != 3 || v.sizes() != k.sizes() || !half_type(type) || kp.dim() != 4 ||
      vp.sizes() != kp.sizes())
    return none();
  const int64_t rows = k.size(0), heads = k.size(1), hd = k.size(2);
  if (heads < 1 || hd < 16 || hd > 256 || hd % 16 || rows >= 1ll << 31 || kp.size(0) < 1 || kp.size(0) >= 1ll << 31 ||
      !page_size(kp.size(1)) || kp.size(2) != heads || kp.size(3) != hd || v.scalar_type() != type ||
      v.device() != dev || kp.scalar_type() != type || kp.device() != dev || vp.scalar_type() != type ||
      vp.device() != dev || !vector(slot, rows, at::kLong, dev))
    return none();
  mkx_store_inputs p;
  std::memset(&p, 0, sizeof(p));
  if (a[6] != Py_None) {
    char* bytes;
    Py_ssize_t size;
    if (!tensor(a[6], pos) || PyBytes_AsStringAndSize(a[7], &bytes, &size) || size != sizeof(mkx_rotary)) {
      PyErr_Clear();
      return none();
    }
    std::memcpy(&p.rot, bytes, sizeof(mkx_rotary));
    const bool flat = pos.dim() == 1;
    if (pos.scalar_type() != at::kInt || pos.device() != dev || (!flat && pos.dim() != 2) ||
        (flat ? 1 : pos.size(0)) != p.rot.axes || pos.size(flat ? 0 : 1) != rows ||
        (rows > 1 && pos.stride(flat ? 0 : 1) != 1))
      return none();
    p.positions = static_cast<const int*>(pos.data_ptr());
    p.pos_stride = flat ? 0 : pos.stride(0);
  }
  long long s2[2], s3[3];
  if (a[5] != Py_None) {
    if (a[6] == Py_None || !tensor(a[5], q) || q.dim() != 3 || q.size(0) != rows || q.size(1) < 1 || q.size(2) != hd ||
        q.scalar_type() != type || q.device() != dev)
      return none();
    if (a[8] == Py_None) {
      out = at::empty_like(q);
    } else if (!tensor(a[8], out) || out.sizes() != q.sizes() || out.scalar_type() != type || out.device() != dev) {
      return none();
    }
    if (!strides(q, s2, SHARED)) return none();
    p.q = q.data_ptr();
    p.q_row = s2[0];
    p.q_head = s2[1];
    if (!strides(out, s2, APART)) return none();
    p.q_out = out.data_ptr();
    p.qo_row = s2[0];
    p.qo_head = s2[1];
    p.heads = (int)q.size(1);
  } else if (a[8] != Py_None) {
    return none();
  }
  for (const Tensor* t : {&k, &v, &kp, &vp, &q, &out})
    if (recorded(*t)) return none();
  if (!strides(k, s2, SHARED)) return none();
  p.k_row = s2[0];
  p.k_head = s2[1];
  if (!strides(v, s2, SHARED)) return none();
  p.v_row = s2[0];
  p.v_head = s2[1];
  if (!strides(kp, s3, APART)) return none();
  p.kp_page = s3[0];
  p.kp_row = s3[1];
  p.kp_head = s3[2];
  if (!strides(vp, s3, APART)) return none();
  p.vp_page = s3[0];
  p.vp_row = s3[1];
  p.vp_head = s3[2];
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.k_pages = kp.data_ptr();
  p.v_pages = vp.data_ptr();
  p.slot = static_cast<const long long*>(slot.data_ptr());
  p.rows = (int)rows;
  p.kv_heads = (int)heads;
  p.head_dim = (int)hd;
  p.dtype = type == at::kBFloat16 ? MKX_BF16 : MKX_FP16;
  p.pages = (int)kp.size(0);
  p.page_rows = (int)kp.size(1);
  const mkx_status st = store_fn(&p, dev.index(), stream_of(dev));
  if (st) return PyLong_FromLong(st);
  for (const Tensor* t : {&kp, &vp, &out}) written(*t);
  if (!out.defined()) Py_RETURN_TRUE;
  if (a[8] != Py_None) return Py_NewRef(a[8]);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// ---- attention ----------------------------------------------------------------------------------
// (never destroyed: the process may end after the CUDA context)
std::mutex& lock = *new std::mutex;
std::map<int, Tensor>& errors = *new std::map<int, Tensor>;  // device -> error word, only ever set by a call
// workspaces of eager calls, which their stream keeps in order
std::map<std::pair<int, cudaStream_t>, Tensor>& spaces = *new std::map<std::pair<int, cudaStream_t>, Tensor>;

// Workspace of a call: its first words are zero between calls. Eager calls of one stream share one; a captured call
// gets its own out of the graph's pool, zeroed by the graph, so that two graphs may be replayed at once.
Tensor space_for(at::Device dev, cudaStream_t stream, size_t size, bool capturing) {
  auto fresh = [&]() {
    Tensor t = at::empty({(int64_t)size}, on(dev, at::kByte));
    t.narrow(0, 0, MKX_ATTEND_TICKETS * 4).zero_();
    return t;
  };
  if (capturing) return fresh();
  std::lock_guard<std::mutex> hold(lock);
  Tensor& t = spaces[{(int)dev.index(), stream}];
  if (!t.defined() || (size_t)t.numel() < size) t = fresh();
  return t;
}
// The error word of a device; null while a graph is being captured before the first call.
int* error_word(at::Device dev, bool capturing) {
  std::lock_guard<std::mutex> hold(lock);
  Tensor& t = errors[dev.index()];
  if (!t.defined()) {
    if (capturing) return nullptr;
    t = at::zeros({1}, on(dev, at::kInt));
    c10::cuda::stream_synchronize(c10::cuda::getCurrentCUDAStream(dev.index()));  // zero before any stream uses it
  }
  return static_cast<int*>(t.data_ptr());
}

// (q, k_pages, v_pages, table, length, start, max_rows (-1: q's rows), causal, window, sinks, scale, out) -> out; False: a
// capture before the first call
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, kp, vp, table, length, start, out;
  long long max_rows, window, sinks;
  if (n != 12 || !tensor(a[0], q) || !tensor(a[1], kp) || !tensor(a[2], vp) || !tensor(a[3], table) ||
      !tensor(a[4], length) || !tensor(a[5], start) || !integer(a[6], max_rows) || !integer(a[8], window) ||
      !integer(a[9], sinks))
    return none();
  const int causal = PyObject_IsTrue(a[7]);
  if (causal < 0) {  // it has no truth value
    PyErr_Clear();
    return none();
  }
  double scale = 0;
  if (a[10] != Py_None) {
    scale = PyFloat_AsDouble(a[10]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return none();
    }
  }
  const at::Device dev = q.device();
  const auto type = q.scalar_type();
  if (!dev.is_cuda() || q.dim() != 3 || !half_type(type) || kp.dim() != 4 || vp.sizes() != kp.sizes()) return none();
  const int64_t rows = q.size(0), heads = q.size(1), hd = q.size(2), b = length.numel();
  if ((hd != 64 && hd != 128) || rows >= 1ll << 31 || kp.size(3) != hd || kp.size(0) < 1 || kp.size(0) >= 1ll << 31 ||
      !page_size(kp.size(1)) || kp.size(2) < 1 || heads < 1 || heads % kp.size(2) || kp.scalar_type() != type ||
      kp.device() != dev || vp.scalar_type() != type || vp.device() != dev || b < 1 || b > MKX_MAX_EPISODES ||
      !vector(length, b, at::kInt, dev) || !vector(start, b + 1, at::kInt, dev) ||
      !table_fits(table, b, kp.size(1), dev) || max_rows < -1 || window < 0 || sinks < 0 ||
      (window > 0 && !causal) || (sinks > 0 && window == 0) || !std::isfinite(scale))
    return none();
  if (a[11] == Py_None) {
    out = at::empty_like(q);
  } else if (!tensor(a[11], out) || out.sizes() != q.sizes() || out.scalar_type() != type || out.device() != dev) {
    return none();
  }
  for (const Tensor* t : {&q, &kp, &vp, &out})
    if (recorded(*t)) return none();
  mkx_attend_inputs p;
  std::memset(&p, 0, sizeof(p));
  long long s2[2], s3[3];
  if (!strides(q, s2, SHARED)) return none();
  p.q_row = s2[0];
  p.q_head = s2[1];
  if (!strides(out, s2, APART)) return none();
  p.o_row = s2[0];
  p.o_head = s2[1];
  if (!strides(kp, s3, APART)) return none();
  p.kp_page = s3[0];
  p.kp_row = s3[1];
  p.kp_head = s3[2];
  if (!strides(vp, s3, APART)) return none();
  p.vp_page = s3[0];
  p.vp_row = s3[1];
  p.vp_head = s3[2];
  p.q = q.data_ptr();
  p.k_pages = kp.data_ptr();
  p.v_pages = vp.data_ptr();
  p.out = out.data_ptr();
  p.table = static_cast<const int*>(table.data_ptr());
  p.length = static_cast<const int*>(length.data_ptr());
  p.start = static_cast<const int*>(start.data_ptr());
  p.rows = (int)rows;
  p.B = (int)b;
  p.heads = (int)heads;
  p.kv_heads = (int)kp.size(2);
  p.head_dim = (int)hd;
  p.dtype = type == at::kBFloat16 ? MKX_BF16 : MKX_FP16;
  p.pages = (int)kp.size(0);
  p.page_rows = (int)kp.size(1);
  p.table_width = (int)table.size(1);
  p.max_rows = (int)(max_rows < 0 || max_rows > rows ? rows : max_rows);
  p.causal = causal;
  p.window = (int)(window < MAX_ROWS ? window : MAX_ROWS);
  p.sinks = (int)(sinks < MAX_ROWS ? sinks : MAX_ROWS);
  p.scale = (float)(a[10] == Py_None ? 1.0 / std::sqrt((double)hd) : scale);
  if (rows > 0) {
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != dev.index()) guard.set_device(dev);
    const cudaStream_t stream = stream_of(dev);
    const bool capturing = c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
    const size_t size = workspace_fn(&p, dev.index());
    if (size == 0) return none();
    p.error = error_word(dev, capturing);
    if (!p.error) Py_RETURN_FALSE;
    const Tensor space = space_for(dev, stream, size, capturing);
    p.workspace = space.data_ptr();
    const mkx_status st = attend_fn(&p, (size_t)space.numel(), dev.index(), stream);
    if (st) return PyLong_FromLong(st);
    written(out);
  }
  if (a[11] != Py_None) return Py_NewRef(a[11]);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// (device index) -> the error word's value, which is zeroed; synchronises. make: allocates it if there is none.
PyObject* error_code(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  long long index;
  if (n != 2 || !integer(a[0], index)) return none();
  const at::Device dev(at::kCUDA, (c10::DeviceIndex)index);
  if (PyObject_IsTrue(a[1]) == 1) {
    c10::cuda::CUDAGuard guard(dev);
    error_word(dev, false);
    Py_RETURN_NONE;
  }
  Tensor t;
  {
    std::lock_guard<std::mutex> hold(lock);
    auto it = errors.find((int)index);
    if (it == errors.end() || !it->second.defined()) return PyLong_FromLong(0);
    t = it->second;
  }
  c10::cuda::CUDAGuard guard(dev);
  c10::cuda::device_synchronize();  // the calls of all streams
  const int code = t.item<int>();
  if (code) {  // the calls that gave up may have left tickets behind
    t.zero_();
    std::lock_guard<std::mutex> hold(lock);
    for (auto& s : spaces)
      if (s.first.first == (int)index) s.second.narrow(0, 0, MKX_ATTEND_TICKETS * 4).zero_();
    c10::cuda::device_synchronize();
  }
  return PyLong_FromLong(code);
  END_HANDLE_TH_ERRORS
}

// (mkx_cache_key of the library, addresses of mkx_cache_plan, mkx_cache_store, mkx_cache_attend, mkx_attend_workspace); None,
// and nothing is bound, if the library was built from another mkx_cache.h
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  long long v[5];
  if (n != 5) return none();
  for (int i = 0; i < 5; ++i)
    if (!integer(a[i], v[i])) return none();
  if ((unsigned long long)v[0] != MKX_CACHE_KEY) return none();
  plan_fn = reinterpret_cast<decltype(plan_fn)>(v[1]);
  store_fn = reinterpret_cast<decltype(store_fn)>(v[2]);
  attend_fn = reinterpret_cast<decltype(attend_fn)>(v[3]);
  workspace_fn = reinterpret_cast<decltype(workspace_fn)>(v[4]);
  Py_RETURN_TRUE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(plan), METHOD(store), METHOD(attend), METHOD(error_code), METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mkx_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mkx_torch(void) { return PyModule_Create(&module); }
