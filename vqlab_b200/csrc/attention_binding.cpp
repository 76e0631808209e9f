// vqlab_b200._native: the Python side of the attention calls (attention.py).
//
// A step's calls on small batches take a few microseconds on the device; checking
// their arguments and building their descriptors in Python took 10 to 15, so that
// part is here.  Each function checks its tensors, allocates its outputs, calls
// the C ABI on the current stream and returns the outputs, or the vqb_status as
// an int, which the Python wrapper turns into the package's exceptions.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include "../../include/vqb.h"

namespace {

using at::Tensor;

// The C ABI's entry points, from the library that the package has loaded.
struct {
  decltype(&::vqb_paged_tables) paged_tables;
  decltype(&::vqb_rotary_append) rotary_append;
  decltype(&::vqb_prefix_attention_workspace_size) workspace_size;
  decltype(&::vqb_prefix_attention) prefix_attention;
} g_abi;

[[noreturn]] void refuse(const std::string& what) { throw c10::ValueError(what, nullptr); }

std::string shape_text(at::IntArrayRef s) {
  std::string t = "[";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + "]";
}

const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

// A contiguous tensor of whole numbers on `dev`; shape: {} = any.
const Tensor& ints(PyObject* o, const char* name, const at::Device& dev, at::ScalarType dt = at::kInt) {
  const Tensor& t = tensor(o, name);
  if (t.scalar_type() != dt || t.device() != dev || !t.is_contiguous())
    refuse(std::string(name) + " must be a contiguous " + at::toString(dt) + " tensor on " + dev.str());
  return t;
}
const Tensor& ints(PyObject* o, const char* name, const at::Device& dev, at::IntArrayRef shape,
                   at::ScalarType dt = at::kInt) {
  const Tensor& t = ints(o, name, dev, dt);
  if (t.sizes() != shape) refuse(std::string(name) + " must have the shape " + shape_text(shape));
  return t;
}

bool is_half(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
vqb_dtype code(at::ScalarType t) { return t == at::kHalf ? VQB_F16 : VQB_BF16; }

// q [N, heads, D] of a call
const Tensor& query(PyObject* o, const char* name) {
  const Tensor& t = tensor(o, name);
  if (!t.is_cuda() || t.dim() != 3 || !is_half(t.scalar_type()) || t.stride(2) != 1)
    refuse(std::string(name) + " must be a CUDA tensor [N, heads, D] with contiguous heads, fp16 or bf16");
  return t;
}
const Tensor& heads(PyObject* o, const char* name, const Tensor& like, at::IntArrayRef shape) {
  const Tensor& t = tensor(o, name);
  if (t.scalar_type() != like.scalar_type() || t.device() != like.device() || t.sizes() != shape || t.stride(-1) != 1)
    refuse(std::string(name) + " must be a " + at::toString(like.scalar_type()) + " tensor on " + like.device().str() +
           " of shape " + shape_text(shape) + " with contiguous heads");
  return t;
}
// k_cache of a call: [pages, kv_heads, page_size, D]
const Tensor& pool(PyObject* o, const Tensor& q) {
  const Tensor& t = tensor(o, "k_cache");
  if (t.dim() != 4) refuse("k_cache must be [pages, kv_heads, page_size, D]");
  return heads(o, "k_cache", q, {t.size(0), t.size(1), t.size(2), q.size(2)});
}

int32_t int32(int64_t v, const char* name) {
  if (v < INT32_MIN || v > INT32_MAX) refuse(std::string(name) + " does not fit 32 bits");
  return static_cast<int32_t>(v);
}
int32_t int32(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return int32(v, name);
}
float real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return static_cast<float>(v);
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
void count(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) throw torch::TypeError("wrong number of arguments");
}

Tensor empty(at::IntArrayRef sizes, at::ScalarType dt, const at::Device& dev) {
  return at::detail::empty_cuda(sizes, dt, dev, std::nullopt);
}
// A tensor in `flat`'s memory from byte `at` on (one allocation for a call's outputs).
Tensor part(const Tensor& flat, int64_t at_byte, at::IntArrayRef sizes, at::ScalarType dt) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(flat.storage()), flat.key_set(), c10::scalarTypeToTypeMeta(dt));
  impl->set_sizes_contiguous(sizes);
  impl->set_storage_offset(at_byte / static_cast<int64_t>(c10::elementSize(dt)));
  return Tensor(std::move(impl));
}

vqb_stream_t stream(const at::Device& dev) {
  return reinterpret_cast<vqb_stream_t>(at::cuda::getCurrentCUDAStream(dev.index()).stream());
}

template <typename T>
T* ptr(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }

PyObject* status(vqb_status st) { return PyLong_FromLong(st); }

// context_lens, new_lens, block_table, free_pages, state, page_size, max_tokens, position_offset, inplace
PyObject* paged_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 9);
  const Tensor& table = tensor(a[2], "block_table");
  if (!table.is_cuda() || table.dim() != 2) refuse("block_table must be a CUDA tensor [R, W]");
  const at::Device dev = table.device();
  ints(a[2], "block_table", dev);
  const int64_t R = table.size(0), W = table.size(1);
  const Tensor& context = ints(a[0], "context_lens", dev, {R});
  const Tensor& fresh = ints(a[1], "new_lens", dev, {R});
  const Tensor& ring = ints(a[3], "free_pages", dev);
  if (ring.dim() != 1) refuse("free_pages must be a ring [F]");
  const Tensor& state = ints(a[4], "state", dev, {4}, at::kLong);
  const int64_t F = ring.size(0);
  vqb_paged_desc d{int32(R, "R"), int32(W, "W"), int32(a[5], "page_size"), int32(F, "F"), int32(a[6], "max_tokens"),
                   int32(a[7], "position_offset")};
  if (d.max_tokens < 0) refuse("max_tokens must not be negative");
  const bool inplace = truth(a[8]);
  const int64_t T = d.max_tokens;
  const c10::cuda::CUDAGuard guard(dev);
  int64_t bytes = 0;
  auto take = [&](int64_t size) {
    const int64_t at = bytes;
    bytes += (size + 15) & ~int64_t(15);
    return at;
  };
  const int64_t at_cu = take(4 * (R + 1)), at_slots = take(4 * T), at_pos = take(4 * T), at_req = take(4 * T);
  const int64_t at_table = inplace ? 0 : take(4 * R * W), at_ring = inplace ? 0 : take(4 * F);
  const int64_t at_state = inplace ? 0 : take(32), at_lens = inplace ? 0 : take(4 * R);
  const Tensor flat = empty({bytes}, at::kByte, dev);
  const Tensor cu = part(flat, at_cu, {R + 1}, at::kInt), slots = part(flat, at_slots, {T}, at::kInt);
  const Tensor pos = part(flat, at_pos, {T}, at::kInt), req = part(flat, at_req, {T}, at::kInt);
  const Tensor table_out = inplace ? table : part(flat, at_table, {R, W}, at::kInt);
  const Tensor ring_out = inplace ? ring : part(flat, at_ring, {F}, at::kInt);
  const Tensor state_out = inplace ? state : part(flat, at_state, {4}, at::kLong);
  const Tensor lens = inplace ? context : part(flat, at_lens, {R}, at::kInt);
  const vqb_status st = g_abi.paged_tables(
      &d, ptr<int32_t>(context), ptr<int32_t>(fresh), ptr<int32_t>(table), ptr<int32_t>(ring), ptr<int64_t>(state),
      ptr<int32_t>(table_out), ptr<int32_t>(ring_out), ptr<int64_t>(state_out), ptr<int32_t>(lens), ptr<int32_t>(cu),
      ptr<int32_t>(slots), ptr<int32_t>(pos), ptr<int32_t>(req), stream(dev));
  if (st != VQB_OK) return status(st);
  const Tensor* outs[8] = {&table_out, &lens, &cu, &slots, &pos, &req, &ring_out, &state_out};
  THPObjectPtr r(PyTuple_New(8));
  if (!r) throw python_error();
  for (int i = 0; i < 8; ++i) PyTuple_SET_ITEM(r.get(), i, THPVariable_Wrap(*outs[i]));
  return r.release();
  END_HANDLE_TH_ERRORS
}

// q, k, v, positions, freq, k_cache, v_cache, slots, interleaved, amplitude, out; k None: q alone
PyObject* rotary_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 11);
  const Tensor& q = query(a[0], "q");
  const at::Device dev = q.device();
  const int64_t N = q.size(0), H = q.size(1), D = q.size(2);
  const Tensor& positions = ints(a[3], "positions", dev);
  const Tensor& freq = ints(a[4], "freq", dev, at::kLong);
  if (positions.numel() < N) refuse("positions must cover the tokens");
  if (2 * freq.numel() > D) refuse("freq holds more pairs than a head has");
  vqb_rotary_desc d{};
  const void *kp = nullptr, *vp = nullptr;
  const int32_t* slots_p = nullptr;
  void *kcp = nullptr, *vcp = nullptr;
  if (a[1] != Py_None) {
    const Tensor& kc = pool(a[5], q);
    const Tensor& vc = heads(a[6], "v_cache", q, kc.sizes());
    const Tensor& k = heads(a[1], "k", q, {N, kc.size(1), D});
    const Tensor& v = heads(a[2], "v", q, {N, kc.size(1), D});
    const Tensor& slots = ints(a[7], "slots", dev);
    if (slots.numel() < N) refuse("slots must cover the tokens");
    d.kv_heads = int32(kc.size(1), "kv_heads");
    d.page_size = int32(kc.size(2), "page_size");
    d.num_pages = int32(kc.size(0), "pages");
    d.k_token_stride = k.stride(0);
    d.k_head_stride = k.stride(1);
    d.v_token_stride = v.stride(0);
    d.v_head_stride = v.stride(1);
    d.kc_page_stride = kc.stride(0);
    d.kc_head_stride = kc.stride(1);
    d.kc_token_stride = kc.stride(2);
    d.vc_page_stride = vc.stride(0);
    d.vc_head_stride = vc.stride(1);
    d.vc_token_stride = vc.stride(2);
    kp = k.data_ptr();
    vp = v.data_ptr();
    kcp = kc.data_ptr();
    vcp = vc.data_ptr();
    slots_p = ptr<int32_t>(slots);
  }
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor out = a[10] == Py_None ? empty(q.sizes(), q.scalar_type(), dev) : heads(a[10], "out", q, q.sizes());
  d.n_tokens = int32(N, "N");
  d.heads = int32(H, "heads");
  d.head_dim = int32(D, "D");
  d.rotary_dim = int32(2 * freq.numel(), "freq");
  d.interleaved = truth(a[8]);
  d.amplitude = real(a[9]);
  d.q_token_stride = q.stride(0);
  d.q_head_stride = q.stride(1);
  d.out_token_stride = out.stride(0);
  d.out_head_stride = out.stride(1);
  const vqb_status st = g_abi.rotary_append(&d, code(q.scalar_type()), q.data_ptr(), kp, vp, ptr<int32_t>(positions),
                                            ptr<int64_t>(freq), slots_p, out.data_ptr(), kcp, vcp, stream(dev));
  if (st != VQB_OK) return status(st);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// q, k_cache, v_cache, block_table, kv_lens, cu_q, max_q_len, max_kv_len, prefix_pages, prefix_len, scale, causal, out,
// return_lse, workspace
PyObject* prefix_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 15);
  const Tensor& q = query(a[0], "q");
  const at::Device dev = q.device();
  const int64_t N = q.size(0), H = q.size(1), D = q.size(2);
  const Tensor& kc = pool(a[1], q);
  const Tensor& vc = heads(a[2], "v_cache", q, kc.sizes());
  if (kc.size(1) < 1 || H % kc.size(1)) refuse("heads must be a multiple of kv_heads");
  const Tensor& lens = ints(a[4], "kv_lens", dev);
  const int64_t R = lens.numel();
  const Tensor& cu = ints(a[5], "cu_q", dev, {R + 1});
  const Tensor& table = ints(a[3], "block_table", dev);
  if (table.dim() != 2 || table.size(0) != R) refuse("block_table must be [R, W]");
  vqb_attention_desc d{};
  d.prefix_len = int32(a[9], "prefix_len");
  const int32_t* prefix = nullptr;
  if (d.prefix_len != 0) {
    if (a[8] == Py_None) refuse("prefix_len needs prefix_pages");
    const Tensor& p = ints(a[8], "prefix_pages", dev);
    if (p.numel() * kc.size(2) < d.prefix_len) refuse("prefix_pages must cover prefix_len");
    prefix = ptr<int32_t>(p);
  }
  d.n_requests = int32(R, "R");
  d.n_tokens = int32(N, "N");
  d.heads = int32(H, "heads");
  d.kv_heads = int32(kc.size(1), "kv_heads");
  d.head_dim = int32(D, "D");
  d.page_size = int32(kc.size(2), "page_size");
  d.num_pages = int32(kc.size(0), "pages");
  d.table_width = int32(table.size(1), "W");
  d.max_q_len = int32(a[6], "max_q_len");
  d.max_kv_len = int32(a[7], "max_kv_len");
  d.causal = truth(a[11]);
  d.scale = a[10] == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(D))) : real(a[10]);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor out = a[12] == Py_None ? empty(q.sizes(), q.scalar_type(), dev) : heads(a[12], "out", q, q.sizes());
  d.q_token_stride = q.stride(0);
  d.q_head_stride = q.stride(1);
  d.out_token_stride = out.stride(0);
  d.out_head_stride = out.stride(1);
  d.kc_page_stride = kc.stride(0);
  d.kc_head_stride = kc.stride(1);
  d.kc_token_stride = kc.stride(2);
  d.vc_page_stride = vc.stride(0);
  d.vc_head_stride = vc.stride(1);
  d.vc_token_stride = vc.stride(2);
  Tensor lse;
  if (truth(a[13])) lse = empty({N, H}, at::kFloat, dev);
  const size_t need = g_abi.workspace_size(&d);
  Tensor ws;
  if (a[14] == Py_None) {
    ws = empty({static_cast<int64_t>(need ? need : 256)}, at::kByte, dev);
  } else {
    ws = tensor(a[14], "workspace");
    if (ws.scalar_type() != at::kByte || ws.device() != dev || !ws.is_contiguous() || static_cast<size_t>(ws.numel()) < need)
      refuse("workspace must be a uint8 CUDA tensor of >= " + std::to_string(need) + " bytes");
  }
  const vqb_status st = g_abi.prefix_attention(&d, code(q.scalar_type()), q.data_ptr(), kc.data_ptr(), vc.data_ptr(),
                                               ptr<int32_t>(table), ptr<int32_t>(lens), ptr<int32_t>(cu), prefix,
                                               out.data_ptr(), lse.defined() ? ptr<float>(lse) : nullptr, ws.data_ptr(),
                                               static_cast<size_t>(ws.numel()), stream(dev));
  if (st != VQB_OK) return status(st);
  if (!lse.defined()) return THPVariable_Wrap(out);
  THPObjectPtr r(PyTuple_New(2));
  if (!r) throw python_error();
  PyTuple_SET_ITEM(r.get(), 0, THPVariable_Wrap(out));
  PyTuple_SET_ITEM(r.get(), 1, THPVariable_Wrap(lse));
  return r.release();
  END_HANDLE_TH_ERRORS
}

// The addresses of vqb_paged_tables, vqb_rotary_append, vqb_prefix_attention_workspace_size, vqb_prefix_attention.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 4);
  void* at[4];
  for (int i = 0; i < 4; ++i) {
    at[i] = PyLong_AsVoidPtr(a[i]);
    if (!at[i]) {
      if (PyErr_Occurred()) throw python_error();
      refuse("bind: a null address");
    }
  }
  g_abi.paged_tables = reinterpret_cast<decltype(g_abi.paged_tables)>(at[0]);
  g_abi.rotary_append = reinterpret_cast<decltype(g_abi.rotary_append)>(at[1]);
  g_abi.workspace_size = reinterpret_cast<decltype(g_abi.workspace_size)>(at[2]);
  g_abi.prefix_attention = reinterpret_cast<decltype(g_abi.prefix_attention)>(at[3]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)); }

PyMethodDef kMethods[] = {
    {"bind", fast<bind>(), METH_FASTCALL, nullptr},
    {"paged_tables", fast<paged_tables>(), METH_FASTCALL, nullptr},
    {"rotary_append", fast<rotary_append>(), METH_FASTCALL, nullptr},
    {"prefix_attention", fast<prefix_attention>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&kModule); }
