// The repeated call of an operator, in C++: reads the tensors' metadata, allocates the result, fills the C-ABI struct and
// launches. A call of ten microseconds on the GPU spent as long again in Python on keys, checks and ctypes.
//
// Every function returns None for anything but the plain, valid case (other types, broadcast or copied operands, a
// missing workspace, another current device, an error of the library): the Python implementation then runs, checks and
// reports. Nothing is decided here that it would decide otherwise.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstring>
#include <memory>
#include <mutex>
#include <vector>

#include "../../include/b200_attn.h"
#include "../../include/b200_decoder.h"

namespace {

constexpr int64_t kHeadDim = 64, kSplitMinKeys = 257;

// Attention workspaces by (device, stream), registered by the Python side when it allocates them.
struct Workspace {
  int64_t device, stream;
  void* ptr;
  int64_t bytes;
};
std::mutex g_workspaces_mutex;
std::vector<Workspace> g_workspaces;

bool find_workspace(int64_t device, int64_t stream, void** ptr, int64_t* bytes) {
  std::lock_guard<std::mutex> lock(g_workspaces_mutex);
  for (const Workspace& w : g_workspaces)
    if (w.device == device && w.stream == stream) {
      *ptr = w.ptr;
      *bytes = w.bytes;
      return true;
    }
  return false;
}

PyObject* py_register_workspace(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "register_workspace(device, stream, pointer, bytes)");
    return nullptr;
  }
  int64_t v[4];
  for (int i = 0; i < 4; ++i) v[i] = static_cast<int64_t>(PyLong_AsUnsignedLongLongMask(args[i]));
  if (PyErr_Occurred()) return nullptr;
  std::lock_guard<std::mutex> lock(g_workspaces_mutex);
  for (Workspace& w : g_workspaces)
    if (w.device == v[0] && w.stream == v[1]) {
      w.ptr = reinterpret_cast<void*>(v[2]);
      w.bytes = v[3];
      Py_RETURN_NONE;
    }
  g_workspaces.push_back(Workspace{v[0], v[1], reinterpret_cast<void*>(v[2]), v[3]});
  Py_RETURN_NONE;
}

const at::Tensor* tensor_of(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool half_type(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
uint32_t dtype_code(const at::Tensor& t) { return t.scalar_type() == at::kHalf ? B200_ATTN_F16 : B200_ATTN_BF16; }

// A plain strided CUDA tensor (no subclass tricks, nothing lazy) on `device` that needs no gradient.
bool plain(const at::Tensor& t, c10::DeviceIndex device) {
  return t.is_cuda() && t.layout() == at::kStrided && t.device().index() == device && !t.is_conj() && !t.is_neg() &&
         !(t.requires_grad() && at::GradMode::is_enabled()) && t.has_storage();
}

at::Tensor empty_like_type(at::IntArrayRef sizes, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, like.scalar_type(), like.device(), std::nullopt);
}

// A call of the library, without the interpreter's lock.
template <typename F>
int launched(F&& f) {
  PyThreadState* state = PyEval_SaveThread();
  const int rc = f();
  PyEval_RestoreThread(state);
  return rc;
}

bool number(PyObject* o, double* v) {
  *v = PyFloat_AsDouble(o);
  if (*v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

// An int and nothing that converts to one, as ctypes has it for the fields these go to.
bool integer(PyObject* o, int64_t* v) {
  if (!PyLong_Check(o)) return false;
  int overflow = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow == 0 && *v >= INT32_MIN && *v <= INT32_MAX;
}

struct View {  // [batch, tokens, heads, 64] in either layout
  int64_t b, n, h, sb, sn, sh;
};
bool view_of(const at::Tensor& t, bool bnhd, View* v) {
  if (t.dim() != 4 || t.size(3) != kHeadDim || t.stride(3) != 1) return false;
  const int tok = bnhd ? 1 : 2, head = bnhd ? 2 : 1;
  *v = View{t.size(0), t.size(tok), t.size(head), t.stride(0), t.stride(tok), t.stride(head)};
  return v->b > 0 && v->n > 0 && v->h > 0;
}
void set_strides(int64_t* s, const View& v) {
  s[0] = v.sb;
  s[1] = v.sn;
  s[2] = v.sh;
}

// attention(q, k, v, scale | None, bnhd, schedule, out | None, bias | None, rel_h | None, rel_w | None, self_only)
PyObject* py_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 11) Py_RETURN_NONE;
  const at::Tensor *q = tensor_of(args[0]), *k = tensor_of(args[1]), *v = tensor_of(args[2]);
  if (q == nullptr || k == nullptr || v == nullptr) Py_RETURN_NONE;
  const bool bnhd = args[4] == Py_True;
  const c10::DeviceIndex device = c10::cuda::current_device();
  if (!half_type(*q) || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || !plain(*q, device) || !plain(*k, device) || !plain(*v, device))
    Py_RETURN_NONE;
  View vq, vk, vv;
  if (!view_of(*q, bnhd, &vq) || !view_of(*k, bnhd, &vk) || !view_of(*v, bnhd, &vv)) Py_RETURN_NONE;
  if (vk.b != vq.b || vk.h != vq.h || vv.b != vq.b || vv.h != vq.h || vv.n != vk.n || (args[10] == Py_True && vk.n != vq.n)) Py_RETURN_NONE;
  if (vq.n > INT32_MAX || vk.n > INT32_MAX || vq.b > INT32_MAX || vq.h > INT32_MAX) Py_RETURN_NONE;

  B200AttnArgs a;
  std::memset(&a, 0, sizeof(a));
  a.struct_size = sizeof(a);
  a.dtype = dtype_code(*q);
  a.q = q->data_ptr();
  a.k = k->data_ptr();
  a.v = v->data_ptr();
  set_strides(a.q_stride, vq);
  set_strides(a.k_stride, vk);
  set_strides(a.v_stride, vv);
  a.batch = static_cast<int32_t>(vq.b);
  a.heads = static_cast<int32_t>(vq.h);
  a.q_tokens = static_cast<int32_t>(vq.n);
  a.kv_tokens = static_cast<int32_t>(vk.n);
  a.head_dim = kHeadDim;
  double scale = 0.125;
  if (args[3] != Py_None && !number(args[3], &scale)) Py_RETURN_NONE;
  a.scale = static_cast<float>(scale);
  int64_t schedule = 0;
  if (!integer(args[5], &schedule)) Py_RETURN_NONE;
  a.schedule = static_cast<int32_t>(schedule);

  if (args[7] != Py_None) {  // a 16-bit bias the kernel fetches in tiles; a broadcast dimension has stride 0
    const at::Tensor* bias = tensor_of(args[7]);
    if (bias == nullptr || args[8] != Py_None || !half_type(*bias) || !plain(*bias, device) || bias->dim() > 4 || bias->dim() < 2) Py_RETURN_NONE;
    int64_t size[4] = {1, 1, 1, 1}, stride[4] = {0, 0, 0, 0};
    for (int64_t i = 0, at = 4 - bias->dim(); i < bias->dim(); ++i, ++at) {
      size[at] = bias->size(i);
      stride[at] = bias->stride(i);
    }
    if (size[3] != vk.n || size[2] != vq.n || stride[3] != 1 || (size[0] != 1 && size[0] != vq.b) || (size[1] != 1 && size[1] != vq.h)) Py_RETURN_NONE;
    for (int i = 0; i < 2; ++i)
      if (size[i] == 1) stride[i] = 0;
    if (reinterpret_cast<uintptr_t>(bias->data_ptr()) % 16 != 0 || stride[0] % 8 != 0 || stride[1] % 8 != 0 || stride[2] % 8 != 0 || stride[0] < 0 ||
        stride[1] < 0 || (stride[2] <= 0 && vq.n > 1))
      Py_RETURN_NONE;
    a.bias = bias->data_ptr();
    a.bias_dtype = dtype_code(*bias);
    for (int i = 0; i < 3; ++i) a.bias_stride[i] = stride[i];
  }
  if (args[8] != Py_None) {
    const at::Tensor *rh = tensor_of(args[8]), *rw = tensor_of(args[9]);
    if (rh == nullptr || rw == nullptr || rh->scalar_type() != rw->scalar_type() || (!half_type(*rh) && rh->scalar_type() != at::kFloat) || !plain(*rh, device) ||
        !plain(*rw, device) || rh->dim() != 4 || rw->dim() != 4)
      Py_RETURN_NONE;
    for (const at::Tensor* t : {rh, rw})
      if (t->size(0) != vq.b || t->size(1) != vq.h || t->size(2) != vq.n || t->stride(3) != 1) Py_RETURN_NONE;
    if (rh->size(3) * rw->size(3) != vk.n) Py_RETURN_NONE;
    a.rel_h = rh->data_ptr();
    a.rel_w = rw->data_ptr();
    a.rel_dtype = rh->scalar_type() == at::kFloat ? B200_ATTN_F32 : dtype_code(*rh);
    a.rel_kh = static_cast<int32_t>(rh->size(3));
    a.rel_kw = static_cast<int32_t>(rw->size(3));
    for (int i = 0; i < 3; ++i) {
      a.rel_h_stride[i] = rh->stride(i);
      a.rel_w_stride[i] = rw->stride(i);
    }
  }
  const int64_t stream = reinterpret_cast<int64_t>(c10::cuda::getCurrentCUDAStream(device).stream());
  if (vk.n >= kSplitMinKeys && !find_workspace(device, stream, &a.workspace, &a.workspace_bytes)) Py_RETURN_NONE;

  at::Tensor out;
  if (args[6] == Py_None) {
    out = empty_like_type({vq.b, vq.n, vq.h, kHeadDim}, *q);
    if (!bnhd) {  // the same memory as [batch, heads, tokens, 64]
      const int64_t sizes[4] = {vq.b, vq.h, vq.n, kHeadDim}, strides[4] = {vq.n * vq.h * kHeadDim, kHeadDim, vq.h * kHeadDim, 1};
      out.unsafeGetTensorImpl()->set_sizes_and_strides(c10::IntArrayRef(sizes), c10::IntArrayRef(strides));
    }
  } else {
    const at::Tensor* given = tensor_of(args[6]);
    if (given == nullptr || given->scalar_type() != q->scalar_type() || !given->is_cuda() || given->device().index() != device || given->sizes() != q->sizes())
      Py_RETURN_NONE;
    out = *given;
  }
  View vo;
  if (!view_of(out, bnhd, &vo)) Py_RETURN_NONE;
  a.o = out.data_ptr();
  set_strides(a.o_stride, vo);
  if (launched([&] { return b200_attn_fwd(&a, reinterpret_cast<void*>(stream)); }) != B200_ATTN_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(out);
}

// Row stride of `t` as [m, n] rows; false where the Python side has to look closer.
bool rows_of(const at::Tensor& t, int64_t m, int64_t n, int64_t* stride) {
  if (t.dim() < 1 || t.size(t.dim() - 1) != n || t.numel() != m * n) return false;
  if (t.is_contiguous()) {
    *stride = n;
    return true;
  }
  if (t.dim() != 2 || t.stride(1) != 1) return false;
  *stride = t.stride(0);
  return true;
}

// gemm(x, w, bias | None, act, scale | None, res | None, out | None)
PyObject* py_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7) Py_RETURN_NONE;
  const at::Tensor *x = tensor_of(args[0]), *w = tensor_of(args[1]);
  if (x == nullptr || w == nullptr) Py_RETURN_NONE;
  const c10::DeviceIndex device = c10::cuda::current_device();
  if (!half_type(*x) || w->scalar_type() != x->scalar_type() || !plain(*x, device) || !plain(*w, device) || x->dim() < 1 || x->numel() == 0 || w->dim() != 2 ||
      !w->is_contiguous())
    Py_RETURN_NONE;
  const int64_t k = x->size(x->dim() - 1), m = x->numel() / k, cols = w->size(0);
  if (w->size(1) != k || m > INT32_MAX || cols > INT32_MAX || k > INT32_MAX) Py_RETURN_NONE;
  B200GemmArgs a;
  std::memset(&a, 0, sizeof(a));
  a.struct_size = sizeof(a);
  a.dtype = dtype_code(*x);
  a.m = static_cast<int32_t>(m);
  a.n = static_cast<int32_t>(cols);
  a.k = static_cast<int32_t>(k);
  int64_t act = 0;
  if (!integer(args[3], &act)) Py_RETURN_NONE;
  a.act = static_cast<int32_t>(act);
  if (!rows_of(*x, m, k, &a.lda)) Py_RETURN_NONE;
  a.x = x->data_ptr();
  a.w = w->data_ptr();
  if (args[2] != Py_None) {
    const at::Tensor* b = tensor_of(args[2]);
    if (b == nullptr || b->scalar_type() != x->scalar_type() || !plain(*b, device) || b->dim() != 1 || b->size(0) != cols || b->stride(0) != 1) Py_RETURN_NONE;
    a.bias = b->data_ptr();
  }
  if (args[4] != Py_None) {
    const at::Tensor* s = tensor_of(args[4]);
    if (s == nullptr || s->scalar_type() != at::kFloat || !plain(*s, device) || s->dim() != 1 || s->size(0) != cols || s->stride(0) != 1) Py_RETURN_NONE;
    a.scale = static_cast<const float*>(s->data_ptr());
  }
  if (args[5] != Py_None) {
    const at::Tensor* r = tensor_of(args[5]);
    if (r == nullptr || r->scalar_type() != x->scalar_type() || !plain(*r, device) || !rows_of(*r, m, cols, &a.lres)) Py_RETURN_NONE;
    a.res = r->data_ptr();
  }
  at::Tensor out;
  if (args[6] == Py_None) {
    c10::SmallVector<int64_t, 5> sizes(x->sizes().begin(), x->sizes().end());
    sizes.back() = cols;
    out = empty_like_type(sizes, *x);
  } else {
    const at::Tensor* given = tensor_of(args[6]);
    if (given == nullptr || given->scalar_type() != x->scalar_type() || !plain(*given, device)) Py_RETURN_NONE;
    out = *given;
  }
  if (!rows_of(out, m, cols, &a.ldy)) Py_RETURN_NONE;
  a.y = out.data_ptr();
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  if (launched([&] { return b200_gemm(&a, stream.stream()); }) != B200_ATTN_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(out);
}

// rope_qk_(qkv, cs, q_scale) -> whether it was launched
PyObject* py_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3) Py_RETURN_FALSE;
  const at::Tensor *x = tensor_of(args[0]), *cs = tensor_of(args[1]);
  if (x == nullptr || cs == nullptr) Py_RETURN_FALSE;
  const c10::DeviceIndex device = c10::cuda::current_device();
  if (!half_type(*x) || !plain(*x, device) || !plain(*cs, device) || x->dim() != 5 || x->size(2) != 3 || x->size(4) != kHeadDim || x->stride(4) != 1 ||
      x->numel() == 0 || cs->scalar_type() != at::kFloat || cs->dim() != 3 || cs->size(1) != 2 || cs->size(2) != kHeadDim / 2 || !cs->is_contiguous() ||
      cs->size(0) > x->size(1) || x->size(0) > INT32_MAX || x->size(1) > INT32_MAX || x->size(3) > INT32_MAX)
    Py_RETURN_FALSE;
  double scale = 1;
  if (!number(args[2], &scale)) Py_RETURN_FALSE;
  B200RopeArgs a;
  std::memset(&a, 0, sizeof(a));
  a.struct_size = sizeof(a);
  a.dtype = dtype_code(*x);
  a.q = x->data_ptr();
  a.k = static_cast<char*>(x->data_ptr()) + 2 * x->stride(2);
  for (int64_t* s : {a.q_stride, a.k_stride}) {
    s[0] = x->stride(0);
    s[1] = x->stride(1);
    s[2] = x->stride(3);
  }
  a.cs = static_cast<const float*>(cs->data_ptr());
  a.batch = static_cast<int32_t>(x->size(0));
  a.heads = static_cast<int32_t>(x->size(3));
  a.tokens = static_cast<int32_t>(x->size(1));
  a.prefix = static_cast<int32_t>(x->size(1) - cs->size(0));
  a.head_dim = kHeadDim;
  a.q_scale = static_cast<float>(scale);
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  if (launched([&] { return b200_rope_qk(&a, stream.stream()); }) != B200_ATTN_OK) Py_RETURN_FALSE;
  Py_RETURN_TRUE;
}

// ---- a token decoder's layers ----

bool heads_type(const at::Tensor& t) { return half_type(t) || t.scalar_type() == at::kFloat; }
uint32_t any_dtype_code(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? B200_ATTN_F32 : dtype_code(t); }
bool fits32(const at::Tensor& t) {
  for (int64_t n : t.sizes())
    if (n > INT32_MAX) return false;
  return true;
}
// A plain CUDA tensor on `device` as above, which may need a gradient but carries no tangent of forward-mode differentiation.
bool on_device(const at::Tensor& t, c10::DeviceIndex device) {
  return t.is_cuda() && t.layout() == at::kStrided && t.device().index() == device && !t.is_conj() && !t.is_neg() && t.has_storage() && !t._fw_grad(0).defined();
}
bool wants_grad(const at::Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }
// A plain, filled tensor of heads with unit last stride.
bool heads_on(const at::Tensor* t, c10::DeviceIndex device) {
  return t != nullptr && on_device(*t, device) && t->dim() == 4 && t->stride(3) == 1 && t->numel() > 0 && fits32(*t);
}
bool heads_of(const at::Tensor* t, c10::DeviceIndex device) { return heads_on(t, device) && plain(*t, device); }
void set_heads(int64_t* s, const at::Tensor& t) {
  for (int i = 0; i < 3; ++i) s[i] = t.stride(i);
}
bool table_of(const at::Tensor* t, c10::DeviceIndex device, int64_t dim) {
  return t != nullptr && plain(*t, device) && t->scalar_type() == at::kFloat && t->dim() == 3 && t->size(1) == 2 && t->size(0) >= 1 && t->size(2) >= 1 && 2 * t->size(2) <= dim &&
         t->is_contiguous() && fits32(*t);
}

// Table and positions (undefined: none) as they go with the tokens of x.
bool turn_of(const at::Tensor& x, PyObject* table, PyObject* positions, c10::DeviceIndex device, at::Tensor* t, at::Tensor* p) {
  if (table == Py_None) return positions == Py_None;
  const at::Tensor* given = tensor_of(table);
  if (!table_of(given, device, x.size(3))) return false;
  *t = *given;
  if (positions == Py_None) return t->size(0) >= x.size(1);
  given = tensor_of(positions);
  if (given == nullptr || !plain(*given, device) || given->scalar_type() != at::kInt) return false;
  *p = *given;
  return (p->dim() == 1 && p->size(0) == x.size(1)) || (p->dim() == 2 && p->size(0) == x.size(0) && p->size(1) == x.size(1));
}

void set_rotary(B200RotaryArgs* a, const at::Tensor& x, const at::Tensor& table, const at::Tensor& positions, bool interleaved) {
  std::memset(a, 0, sizeof(*a));
  a->struct_size = sizeof(*a);
  a->dtype = a->weight_dtype = any_dtype_code(x);
  a->batch = static_cast<int32_t>(x.size(0));
  a->tokens = static_cast<int32_t>(x.size(1));
  a->head_dim = static_cast<int32_t>(x.size(3));
  a->interleaved = interleaved;
  if (table.defined()) {
    a->cs = static_cast<const float*>(table.data_ptr());
    a->rot = static_cast<int32_t>(2 * table.size(2));
    a->table_rows = static_cast<int32_t>(table.size(0));
  }
  if (positions.defined()) {
    a->positions = static_cast<const int32_t*>(positions.data_ptr());
    a->pos_stride[0] = positions.dim() == 2 ? positions.stride(0) : 0;
    a->pos_stride[1] = positions.stride(-1);
  }
}

// One tensor of a call: x and y, or, with g, what goes backward.
void add_heads(B200RotaryArgs* a, const at::Tensor& x, const at::Tensor& y, const at::Tensor& g = {}) {
  B200Heads& h = a->heads[a->tensors++];
  h.x = x.defined() ? x.data_ptr() : nullptr;
  h.y = y.data_ptr();
  if (x.defined()) set_heads(h.x_stride, x);
  set_heads(h.y_stride, y);
  if (g.defined()) {
    h.g = g.data_ptr();
    set_heads(h.g_stride, g);
  }
  h.heads = static_cast<int32_t>(y.size(2));
}

// Scratch for the sums behind the weights' gradients by (device, stream), kept until the process ends; a capture gets its own.
struct Scratch {
  int64_t device, stream;
  at::Tensor* memory;
};
std::vector<Scratch> g_rotary_scratch;
constexpr int64_t kHeaderBytes = 256;  // zeroed

at::Tensor rotary_scratch(const at::Tensor& like, const c10::cuda::CUDAStream& stream) {
  const int64_t device = like.device().index(), id = reinterpret_cast<int64_t>(stream.stream());
  std::lock_guard<std::mutex> lock(g_workspaces_mutex);
  for (const Scratch& s : g_rotary_scratch)
    if (s.device == device && s.stream == id) return *s.memory;
  int64_t bytes = 0;
  TORCH_CHECK(b200_rotary_workspace(&bytes) == B200_ATTN_OK, "rotary workspace: ", b200_attn_last_error());
  const at::Tensor memory = at::empty({bytes}, like.options().dtype(at::kByte).requires_grad(false));
  memory.narrow(0, 0, kHeaderBytes).zero_();
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(stream.stream(), &capture) == cudaSuccess && capture == cudaStreamCaptureStatusNone) g_rotary_scratch.push_back({device, id, new at::Tensor(memory)});
  return memory;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A gradient that comes in, as the kernels take it.
at::Tensor incoming(const at::Tensor& g, const at::Tensor& like) {
  if (!g.defined()) return at::zeros_like(like, at::MemoryFormat::Contiguous);
  return g.stride(-1) == 1 || g.size(-1) == 1 ? g : g.contiguous();
}
// Gradients that must not be differentiated again, should somebody try (the kernels have no second derivative).
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list marked;
  for (const at::Tensor& g : grads) marked.push_back(g.defined() ? g.detach().requires_grad_(true) : g);
  auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable", static_cast<int64_t>(marked.size()));
  return (*error)(std::move(marked));
}

at::Tensor turned(const at::Tensor& x, const at::Tensor& table, const at::Tensor& positions, bool interleaved) {
  at::Tensor y = empty_like_type(x.sizes(), x);
  B200RotaryArgs a;
  set_rotary(&a, x, table, positions, interleaved);
  add_heads(&a, x, y);
  TORCH_CHECK(b200_rotary(&a, c10::cuda::getCurrentCUDAStream(x.device().index()).stream()) == B200_ATTN_OK, "rotary: ", b200_attn_last_error());
  return y;
}

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& table, const at::Tensor& positions, bool interleaved) {
    ctx->save_for_backward({table, positions});
    ctx->saved_data["interleaved"] = interleaved;
    return turned(x, table, positions, interleaved);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list result(4);
    {
      const at::NoGradGuard guard;
      const c10::cuda::CUDAGuard on(grads[0].device());
      const at::Tensor g = incoming(grads[0], grads[0]);
      result[0] = empty_like_type(g.sizes(), g);
      B200RotaryArgs a;
      set_rotary(&a, g, saved[0], saved[1], ctx->saved_data["interleaved"].toBool());
      a.backward = 1;
      add_heads(&a, {}, result[0], g);
      TORCH_CHECK(b200_rotary(&a, c10::cuda::getCurrentCUDAStream(g.device().index()).stream()) == B200_ATTN_OK, "rotary: ", b200_attn_last_error());
    }
    return once(std::move(result));
  }
};

// rotary(x, table, positions | None, interleaved)
PyObject* py_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4 || !PyBool_Check(args[3]) || args[1] == Py_None) Py_RETURN_NONE;
  const at::Tensor* x = tensor_of(args[0]);
  const c10::DeviceIndex device = c10::cuda::current_device();
  at::Tensor table, positions;
  if (!heads_on(x, device) || !heads_type(*x) || !turn_of(*x, args[1], args[2], device, &table, &positions)) Py_RETURN_NONE;
  const bool interleaved = args[3] == Py_True;
  return THPVariable_Wrap(wants_grad(*x) ? RotaryFunction::apply(*x, table, positions, interleaved) : turned(*x, table, positions, interleaved));
}

// x, weights (undefined: none) and results of the two tensors.
variable_list normed(const at::Tensor* x, const at::Tensor* w, const at::Tensor& table, const at::Tensor& positions, double eps, bool interleaved) {
  B200RotaryArgs a;
  set_rotary(&a, x[0], table, positions, interleaved);
  a.norm = 1;
  a.eps = static_cast<float>(eps);
  variable_list y;
  for (int k = 0; k < 2; ++k) {
    y.push_back(empty_like_type(x[k].sizes(), x[k]));
    add_heads(&a, x[k], y[k]);
    if (!w[k].defined()) continue;
    a.heads[k].w = w[k].data_ptr();
    a.weight_dtype = any_dtype_code(w[k]);
  }
  TORCH_CHECK(b200_rotary(&a, c10::cuda::getCurrentCUDAStream(x[0].device().index()).stream()) == B200_ATTN_OK, "qk_norm_rotary: ", b200_attn_last_error());
  return y;
}

struct QkNormRotaryFunction : torch::autograd::Function<QkNormRotaryFunction> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& table, const at::Tensor& positions, double eps, bool interleaved) {
    ctx->save_for_backward({q, k, wq, wk, table, positions});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    const at::Tensor x[2] = {q, k}, w[2] = {wq, wk};
    return normed(x, w, table, positions, eps, interleaved);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list result(8);
    {
      const at::NoGradGuard guard;
      const c10::cuda::CUDAGuard on(saved[0].device());
      const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(saved[0].device().index());
      B200RotaryArgs a;
      set_rotary(&a, saved[0], saved[4], saved[5], ctx->saved_data["interleaved"].toBool());
      a.norm = a.backward = 1;
      a.eps = static_cast<float>(ctx->saved_data["eps"].toDouble());
      at::Tensor scratch, g[2];
      for (int i = 0; i < 2; ++i) {
        const at::Tensor &x = saved[i], &w = saved[2 + i];
        g[i] = incoming(grads[i], x);
        result[i] = empty_like_type(x.sizes(), x);
        add_heads(&a, x, result[i], g[i]);
        a.heads[i].w = w.data_ptr();
        a.weight_dtype = any_dtype_code(w);
        if (!ctx->needs_input_grad(2 + i)) continue;
        result[2 + i] = empty_like_type(w.sizes(), w);
        a.heads[i].dw = result[2 + i].data_ptr();
        if (!scratch.defined()) scratch = rotary_scratch(x, stream);
        a.workspace = scratch.data_ptr();
        a.workspace_bytes = scratch.numel();
      }
      TORCH_CHECK(b200_rotary(&a, stream.stream()) == B200_ATTN_OK, "qk_norm_rotary: ", b200_attn_last_error());
    }
    return once(std::move(result));
  }
};

// qk_norm_rotary(q, k, q_weight | None, k_weight | None, table | None, positions | None, eps, interleaved)
PyObject* py_qk_norm_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 8 || !PyBool_Check(args[7])) Py_RETURN_NONE;
  const c10::DeviceIndex device = c10::cuda::current_device();
  const at::Tensor* x[2] = {tensor_of(args[0]), tensor_of(args[1])};
  double eps = 0;
  if (!heads_on(x[0], device) || !heads_on(x[1], device) || !heads_type(*x[0]) || x[1]->scalar_type() != x[0]->scalar_type() || !number(args[6], &eps) || !(eps >= 0)) Py_RETURN_NONE;
  for (int i : {0, 1, 3})
    if (x[1]->size(i) != x[0]->size(i)) Py_RETURN_NONE;
  at::Tensor table, positions, w[2];
  if (!turn_of(*x[0], args[4], args[5], device, &table, &positions)) Py_RETURN_NONE;
  bool grad = wants_grad(*x[0]) || wants_grad(*x[1]);
  for (int k = 0; k < 2; ++k) {
    if (args[2 + k] == Py_None) continue;
    const at::Tensor* given = tensor_of(args[2 + k]);
    if (given == nullptr || !on_device(*given, device) || given->dim() != 1 || given->size(0) != x[0]->size(3) || !given->is_contiguous()) Py_RETURN_NONE;
    if (given->scalar_type() != x[0]->scalar_type() && given->scalar_type() != at::kFloat) Py_RETURN_NONE;
    if (k == 1 && w[0].defined() && w[0].scalar_type() != given->scalar_type()) Py_RETURN_NONE;
    w[k] = *given;
    grad = grad || wants_grad(w[k]);
  }
  if (grad && (!w[0].defined() || !w[1].defined())) Py_RETURN_NONE;  // the Python side has the gradient for any mix
  const bool interleaved = args[7] == Py_True;
  const at::Tensor both[2] = {*x[0], *x[1]};
  const variable_list y = grad ? QkNormRotaryFunction::apply(both[0], both[1], w[0], w[1], table, positions, eps, interleaved) : normed(both, w, table, positions, eps, interleaved);
  return Py_BuildValue("(NN)", THPVariable_Wrap(y[0]), THPVariable_Wrap(y[1]));
}

// Cache, page table and lengths of a call on `batch` sequences.
template <typename A>
bool set_cache(A* a, PyObject* cache, PyObject* page_table, PyObject* lengths, int64_t batch, c10::DeviceIndex device) {
  const at::Tensor *c = tensor_of(cache), *t = tensor_of(page_table), *l = tensor_of(lengths);
  if (c == nullptr || t == nullptr || l == nullptr || !plain(*c, device) || !plain(*t, device) || !plain(*l, device)) return false;
  if (c->scalar_type() != at::kByte || c->dim() != 4 || !c->is_contiguous() || c->numel() == 0 || !fits32(*c)) return false;
  if (c->size(3) != 16 * (64 + 8) && c->size(3) != 16 * (128 + 8)) return false;
  if (t->scalar_type() != at::kInt || t->dim() != 2 || t->size(0) != batch || t->size(1) < 1 || t->stride(1) != 1 || !fits32(*t)) return false;
  if (l->scalar_type() != at::kInt || l->dim() != 1 || l->size(0) != batch || !l->is_contiguous()) return false;
  if (c->size(2) > INT32_MAX / 16) return false;
  a->struct_size = sizeof(*a);
  a->batch = static_cast<int32_t>(batch);
  a->kv_heads = static_cast<int32_t>(c->size(1));
  a->head_dim = static_cast<int32_t>(c->size(3) / 16 - 8);
  a->page = static_cast<int32_t>(16 * c->size(2));
  a->pages = static_cast<int32_t>(c->size(0));
  a->table_pages = static_cast<int32_t>(t->size(1));
  a->cache = static_cast<uint8_t*>(c->data_ptr());
  a->page_table = static_cast<const int32_t*>(t->data_ptr());
  a->table_stride = t->stride(0);
  a->lengths = static_cast<const int32_t*>(l->data_ptr());
  return true;
}

// kv4_append_(cache, k, v, page_table, lengths, table | None, interleaved, q | None) -> the turned q, or True without q
PyObject* py_kv4_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 8 || !PyBool_Check(args[6])) Py_RETURN_NONE;
  const c10::DeviceIndex device = c10::cuda::current_device();
  const at::Tensor *k = tensor_of(args[1]), *v = tensor_of(args[2]), *q = tensor_of(args[7]);
  if (!heads_of(k, device) || !heads_of(v, device) || !half_type(*k) || v->scalar_type() != k->scalar_type() || v->sizes() != k->sizes()) Py_RETURN_NONE;
  B200Kv4Args a;
  std::memset(&a, 0, sizeof(a));
  if (!set_cache(&a, args[0], args[3], args[4], k->size(0), device) || k->size(2) != a.kv_heads || k->size(3) != a.head_dim) Py_RETURN_NONE;
  if (args[5] != Py_None) {
    const at::Tensor* t = tensor_of(args[5]);
    if (!table_of(t, device, a.head_dim)) Py_RETURN_NONE;
    a.cs = static_cast<const float*>(t->data_ptr());
    a.rot = static_cast<int32_t>(2 * t->size(2));
    a.table_rows = static_cast<int32_t>(t->size(0));
  }
  a.dtype = dtype_code(*k);
  a.tokens = static_cast<int32_t>(k->size(1));
  a.interleaved = args[6] == Py_True;
  a.k = k->data_ptr();
  a.v = v->data_ptr();
  set_heads(a.k_stride, *k);
  set_heads(a.v_stride, *v);
  at::Tensor out;
  if (args[7] != Py_None) {
    if (!heads_of(q, device) || q->scalar_type() != k->scalar_type() || q->size(0) != k->size(0) || q->size(1) != k->size(1) || q->size(3) != k->size(3)) Py_RETURN_NONE;
    out = empty_like_type(q->sizes(), *q);
    a.q_heads = static_cast<int32_t>(q->size(2));
    a.q = q->data_ptr();
    a.q_out = out.data_ptr();
    set_heads(a.q_stride, *q);
    set_heads(a.q_out_stride, out);
  }
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  if (launched([&] { return b200_kv4_append(&a, stream.stream()); }) != B200_ATTN_OK) Py_RETURN_NONE;
  if (args[7] == Py_None) Py_RETURN_TRUE;
  return THPVariable_Wrap(out);
}

// kv4_read(cache, page_table, lengths, tokens, True: fp16 | False: bf16 | None)
PyObject* py_kv4_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5 || !PyBool_Check(args[4])) Py_RETURN_NONE;
  const c10::DeviceIndex device = c10::cuda::current_device();
  const at::Tensor *c = tensor_of(args[0]), *l = tensor_of(args[2]);
  int64_t tokens = 0;
  if (c == nullptr || l == nullptr || l->dim() != 1 || l->size(0) < 1 || !integer(args[3], &tokens) || tokens < 1) Py_RETURN_NONE;
  B200Kv4Args a;
  std::memset(&a, 0, sizeof(a));
  if (!set_cache(&a, args[0], args[1], args[2], l->size(0), device)) Py_RETURN_NONE;
  const bool f16 = args[4] == Py_True;
  a.dtype = f16 ? B200_ATTN_F16 : B200_ATTN_BF16;
  a.tokens = static_cast<int32_t>(tokens);
  const int64_t sizes[4] = {a.batch, tokens, a.kv_heads, a.head_dim};
  at::Tensor k = at::detail::empty_cuda(sizes, f16 ? at::kHalf : at::kBFloat16, c->device(), std::nullopt);
  at::Tensor v = at::detail::empty_cuda(sizes, f16 ? at::kHalf : at::kBFloat16, c->device(), std::nullopt);
  a.k_out = k.data_ptr();
  a.v_out = v.data_ptr();
  set_heads(a.k_out_stride, k);
  set_heads(a.v_out_stride, v);
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  if (launched([&] { return b200_kv4_read(&a, stream.stream()); }) != B200_ATTN_OK) Py_RETURN_NONE;
  return Py_BuildValue("(NN)", THPVariable_Wrap(k), THPVariable_Wrap(v));
}

// Workspace and counters of attention over the cache, registered like the attention workspaces above.
struct Kv4Workspace {
  int64_t v[6];  // device, stream, workspace, bytes, counters, words
};
std::vector<Kv4Workspace> g_kv4_workspaces;

PyObject* py_register_kv4_workspace(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "register_kv4_workspace(device, stream, workspace, bytes, counters, words)");
    return nullptr;
  }
  Kv4Workspace w;
  for (int i = 0; i < 6; ++i) w.v[i] = static_cast<int64_t>(PyLong_AsUnsignedLongLongMask(args[i]));
  if (PyErr_Occurred()) return nullptr;
  std::lock_guard<std::mutex> lock(g_workspaces_mutex);
  for (Kv4Workspace& had : g_kv4_workspaces)
    if (had.v[0] == w.v[0] && had.v[1] == w.v[1]) {
      had = w;
      Py_RETURN_NONE;
    }
  g_kv4_workspaces.push_back(w);
  Py_RETURN_NONE;
}

// kv4_attention(q, cache, page_table, lengths, scale | None)
PyObject* py_kv4_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) Py_RETURN_NONE;
  const c10::DeviceIndex device = c10::cuda::current_device();
  const at::Tensor* q = tensor_of(args[0]);
  if (!heads_of(q, device) || !half_type(*q)) Py_RETURN_NONE;
  B200Kv4AttnArgs a;
  std::memset(&a, 0, sizeof(a));
  if (!set_cache(&a, args[1], args[2], args[3], q->size(0), device) || q->size(3) != a.head_dim || q->size(2) % a.kv_heads != 0) Py_RETURN_NONE;
  double scale = 0;
  if (args[4] == Py_None) a.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(a.head_dim)));
  else if (number(args[4], &scale)) a.scale = static_cast<float>(scale);
  else Py_RETURN_NONE;
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  {
    std::lock_guard<std::mutex> lock(g_workspaces_mutex);
    for (const Kv4Workspace& w : g_kv4_workspaces)
      if (w.v[0] == device && w.v[1] == reinterpret_cast<int64_t>(stream.stream())) {
        a.workspace = reinterpret_cast<void*>(w.v[2]);
        a.workspace_bytes = w.v[3];
        a.counters = reinterpret_cast<uint32_t*>(w.v[4]);
        a.counter_words = w.v[5];
      }
  }
  if (a.workspace == nullptr) Py_RETURN_NONE;
  at::Tensor out = empty_like_type(q->sizes(), *q);
  a.dtype = dtype_code(*q);
  a.queries = static_cast<int32_t>(q->size(1));
  a.q_heads = static_cast<int32_t>(q->size(2));
  a.q = q->data_ptr();
  a.o = out.data_ptr();
  set_heads(a.q_stride, *q);
  set_heads(a.o_stride, out);
  if (launched([&] { return b200_kv4_attention(&a, stream.stream()); }) != B200_ATTN_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(out);
}

// sam_rel_terms(q, rel_pos_h, rel_pos_w, side)
PyObject* py_rel_terms(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4) Py_RETURN_NONE;
  const at::Tensor *q = tensor_of(args[0]), *ph = tensor_of(args[1]), *pw = tensor_of(args[2]);
  int64_t side = 0;
  if (q == nullptr || ph == nullptr || pw == nullptr || !integer(args[3], &side)) Py_RETURN_NONE;
  const c10::DeviceIndex device = c10::cuda::current_device();
  View v;
  if (!half_type(*q) || !plain(*q, device) || !view_of(*q, true, &v) || side < 2 || side > 64 || v.n != side * side || v.b > INT32_MAX || v.h > INT32_MAX) Py_RETURN_NONE;
  for (const at::Tensor* t : {ph, pw})
    if (t->scalar_type() != q->scalar_type() || !plain(*t, device) || t->dim() != 2 || t->size(0) != 2 * side - 1 || t->size(1) != kHeadDim || !t->is_contiguous())
      Py_RETURN_NONE;
  at::Tensor rel_h = empty_like_type({v.b, v.h, v.n, side}, *q), rel_w = empty_like_type({v.b, v.h, v.n, side}, *q);
  B200RelTermsArgs a;
  std::memset(&a, 0, sizeof(a));
  a.struct_size = sizeof(a);
  a.dtype = dtype_code(*q);
  a.q = q->data_ptr();
  set_strides(a.q_stride, v);
  a.rel_pos_h = ph->data_ptr();
  a.rel_pos_w = pw->data_ptr();
  a.rel_h = rel_h.data_ptr();
  a.rel_w = rel_w.data_ptr();
  a.batch = static_cast<int32_t>(v.b);
  a.heads = static_cast<int32_t>(v.h);
  a.side = static_cast<int32_t>(side);
  a.head_dim = kHeadDim;
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  if (launched([&] { return b200_sam_rel_terms(&a, stream.stream()); }) != B200_ATTN_OK) Py_RETURN_NONE;
  PyObject *h = THPVariable_Wrap(rel_h), *w = THPVariable_Wrap(rel_w);
  PyObject* pair = PyTuple_Pack(2, h, w);
  Py_DECREF(h);
  Py_DECREF(w);
  return pair;
}

// What an encoder's table of parameter addresses was made from (encoder.py: Snapshot). The tensors are held, so an address
// cannot come to mean another one while it is compared with.
struct Fact {
  at::Tensor tensor;
  const void* ptr;
  c10::SmallVector<int64_t, 4> sizes, strides;
};
using Facts = std::vector<Fact>;
constexpr const char* kFactsName = "_b200host.snapshot";

void free_facts(PyObject* capsule) { delete static_cast<Facts*>(PyCapsule_GetPointer(capsule, kFactsName)); }

// Calls f(tensor) for every value of every dictionary in the tuple `dicts`; false as soon as f says so or one is no tensor.
template <typename F>
bool for_each_tensor(PyObject* dicts, F&& f) {
  if (!PyTuple_Check(dicts)) return false;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(dicts); ++i) {
    PyObject* d = PyTuple_GET_ITEM(dicts, i);
    if (!PyDict_Check(d)) return false;
    PyObject *key = nullptr, *value = nullptr;
    for (Py_ssize_t at = 0; PyDict_Next(d, &at, &key, &value);) {
      const at::Tensor* t = tensor_of(value);
      if (t == nullptr || !t->has_storage() || !f(*t)) return false;
    }
  }
  return true;
}

// snapshot(dicts) -> capsule, or None for anything but dictionaries of plain tensors
PyObject* py_snapshot(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 1) Py_RETURN_NONE;
  auto facts = std::make_unique<Facts>();
  const auto take = [&](const at::Tensor& t) {
    facts->push_back(Fact{t, t.const_data_ptr(), {t.sizes().begin(), t.sizes().end()}, {t.strides().begin(), t.strides().end()}});
    return true;
  };
  if (!for_each_tensor(args[0], take)) Py_RETURN_NONE;
  PyObject* capsule = PyCapsule_New(facts.get(), kFactsName, free_facts);
  if (capsule != nullptr) facts.release();
  return capsule;
}

// unchanged(capsule, dicts): the same tensors in the same places
PyObject* py_unchanged(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2 || !PyCapsule_IsValid(args[0], kFactsName)) Py_RETURN_FALSE;
  const Facts& facts = *static_cast<Facts*>(PyCapsule_GetPointer(args[0], kFactsName));
  size_t i = 0;
  const auto same = [&](const at::Tensor& t) {
    if (i >= facts.size()) return false;
    const Fact& f = facts[i++];
    return t.is_same(f.tensor) && t.const_data_ptr() == f.ptr && t.sizes().equals(f.sizes) && t.strides().equals(f.strides);
  };
  if (for_each_tensor(args[1], same) && i == facts.size()) Py_RETURN_TRUE;
  Py_RETURN_FALSE;
}

// C++ exceptions (an allocation that fails) must not cross into the interpreter: the Python side runs and reports.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    return F(self, args, n);
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<F>));
}

PyMethodDef methods[] = {
    {"attention", fast<py_attention>(), METH_FASTCALL, nullptr},
    {"gemm", fast<py_gemm>(), METH_FASTCALL, nullptr},
    {"rope_qk_", fast<py_rope>(), METH_FASTCALL, nullptr},
    {"sam_rel_terms", fast<py_rel_terms>(), METH_FASTCALL, nullptr},
    {"snapshot", fast<py_snapshot>(), METH_FASTCALL, nullptr},
    {"unchanged", fast<py_unchanged>(), METH_FASTCALL, nullptr},
    {"rotary", fast<py_rotary>(), METH_FASTCALL, nullptr},
    {"qk_norm_rotary", fast<py_qk_norm_rotary>(), METH_FASTCALL, nullptr},
    {"kv4_append_", fast<py_kv4_append>(), METH_FASTCALL, nullptr},
    {"kv4_read", fast<py_kv4_read>(), METH_FASTCALL, nullptr},
    {"kv4_attention", fast<py_kv4_attention>(), METH_FASTCALL, nullptr},
    {"register_kv4_workspace", fast<py_register_kv4_workspace>(), METH_FASTCALL, nullptr},
    {"register_workspace", fast<py_register_workspace>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

#ifndef B200_SOURCE_HASH
#define B200_SOURCE_HASH "0000000000000000"
#endif
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_b200host", "b200attn-src:" B200_SOURCE_HASH, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__b200host(void) { return PyModule_Create(&module_def); }
