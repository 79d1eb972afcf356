// The calls of decode.py, logits.py and beam.py without Python in between, for plain CUDA tensors that the kernels can read in place.  Whatever they do not cover they leave, untouched, to the Python code (they return None), which also raises all errors.
// A step's kernels take a few us; through Python and ctypes a call of the attention over 187 tokens took 24 us and one of the logits 30,
// here 6 and 6.
#include "host_common.h"

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>

#include <algorithm>
#include <cmath>
#include <vector>

namespace {

constexpr const char* kName = "pbs_attn_b200.paged_cache";

// A cache's struct, which lives as long as the Python object that owns this.
struct Cache {
  const pbs_paged_cache_t* c;
  int device;
  at::ScalarType type;
  decltype(&pbs_paged_append) append;
  decltype(&pbs_paged_gather) gather;
  decltype(&pbs_paged_attn) attn;
  decltype(&pbs_paged_attn_workspace) workspace;
};

Cache* get(PyObject* capsule) { return static_cast<Cache*>(PyCapsule_GetPointer(capsule, kName)); }
void destroy(PyObject* capsule) { delete static_cast<Cache*>(PyCapsule_GetPointer(capsule, kName)); }

// paged_attach(struct, device, append, gather, attn, workspace): addresses -> the cache's object here
PyObject* py_attach(PyObject*, PyObject* args) {
  unsigned long long c, f[4];
  int device;
  if (!PyArg_ParseTuple(args, "KiKKKK", &c, &device, &f[0], &f[1], &f[2], &f[3])) return nullptr;
  const auto* cache = reinterpret_cast<const pbs_paged_cache_t*>(c);
  return PyCapsule_New(new Cache{cache, device, cache->dtype == PBS_BF16 ? at::kBFloat16 : at::kHalf, reinterpret_cast<decltype(&pbs_paged_append)>(f[0]),
                                 reinterpret_cast<decltype(&pbs_paged_gather)>(f[1]), reinterpret_cast<decltype(&pbs_paged_attn)>(f[2]),
                                 reinterpret_cast<decltype(&pbs_paged_attn_workspace)>(f[3])},
                       kName, destroy);
}

bool plain(PyObject* o) { return THPVariable_CheckExact(o) && THPVariable_Unpack(o).layout() == at::kStrided; }

// A tensor of integers or floats on the device whose last dimension is dense.
bool dense_on(PyObject* o, int device, at::ScalarType type, int64_t dims) {
  if (!plain(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.device().index() == device && t.scalar_type() == type && t.dim() == dims && (t.size(dims - 1) <= 1 || t.stride(dims - 1) == 1);
}

bool rows_of(const Cache* c, PyObject* o, int64_t B, int64_t heads, int64_t S) {        // (B, heads, S, D) of the cache's type; heads < 0: a multiple of its
  if (!plain(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.device().index() != c->device || t.scalar_type() != c->type || t.dim() != 4) return false;
  if (t.size(0) != B || t.size(2) != S || t.size(3) != c->c->head_dim) return false;
  if (heads >= 0 ? t.size(1) != heads : t.size(1) == 0 || t.size(1) % c->c->kv_heads != 0) return false;
  return readable(t, false);
}

bool batch_of(const Cache* c, PyObject* table, PyObject* lens, PyObject* new_lens, int64_t B, int64_t S, pbs_paged_batch_t* out) {
  if (*const_cast<volatile int32_t*>(c->c->status) != 0) return false;                  // Python tells of the fault
  if (B < 1 || S < 1 || B > INT32_MAX || S > INT32_MAX) return false;
  if (!dense_on(table, c->device, at::kInt, 2) || !dense_on(lens, c->device, at::kInt, 1)) return false;
  const at::Tensor &t = THPVariable_Unpack(table), &l = THPVariable_Unpack(lens);
  if (t.size(0) != B || l.size(0) != B || t.size(1) < 1 || t.size(1) > INT32_MAX) return false;
  *out = pbs_paged_batch_t{};
  if (new_lens != Py_None) {
    if (!dense_on(new_lens, c->device, at::kInt, 1) || THPVariable_Unpack(new_lens).size(0) != B) return false;
    out->new_lens = static_cast<const int32_t*>(THPVariable_Unpack(new_lens).data_ptr());
  }
  out->block_table = static_cast<const int32_t*>(t.data_ptr());
  out->table_stride = t.stride(0);
  out->seq_lens = static_cast<const int32_t*>(l.data_ptr());
  out->max_pages = (int32_t)t.size(1);
  out->batch = (int32_t)B;
  out->new_tokens = (int32_t)S;
  return true;
}

// Memory for partial results, one piece a stream, or a stream of a capture: calls there come after one another.  A capture's comes from
// its graph's own pool and is cleared by the graph, once for all its calls.
// What one kind of call leaves behind in an error is nothing to the others: each has its own.
enum Kind { kAttention, kBeams };
struct Space {
  Kind kind;
  int device;
  cudaStream_t st;
  unsigned long long capture;                                      // 0: none
  at::Tensor memory;
};

constexpr int kMaxSpaces = 8;                                      // of a kind, so that one kind takes no other's

// In the order of their last use.  (Never destroyed: the interpreter ends after the allocator that they would go back to.)
std::vector<Space>& spaces() {
  static auto* s = new std::vector<Space>;
  return *s;
}

// The place of a stream's memory, which is what `memory` is undefined for where there is none yet.  What makes room are the captures before
// this one, whose graphs no longer ask (what they hold would keep those graphs' pools), then what was used longest ago.
at::Tensor& space_of(Kind kind, int device, cudaStream_t st, unsigned long long capture) {
  std::vector<Space>& s = spaces();
  for (size_t i = s.size(); i-- > 0;) {
    if (s[i].kind != kind || s[i].device != device || s[i].st != st || s[i].capture != capture) continue;
    std::rotate(s.begin() + i, s.begin() + i + 1, s.end());
    return s.back().memory;
  }
  s.erase(std::remove_if(s.begin(), s.end(), [&](const Space& x) { return x.capture != 0 && x.capture != capture; }), s.end());
  const auto same = [&](const Space& x) { return x.kind == kind; };
  if (std::count_if(s.begin(), s.end(), same) >= kMaxSpaces) s.erase(std::find_if(s.begin(), s.end(), same));
  s.push_back(Space{kind, device, st, capture, at::Tensor()});
  return s.back().memory;
}

// New memory of `need` bytes, its counters 0.  An undefined tensor where that failed.
at::Tensor new_space(int64_t need, const at::TensorOptions& opt, cudaStream_t st) {
  at::Tensor t = at::empty({need}, opt.dtype(at::kByte));
  if (cudaMemsetAsync(t.data_ptr(), 0, PBS_PAGED_COUNTER_BYTES, st) != cudaSuccess) return at::Tensor();
  return t;
}

// paged_attn(cache, q, table, lens, new_lens, scale, out): the result, or None
PyObject* py_attn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) { PyErr_SetString(PyExc_TypeError, "paged_attn takes 7 arguments"); return nullptr; }
  Cache* c = get(a[0]);
  if (!c) return nullptr;
  if (!plain(a[1]) || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
  const at::Tensor& q = THPVariable_Unpack(a[1]);
  if (q.dim() != 4) Py_RETURN_NONE;
  pbs_paged_batch_t batch;
  if (!rows_of(c, a[1], q.size(0), -1, q.size(2)) || !batch_of(c, a[2], a[3], a[4], q.size(0), q.size(2), &batch)) Py_RETURN_NONE;
  double scale = 1.0 / std::sqrt((double)c->c->head_dim);
  if (a[5] != Py_None) {
    if (!PyFloat_CheckExact(a[5])) Py_RETURN_NONE;
    scale = PyFloat_AS_DOUBLE(a[5]);
  }
  if (a[6] != Py_None && !rows_of(c, a[6], q.size(0), q.size(1), q.size(2))) Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)c->device);
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)c->device).stream();
  cudaStreamCaptureStatus status;
  unsigned long long capture = 0;
  if (cudaStreamGetCaptureInfo(st, &status, &capture) != cudaSuccess || status == cudaStreamCaptureStatusInvalidated) Py_RETURN_NONE;
  if (status == cudaStreamCaptureStatusNone) capture = 0;
  at::Tensor out = a[6] == Py_None ? at::empty_like(q) : THPVariable_Unpack(a[6]);
  if (!readable(out, false)) Py_RETURN_NONE;
  at::Tensor& space = space_of(kAttention, c->device, st, capture);
  int rc = PBS_ERR_SHAPE;
  for (int round = 0; rc == PBS_ERR_SHAPE && round < 2; ++round) {
    if (round == 1 || !space.defined()) {                          // too small, perhaps
      int64_t need = 0;
      if (c->workspace(c->c, &batch, (int32_t)q.size(1), &need) != PBS_OK || (space.defined() && need <= space.numel())) Py_RETURN_NONE;
      space = new_space(need, at::TensorOptions().device(at::Device(at::kCUDA, (c10::DeviceIndex)c->device)), st);
      if (!space.defined()) Py_RETURN_NONE;
    }
    rc = c->attn(c->c, &batch, (int32_t)q.size(1), q.data_ptr(), q.strides().data(), out.data_ptr(), out.strides().data(), (float)scale,
                 space.data_ptr(), space.numel(), st);
  }
  if (rc != PBS_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// paged_append(cache, k, v, table, lens, new_lens, cos, sin, q, q_out): the rotated queries, True where there are none, or None
PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10) { PyErr_SetString(PyExc_TypeError, "paged_append takes 10 arguments"); return nullptr; }
  Cache* c = get(a[0]);
  if (!c) return nullptr;
  if (!plain(a[1]) || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
  const at::Tensor& k = THPVariable_Unpack(a[1]);
  if (k.dim() != 4) Py_RETURN_NONE;
  const int64_t B = k.size(0), S = k.size(2);
  pbs_paged_batch_t batch;
  if (!rows_of(c, a[1], B, c->c->kv_heads, S) || !rows_of(c, a[2], B, c->c->kv_heads, S) || !batch_of(c, a[3], a[4], a[5], B, S, &batch)) Py_RETURN_NONE;
  const at::Tensor& v = THPVariable_Unpack(a[2]);
  const void *cos = nullptr, *sin = nullptr;
  int64_t cs[3] = {0, 0, 1};
  int32_t rows = 0;
  if ((a[6] == Py_None) != (a[7] == Py_None)) Py_RETURN_NONE;
  if (a[6] != Py_None) {
    if (!plain(a[6]) || !plain(a[7])) Py_RETURN_NONE;
    const at::Tensor &ct = THPVariable_Unpack(a[6]), &stb = THPVariable_Unpack(a[7]);
    const int64_t dims = ct.dim();
    if ((dims != 2 && dims != 3) || !dense_on(a[6], c->device, c->type, dims) || !dense_on(a[7], c->device, c->type, dims)) Py_RETURN_NONE;
    if (ct.sizes() != stb.sizes() || ct.strides() != stb.strides() || ct.size(dims - 1) != c->c->head_dim) Py_RETURN_NONE;
    cos = ct.data_ptr();
    sin = stb.data_ptr();
    cs[1] = ct.stride(dims - 2);
    if (dims == 2) {
      if (ct.size(0) < 1 || ct.size(0) > INT32_MAX) Py_RETURN_NONE;
      rows = (int32_t)ct.size(0);
    } else {
      if (ct.size(1) != S || (ct.size(0) != 1 && ct.size(0) != B)) Py_RETURN_NONE;
      cs[0] = ct.size(0) > 1 ? ct.stride(0) : 0;
    }
  }
  if (a[8] != Py_None && (!cos || !rows_of(c, a[8], B, -1, S))) Py_RETURN_NONE;
  if (a[9] != Py_None && (a[8] == Py_None || !rows_of(c, a[9], B, THPVariable_Unpack(a[8]).size(1), S))) Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)c->device);
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)c->device).stream();
  at::Tensor out;
  const at::Tensor* q = nullptr;
  if (a[8] != Py_None) {
    q = &THPVariable_Unpack(a[8]);
    out = a[9] == Py_None ? at::empty_like(*q) : THPVariable_Unpack(a[9]);
    if (!readable(out, false)) Py_RETURN_NONE;
  }
  const int rc = c->append(c->c, &batch, k.data_ptr(), k.strides().data(), v.data_ptr(), v.strides().data(), q ? (int32_t)q->size(1) : 0,
                           q ? q->data_ptr() : nullptr, q ? q->strides().data() : nullptr, q ? out.data_ptr() : nullptr,
                           q ? out.strides().data() : nullptr, cos, sin, cs, rows, st);
  if (rc != PBS_OK) Py_RETURN_NONE;
  if (!q) Py_RETURN_TRUE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// paged_gather(cache, table, lens, count, new_lens): (keys, values), or None
PyObject* py_gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) { PyErr_SetString(PyExc_TypeError, "paged_gather takes 5 arguments"); return nullptr; }
  Cache* c = get(a[0]);
  if (!c) return nullptr;
  if (!PyLong_CheckExact(a[3]) || !dense_on(a[2], c->device, at::kInt, 1) || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
  int over = 0;
  const int64_t S = PyLong_AsLongLongAndOverflow(a[3], &over), B = THPVariable_Unpack(a[2]).size(0), H = c->c->kv_heads, D = c->c->head_dim;
  pbs_paged_batch_t batch;
  if (over || !batch_of(c, a[1], a[2], a[4], B, S, &batch)) Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)c->device);
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)c->device).stream();
  const int64_t sizes[4] = {B, H, S, D}, strides[4] = {S * H * D, D, H * D, 1};
  const auto opt = at::TensorOptions().dtype(c->type).device(at::Device(at::kCUDA, (c10::DeviceIndex)c->device));
  at::Tensor k = at::empty_strided(at::IntArrayRef(sizes, 4), at::IntArrayRef(strides, 4), opt);
  at::Tensor v = at::empty_strided(at::IntArrayRef(sizes, 4), at::IntArrayRef(strides, 4), opt);
  if (c->gather(c->c, &batch, k.data_ptr(), strides, v.data_ptr(), strides, st) != PBS_OK) Py_RETURN_NONE;
  THPObjectPtr first(THPVariable_Wrap(std::move(k))), second(THPVariable_Wrap(std::move(v)));
  if (!first || !second) return nullptr;
  return PyTuple_Pack(2, first.get(), second.get());
  END_HANDLE_TH_ERRORS
}

// A penalty: nothing, a number, or (B,) float32.
bool penalty(PyObject* o, int device, int64_t B, float* all, const float** rows) {
  if (o == Py_None) return true;
  if (PyFloat_CheckExact(o)) {
    *all = (float)PyFloat_AS_DOUBLE(o);
    return true;
  }
  if (!dense_on(o, device, at::kFloat, 1) || THPVariable_Unpack(o).size(0) != B) return false;
  *rows = static_cast<const float*>(THPVariable_Unpack(o).data_ptr());
  return true;
}

// Ids of rows of B, int32 or int64; false where they are neither.
bool ids_of(PyObject* o, int device, int64_t B, const void** p, int64_t* stride, int32_t* per_row, int32_t* bytes) {
  if (o == Py_None) return true;
  const bool wide = dense_on(o, device, at::kLong, 2);
  if (!wide && !dense_on(o, device, at::kInt, 2)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.size(0) != B || t.size(1) >= (1 << 30)) return false;
  *p = t.data_ptr();
  *stride = t.stride(0);
  *per_row = (int32_t)t.size(1);
  *bytes = wide ? 8 : 4;
  return true;
}

// process_logits(function, logits, tokens, token_lens, prompt_lens, repetition, frequency, presence, bias_ids, bias_values, allowed, out): the result, or None
PyObject* py_logits(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12) { PyErr_SetString(PyExc_TypeError, "process_logits takes 12 arguments"); return nullptr; }
  const auto fn = reinterpret_cast<decltype(&pbs_process_logits)>(PyLong_AsUnsignedLongLong(a[0]));
  if (!fn) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no function"); return nullptr; }
  if (!plain(a[1]) || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
  const at::Tensor& x = THPVariable_Unpack(a[1]);
  const auto type = x.scalar_type();
  if (!x.is_cuda() || (type != at::kBFloat16 && type != at::kHalf && type != at::kFloat) || !dense_on(a[1], x.device().index(), type, 2)) Py_RETURN_NONE;
  const int device = x.device().index();
  const int64_t B = x.size(0), V = x.size(1);
  if (B < 1 || V < 1 || B > 65535 || V > (1 << 30)) Py_RETURN_NONE;
  pbs_logits_t g = {};
  g.dtype = type == at::kBFloat16 ? PBS_BF16 : type == at::kHalf ? PBS_FP16 : PBS_FP32;
  g.rows = (int32_t)B;
  g.vocab = (int32_t)V;
  g.repetition_all = 1.f;
  if (!ids_of(a[2], device, B, &g.tokens, &g.tokens_stride, &g.history, &g.token_bytes)) Py_RETURN_NONE;
  for (int i = 3; i <= 4; ++i) {
    if (a[i] == Py_None) continue;
    if (!dense_on(a[i], device, at::kInt, 1) || THPVariable_Unpack(a[i]).size(0) != B) Py_RETURN_NONE;
    (i == 3 ? g.token_lens : g.prompt_lens) = static_cast<const int32_t*>(THPVariable_Unpack(a[i]).data_ptr());
  }
  if (!penalty(a[5], device, B, &g.repetition_all, &g.repetition) || !penalty(a[6], device, B, &g.frequency_all, &g.frequency) ||
      !penalty(a[7], device, B, &g.presence_all, &g.presence))
    Py_RETURN_NONE;
  if (!(g.repetition_all > 0.f) || (a[2] == Py_None && (a[5] != Py_None || a[6] != Py_None || a[7] != Py_None))) Py_RETURN_NONE;
  if ((a[8] == Py_None) != (a[9] == Py_None) || !ids_of(a[8], device, B, &g.bias_ids, &g.bias_ids_stride, &g.biases, &g.bias_id_bytes)) Py_RETURN_NONE;
  if (a[9] != Py_None) {
    if (!dense_on(a[9], device, at::kFloat, 2)) Py_RETURN_NONE;
    const at::Tensor& b = THPVariable_Unpack(a[9]);
    if (b.size(0) != B || b.size(1) != g.biases) Py_RETURN_NONE;
    g.bias_values = static_cast<const float*>(b.data_ptr());
    g.bias_values_stride = b.stride(0);
  }
  if (a[10] != Py_None) {
    if (!dense_on(a[10], device, at::kInt, 2)) Py_RETURN_NONE;
    const at::Tensor& m = THPVariable_Unpack(a[10]);
    if ((m.size(0) != B && m.size(0) != 1) || m.size(1) != (V + 31) / 32) Py_RETURN_NONE;
    g.allowed = static_cast<const uint32_t*>(m.data_ptr());
    g.allowed_stride = m.size(0) > 1 ? m.stride(0) : 0;
  }
  if (a[11] != Py_None) {
    if (!dense_on(a[11], device, type, 2) || THPVariable_Unpack(a[11]).sizes() != x.sizes()) Py_RETURN_NONE;
  }
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  at::Tensor out = a[11] == Py_None ? at::empty(x.sizes(), x.options()) : THPVariable_Unpack(a[11]);
  g.logits = x.data_ptr();
  g.out = out.data_ptr();
  g.logits_stride = x.stride(0);
  g.out_stride = out.stride(0);
  if (fn(&g, st) != PBS_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// paged_reorder(function, caches, table, lens, beams): True, or False where Python has to do it
PyObject* py_reorder(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5 || !PyList_CheckExact(a[1])) { PyErr_SetString(PyExc_TypeError, "paged_reorder takes 5 arguments, the second a list"); return nullptr; }
  const auto fn = reinterpret_cast<decltype(&pbs_paged_reorder)>(PyLong_AsUnsignedLongLong(a[0]));
  if (!fn) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no function"); return nullptr; }
  const Py_ssize_t layers = PyList_GET_SIZE(a[1]);
  std::vector<const pbs_paged_cache_t*> caches((size_t)layers);
  Cache* first = nullptr;
  for (Py_ssize_t i = 0; i < layers; ++i) {
    PyObject* o = PyList_GET_ITEM(a[1], i);
    if (!PyCapsule_IsValid(o, kName)) Py_RETURN_FALSE;
    Cache* c = get(o);
    if (!first) first = c;
    if (c->device != first->device) Py_RETURN_FALSE;
    caches[(size_t)i] = c->c;
  }
  if (!first || layers > INT32_MAX || !dense_on(a[3], first->device, at::kInt, 1) || !dense_on(a[4], first->device, at::kInt, 2) ||
      at::impl::torch_function_mode_enabled())
    Py_RETURN_FALSE;
  const at::Tensor& beams = THPVariable_Unpack(a[4]);
  const int64_t rows = THPVariable_Unpack(a[3]).size(0);
  pbs_paged_batch_t batch;
  if (!batch_of(first, a[2], a[3], Py_None, rows, 1, &batch) || beams.size(0) * beams.size(1) != rows) Py_RETURN_FALSE;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)first->device);
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)first->device).stream();
  if (fn(caches.data(), (int32_t)layers, &batch, const_cast<int32_t*>(batch.block_table), (int32_t)beams.size(1), static_cast<const int32_t*>(beams.data_ptr()),
         beams.stride(0), st) != PBS_OK)
    Py_RETURN_FALSE;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// beam_select(function, workspace_function, logits, scores, keep): (scores, beams, tokens), or None
PyObject* py_beams(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) { PyErr_SetString(PyExc_TypeError, "beam_select takes 5 arguments"); return nullptr; }
  const auto fn = reinterpret_cast<decltype(&pbs_beam_select)>(PyLong_AsUnsignedLongLong(a[0]));
  const auto ws = reinterpret_cast<decltype(&pbs_beam_select_workspace)>(PyLong_AsUnsignedLongLong(a[1]));
  if (!fn || !ws) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no function"); return nullptr; }
  if (!plain(a[2]) || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
  const at::Tensor& x = THPVariable_Unpack(a[2]);
  const auto type = x.scalar_type();
  if (!x.is_cuda() || (type != at::kBFloat16 && type != at::kHalf && type != at::kFloat)) Py_RETURN_NONE;
  const int device = x.device().index();
  if (!dense_on(a[2], device, type, 2) || !dense_on(a[3], device, at::kFloat, 2)) Py_RETURN_NONE;
  const at::Tensor& s = THPVariable_Unpack(a[3]);
  const int64_t B = s.size(0), N = s.size(1);
  int64_t keep = 2 * N;
  if (a[4] != Py_None) {
    int over = 0;
    if (!PyLong_CheckExact(a[4])) Py_RETURN_NONE;
    keep = PyLong_AsLongLongAndOverflow(a[4], &over);
    if (over) Py_RETURN_NONE;
  }
  if (B < 1 || N < 1 || B > 1024 || N > 32 || x.size(0) != B * N || x.size(1) < 1 || x.size(1) > (1 << 30) || keep < 1 || keep > 64) Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  cudaStreamCaptureStatus status;
  unsigned long long capture = 0;
  if (cudaStreamGetCaptureInfo(st, &status, &capture) != cudaSuccess || status == cudaStreamCaptureStatusInvalidated) Py_RETURN_NONE;
  if (status == cudaStreamCaptureStatusNone) capture = 0;
  const auto opt = at::TensorOptions().device(at::Device(at::kCUDA, (c10::DeviceIndex)device));
  at::Tensor scores = at::empty({B, keep}, opt.dtype(at::kFloat)), beams = at::empty({B, keep}, opt.dtype(at::kInt)), tokens = at::empty({B, keep}, opt.dtype(at::kLong));
  pbs_beam_select_t g = {};
  g.dtype = type == at::kBFloat16 ? PBS_BF16 : type == at::kHalf ? PBS_FP16 : PBS_FP32;
  g.batch = (int32_t)B;
  g.beams = (int32_t)N;
  g.vocab = (int32_t)x.size(1);
  g.keep = (int32_t)keep;
  g.logits = x.data_ptr();
  g.logits_stride = x.stride(0);
  g.scores = static_cast<const float*>(s.data_ptr());
  g.scores_stride = s.stride(0);
  g.out_scores = static_cast<float*>(scores.data_ptr());
  g.out_beams = static_cast<int32_t*>(beams.data_ptr());
  g.out_tokens = static_cast<int64_t*>(tokens.data_ptr());
  at::Tensor& space = space_of(kBeams, device, st, capture);
  int rc = PBS_ERR_SHAPE;
  for (int round = 0; rc == PBS_ERR_SHAPE && round < 2; ++round) {
    if (round == 1 || !space.defined()) {                          // too small, perhaps
      int64_t need = 0;
      if (ws(&g, &need) != PBS_OK || (space.defined() && need <= space.numel())) Py_RETURN_NONE;
      space = new_space(need, opt, st);
      if (!space.defined()) Py_RETURN_NONE;
    }
    rc = fn(&g, space.data_ptr(), space.numel(), st);
  }
  if (rc != PBS_OK) Py_RETURN_NONE;
  THPObjectPtr o0(THPVariable_Wrap(std::move(scores))), o1(THPVariable_Wrap(std::move(beams))), o2(THPVariable_Wrap(std::move(tokens)));
  if (!o0 || !o1 || !o2) return nullptr;
  return PyTuple_Pack(3, o0.get(), o1.get(), o2.get());
  END_HANDLE_TH_ERRORS
}

// paged_forget(): the next calls make new workspaces
PyObject* py_forget(PyObject*, PyObject*) {
  spaces().clear();
  Py_RETURN_NONE;
}

template <class F>
PyCFunction fast(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)); }

}  // namespace

PyMethodDef pbs_decode_methods[] = {
    {"paged_attach", py_attach, METH_VARARGS, "paged_attach(struct, device, append, gather, attn, workspace): addresses -> the cache's object here"},
    {"paged_forget", py_forget, METH_NOARGS, "paged_forget(): workspaces are made anew"},
    {"paged_append", fast(py_append), METH_FASTCALL, "paged_append(cache, k, v, table, lens, new_lens, cos, sin, q, q_out): the rotated queries, True, or None where Python has to do it"},
    {"paged_gather", fast(py_gather), METH_FASTCALL, "paged_gather(cache, table, lens, count, new_lens): (keys, values), or None where Python has to do it"},
    {"paged_attn", fast(py_attn), METH_FASTCALL, "paged_attn(cache, q, table, lens, new_lens, scale, out): the result, or None where Python has to do it"},
    {"paged_reorder", fast(py_reorder), METH_FASTCALL, "paged_reorder(function, caches, table, lens, beams): True, or False where Python has to do it"},
    {"beam_select", fast(py_beams), METH_FASTCALL, "beam_select(function, workspace_function, logits, scores, keep): (scores, beams, tokens), or None where Python has to do it"},
    {"process_logits", fast(py_logits), METH_FASTCALL, "process_logits(function, logits, ...): the result, or None where Python has to do it"},
    {nullptr, nullptr, 0, nullptr}};
