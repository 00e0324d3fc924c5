// The five entry points of flash_attn_2_cuda for the calls that need nothing but their outputs allocated: plain tensors whose
// shapes, types and alignment the kernels take as they are.  Each function returns None for any other call (dropout, padding,
// copies, given outputs, every error): flash_attn_2_cuda/__init__.py does those, with the same C ABI underneath.
//
// Why native: filling the argument struct and checking the operands took 26 us (forward) and 47 us (backward) of interpreter
// time per call, next to kernels of 10 to 30 us for a short prompt, a small training step or a decode step.
//
// Behind them the calls for drafted trees, positions with several axes and paged caches, which have no other host code: they check all that they
// are given and raise RuntimeError.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <initializer_list>
#include <limits>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "fa_b200.h"

namespace {

using at::Tensor;
using MaybeTensor = std::optional<Tensor>;

// An ordinary dense CUDA tensor on device `dev` (no subclass, no tracing or functorch wrapper)
bool ordinary(const Tensor& t, c10::Device dev) {
  return t.defined() && t.is_cuda() && t.device() == dev && t.layout() == at::kStrided &&
         !t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchGradWrapper,
                                                   c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::Functionalize}));
}

bool has_shape(const Tensor& t, std::initializer_list<int64_t> shape) { return t.sizes() == c10::IntArrayRef(shape); }

// What the kernels take without a copy: 16-byte pieces everywhere, and no dim that repeats its elements
bool direct(const Tensor& t, bool may_repeat = false) {
  if (t.stride(-1) != 1 || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15)) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.stride(i) % 8 || (t.stride(i) == 0 && !may_repeat)) return false;
  return true;
}

FaTensor view(const Tensor& t) {  // (batch, seq, head, dim), or packed (total, head, dim)
  if (t.dim() == 3) return FaTensor{t.data_ptr(), 0, t.stride(0), t.stride(1)};
  return FaTensor{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

bool takes(const Tensor& q) {
  if (!q.defined() || !q.is_cuda()) return false;
  if (q.scalar_type() != at::kHalf && q.scalar_type() != at::kBFloat16) return false;
  return q.device().index() == c10::cuda::current_device() && ordinary(q, q.device());
}

int32_t code(const Tensor& q) { return q.scalar_type() == at::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_FP16; }

// csrc/flash_attn/flash_api.cpp:113-114, 297: a window open on one side gets seqlen_k there
void windows(bool causal, int64_t seqlen_k, int64_t& wl, int64_t& wr) {
  if (causal) wr = 0;
  if (wl < 0 && wr >= 0) wl = seqlen_k;
  if (wl >= 0 && wr < 0) wr = seqlen_k;
}

bool fits(std::initializer_list<int64_t> values) {
  for (int64_t v : values)
    if (v < std::numeric_limits<int32_t>::min() || v > std::numeric_limits<int32_t>::max()) return false;
  return true;
}

int sm_count(c10::Device) { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

fa_stream_t stream_of(const Tensor& q) { return reinterpret_cast<fa_stream_t>(at::cuda::getCurrentCUDAStream(q.device().index()).stream()); }

void check(int status, const char* what) {
  if (status) throw std::runtime_error(std::string(what) + ": " + fa_last_error());
}

bool int32_vector(const Tensor& t, c10::Device dev, int64_t n) {
  return ordinary(t, dev) && t.scalar_type() == at::kInt && t.dim() == 1 && t.numel() == n && t.is_contiguous();
}

// fwd / varlen_fwd: [out, q, k, v, out, softmax_lse, None, rng_state]
// varlen: which of the two was called; packed operands without their offsets are an error, not a padded batch
py::object fwd(bool varlen, const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& cu_q, const MaybeTensor& cu_k, int64_t max_q,
               int64_t max_k, double scale, bool causal, int64_t wl, int64_t wr) {
  if (cu_q.has_value() != varlen || cu_k.has_value() != varlen) return py::none();
  if (!takes(q) || q.dim() != (varlen ? 3 : 4) || getenv("FA_B200_FWD_SPLITS")) return py::none();
  const c10::Device dev = q.device();
  for (const Tensor* t : {&k, &v})
    if (!ordinary(*t, dev) || t->scalar_type() != q.scalar_type() || t->dim() != q.dim()) return py::none();
  const int64_t heads = q.size(-2), heads_k = k.size(-2), d = q.size(-1);
  int64_t batch, sq, sk, total_q = 0, total_k = 0;
  if (varlen) {
    total_q = q.size(0), total_k = k.size(0);
    batch = cu_q->numel() - 1, sq = max_q, sk = max_k;
    if (!int32_vector(*cu_q, dev, batch + 1) || !int32_vector(*cu_k, dev, batch + 1) || total_q <= 0 || total_k <= 0) return py::none();
    if (!has_shape(k, {total_k, heads_k, d}) || !has_shape(v, {total_k, heads_k, d})) return py::none();
  } else {
    batch = q.size(0), sq = q.size(1), sk = k.size(1);
    if (!has_shape(k, {batch, sk, heads_k, d}) || !has_shape(v, {batch, sk, heads_k, d})) return py::none();
    if (sq == 1) return py::none();  // (may change places with the heads of a group)
  }
  if (batch <= 0 || sq <= 0 || sk <= 0 || d <= 0 || d > 256 || d % 8 || heads_k <= 0 || heads <= 0 || heads % heads_k) return py::none();
  if (!direct(q) || !direct(k) || !direct(v)) return py::none();
  windows(causal, sk, wl, wr);
  if (!fits({batch, sq, sk, heads, wl, wr, total_q, total_k, heads / heads_k * sq})) return py::none();

  const auto f32 = q.options().dtype(at::kFloat).requires_grad(false);
  Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
  Tensor lse = at::empty({batch, heads, sq}, f32);
  Tensor rng = at::empty({2}, f32.dtype(at::kLong));
  FaFwdArgs a = {};
  a.q = view(q), a.k = view(k), a.v = view(v), a.out = view(out);
  a.softmax_lse = static_cast<float*>(lse.data_ptr());
  a.lse_seqlen = a.seqlen_q = sq;
  a.batch = batch, a.seqlen_k = sk, a.heads = heads, a.heads_k = heads_k, a.head_dim = d;
  a.dtype = code(q), a.softmax_scale = scale;
  a.window_left = wl, a.window_right = wr;
  a.num_splits = 1;
  Tensor lse_acc, out_acc;
  if (varlen) {
    a.cu_seqlens_q = static_cast<int32_t*>(cu_q->data_ptr()), a.cu_seqlens_k = static_cast<int32_t*>(cu_k->data_ptr());
    a.total_q = total_q, a.total_k = total_k;
  } else {
    // the heads of a group share the kernel's 128-row tiles
    const int n = fa_fwd_num_splits(batch, heads_k, sq * (heads / heads_k), sk, d, sm_count(dev));
    if (n > 1) {
      lse_acc = at::empty({n, batch, heads, sq}, f32);
      out_acc = at::empty({n, batch, heads, sq, d}, f32);
      a.num_splits = n, a.lse_accum = static_cast<float*>(lse_acc.data_ptr()), a.out_accum = static_cast<float*>(out_acc.data_ptr());
    }
  }
  int status;
  {
    const fa_stream_t st = stream_of(q);
    py::gil_scoped_release unlocked;
    status = fa_fwd(&a, st);
  }
  check(status, varlen ? "flash_attn_2_cuda.varlen_fwd" : "flash_attn_2_cuda.fwd");
  py::list r(8);
  r[0] = out, r[1] = q, r[2] = k, r[3] = v, r[4] = out, r[5] = lse, r[6] = py::none(), r[7] = rng;
  return r;
}

// bwd / varlen_bwd: [dq, dk, dv, softmax_d]
py::object bwd(bool varlen, const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& lse,
               const MaybeTensor& dq_, const MaybeTensor& dk_, const MaybeTensor& dv_, const MaybeTensor& cu_q, const MaybeTensor& cu_k,
               int64_t max_q, int64_t max_k, double scale, bool causal, int64_t wl, int64_t wr, bool deterministic) {
  if (cu_q.has_value() != varlen || cu_k.has_value() != varlen) return py::none();
  if (!takes(q) || q.dim() != (varlen ? 3 : 4) || !dq_ || !dk_ || !dv_) return py::none();
  const c10::Device dev = q.device();
  const Tensor &dq = *dq_, &dk = *dk_, &dv = *dv_;
  for (const Tensor* t : {&dout, &k, &v, &out, &dq, &dk, &dv})
    if (!ordinary(*t, dev) || t->scalar_type() != q.scalar_type() || t->dim() != q.dim()) return py::none();
  const int64_t heads = q.size(-2), heads_k = k.size(-2), d = q.size(-1);
  int64_t batch, sq, sk, total_q = 0, total_k = 0;
  if (varlen) {
    total_q = q.size(0), total_k = k.size(0);
    batch = cu_q->numel() - 1, sq = max_q, sk = max_k;
    if (!int32_vector(*cu_q, dev, batch + 1) || !int32_vector(*cu_k, dev, batch + 1) || total_q <= 0 || total_k <= 0) return py::none();
    if (!has_shape(k, {total_k, heads_k, d})) return py::none();
  } else {
    batch = q.size(0), sq = q.size(1), sk = k.size(1);
    if (!has_shape(k, {batch, sk, heads_k, d})) return py::none();
  }
  if (v.sizes() != k.sizes() || dk.sizes() != k.sizes() || dv.sizes() != k.sizes() || dout.sizes() != q.sizes() || out.sizes() != q.sizes() ||
      dq.sizes() != q.sizes())
    return py::none();
  if (batch <= 0 || sq <= 0 || sk <= 0 || d <= 0 || d > 256 || d % 8 || heads_k <= 0 || heads <= 0 || heads % heads_k) return py::none();
  for (const Tensor* t : {&dout, &q, &k, &v, &out, &dq, &dk, &dv})
    if (!direct(*t)) return py::none();
  if (!ordinary(lse, dev) || lse.scalar_type() != at::kFloat || lse.dim() != 3) return py::none();
  windows(causal, sk, wl, wr);
  const int64_t d_seqlen = (sq + 127) / 128 * 128;
  if (!fits({batch, d_seqlen, sk, heads, wl, wr, total_q, total_k, lse.size(-1)})) return py::none();

  const auto f32 = q.options().dtype(at::kFloat).requires_grad(false);
  Tensor softmax_d = at::empty({batch, heads, d_seqlen}, f32);
  Tensor dq_accum = at::empty({fa_bwd_workspace_bytes(batch, sq, heads, d, total_q, varlen) / 4}, f32);
  FaBwdArgs a = {};
  a.q = view(q), a.k = view(k), a.v = view(v), a.out = view(out), a.dout = view(dout);
  a.dq = view(dq), a.dk = view(dk), a.dv = view(dv);
  a.softmax_lse = static_cast<float*>(lse.data_ptr()), a.lse_seqlen = lse.size(-1);
  a.softmax_d = static_cast<float*>(softmax_d.data_ptr()), a.d_seqlen = d_seqlen;
  a.dq_accum = static_cast<float*>(dq_accum.data_ptr());
  a.batch = batch, a.seqlen_q = sq, a.seqlen_k = sk, a.heads = heads, a.heads_k = heads_k, a.head_dim = d;
  a.dtype = code(q), a.softmax_scale = scale;
  a.window_left = wl, a.window_right = wr;
  if (varlen) {
    a.cu_seqlens_q = static_cast<int32_t*>(cu_q->data_ptr()), a.cu_seqlens_k = static_cast<int32_t*>(cu_k->data_ptr());
    a.total_q = total_q, a.total_k = total_k;
  }
  a.deterministic = deterministic;
  int status;
  {
    const fa_stream_t st = stream_of(q);
    py::gil_scoped_release unlocked;
    status = fa_bwd(&a, st);
  }
  check(status, varlen ? "flash_attn_2_cuda.varlen_bwd" : "flash_attn_2_cuda.bwd");
  py::list r(4);
  r[0] = dq, r[1] = dk, r[2] = dv, r[3] = softmax_d;
  return r;
}

// fwd_kvcache: [out, softmax_lse]
py::object fwd_kvcache(const Tensor& q_in, const Tensor& kc, const Tensor& vc, const MaybeTensor& k, const MaybeTensor& v,
                       const MaybeTensor& lens, const MaybeTensor& cos, const MaybeTensor& sin, const MaybeTensor& batch_idx, double scale,
                       bool causal, int64_t wl, int64_t wr, bool interleaved, int64_t num_splits, const MaybeTensor& table) {
  if (!takes(q_in) || q_in.dim() != 4) return py::none();
  const c10::Device dev = q_in.device();
  const auto dtype = q_in.scalar_type();
  for (const Tensor* t : {&kc, &vc})
    if (!ordinary(*t, dev) || t->scalar_type() != dtype || t->dim() != 4 || !direct(*t, /*may_repeat=*/true)) return py::none();
  Tensor q = q_in;
  const int64_t batch = q.size(0), batch_c = kc.size(0), heads_k = kc.size(2), d = q.size(3);
  int64_t sq = q.size(1), heads = q.size(2), cap = kc.size(1), page = 0;
  if (vc.sizes() != kc.sizes() || kc.size(3) != d) return py::none();
  if (batch <= 0 || batch_c <= 0 || sq <= 0 || cap <= 0 || d <= 0 || d > 256 || d % 8 || heads_k <= 0 || heads <= 0 || heads % heads_k) return py::none();
  if (table) {
    if (!ordinary(*table, dev) || table->scalar_type() != at::kInt || table->dim() != 2 || table->size(0) != batch || table->stride(1) != 1 ||
        batch_idx || cap % 64)
      return py::none();
    page = cap;
    cap = table->size(1) * page;
    if (cap <= 0) return py::none();
  } else if (!batch_idx && batch_c < batch) {
    return py::none();
  }
  if (sq == 1) causal = false;
  windows(causal, cap, wl, wr);
  if (!direct(q)) return py::none();
  // one token: the heads of a group are the rows of a call (csrc/flash_attn/flash_api.cpp:299-307)
  const bool swapped = sq == 1 && heads > heads_k && wl < 0 && wr < 0;
  if (swapped) {
    if (!q.is_contiguous()) return py::none();
    sq = heads / heads_k, heads = heads_k;
    q = q.view({batch, heads, sq, d}).transpose(1, 2);
  }
  FaKvcacheArgs a = {};
  int64_t sn = 0;
  if (k) {
    if (!v || !lens || (sq > cap && !swapped)) return py::none();
    sn = k->size(1);
    for (const Tensor* t : {&*k, &*v})
      if (!ordinary(*t, dev) || t->scalar_type() != dtype || !has_shape(*t, {batch, sn, heads_k, d}) || !direct(*t, true)) return py::none();
    a.knew = view(*k), a.vnew = view(*v);
  }
  if (lens) {
    if (!int32_vector(*lens, dev, batch)) return py::none();
    a.cache_seqlens = static_cast<int32_t*>(lens->data_ptr());
  }
  if (batch_idx) {
    if (!int32_vector(*batch_idx, dev, batch)) return py::none();
    a.cache_batch_idx = static_cast<int32_t*>(batch_idx->data_ptr());
  }
  if (cos) {
    if (!k || !sin || cos->dim() != 2 || sin->sizes() != cos->sizes()) return py::none();
    for (const Tensor* t : {&*cos, &*sin})
      if (!ordinary(*t, dev) || t->scalar_type() != dtype || !t->is_contiguous()) return py::none();
    a.rotary_dim = cos->size(1) * 2, a.seqlen_ro = cos->size(0), a.rotary_interleaved = interleaved;
    if (a.rotary_dim <= 0 || a.rotary_dim > d || a.rotary_dim % 16 || cos->size(0) < cap) return py::none();
    a.rotary_cos = cos->data_ptr(), a.rotary_sin = sin->data_ptr();
  }
  if (num_splits < 0 || num_splits > 128 || !fits({batch, batch_c, cap, sq, heads, sn, wl, wr})) return py::none();

  const auto f32 = q.options().dtype(at::kFloat).requires_grad(false);
  const auto same = q.options().requires_grad(false);
  // (swapped: laid out as the caller sees it, so that no copy follows)
  Tensor out = swapped ? at::empty({batch, heads, sq, d}, same).transpose(1, 2) : at::empty({batch, sq, heads, d}, same);
  Tensor lse = at::empty({batch, heads, sq}, f32);
  a.q = view(q), a.kcache = view(kc), a.vcache = view(vc), a.out = view(out);
  a.softmax_lse = static_cast<float*>(lse.data_ptr());
  a.batch = batch, a.batch_cache = batch_c, a.seqlen_q = sq, a.seqlen_cache = cap, a.seqlen_new = sn;
  a.heads = heads, a.heads_k = heads_k, a.head_dim = d;
  a.dtype = code(q), a.softmax_scale = scale;
  a.window_left = wl, a.window_right = wr;
  a.q_rows_share_position = swapped;
  a.num_splits = num_splits;
  if (table) a.block_table = static_cast<int32_t*>(table->data_ptr()), a.block_table_stride = table->stride(0), a.page_block_size = page;
  int64_t lse_bytes = 0, out_bytes = 0;
  const int n = fa_kvcache_plan(&a, sm_count(dev), &lse_bytes, &out_bytes);
  if (n < 0) check(1, "flash_attn_2_cuda.fwd_kvcache");
  a.num_splits = n;  // what the workspaces are sized for
  Tensor lse_acc, out_acc, q_rot;
  if (n > 1) {
    lse_acc = at::empty({lse_bytes / 4}, f32);
    out_acc = at::empty({out_bytes / 4}, f32);
    a.lse_accum = static_cast<float*>(lse_acc.data_ptr()), a.out_accum = static_cast<float*>(out_acc.data_ptr());
  }
  if (cos) {
    q_rot = at::empty({batch, sq, heads, d}, same);
    a.q_rotated = q_rot.data_ptr();
  }
  int status;
  {
    const fa_stream_t st = stream_of(q);
    py::gil_scoped_release unlocked;
    status = fa_fwd_kvcache(&a, st);
  }
  check(status, "flash_attn_2_cuda.fwd_kvcache");
  if (swapped) {
    out = out.transpose(1, 2).view({batch, 1, heads * sq, d});
    lse = lse.view({batch, heads * sq, 1});
  }
  py::list r(2);
  r[0] = out, r[1] = lse;
  return r;
}

// ------------------------------------------------------------------------------------------------
// Trees of drafted tokens, positions with several axes, paged caches.  Shapes and types are checked before devices.
// (texts alone: a message is put together only where it is thrown)
void require(bool fine, const char* what, const char* more = "") {
  if (!fine) throw std::runtime_error(std::string(what) + more);
}

bool is_type(const Tensor& t, at::ScalarType type, int64_t dims) { return t.defined() && t.scalar_type() == type && t.dim() == dims; }

void require_rows(const Tensor& t, const char* name, int64_t dims, at::ScalarType like) {
  require(t.defined() && t.dim() == dims, name, dims == 4 ? " must have 4 dimensions" : " has the wrong number of dimensions");
  require(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, name, ": only fp16 and bf16 data type");
  require(t.scalar_type() == like, name, " must have the same dtype as query");
}

// all on the device of the first
void require_device(std::initializer_list<const Tensor*> ts) {
  const Tensor* first = nullptr;
  for (const Tensor* t : ts) {
    if (!t || !t->defined()) continue;
    if (!first) first = t;
    require(t->is_cuda(), "Input tensor must be on CUDA device");
    require(t->device() == first->device() && ordinary(*t, first->device()), "all tensors must be ordinary tensors on the same device");
  }
}

// Two tensors of which a call writes one must not start at the same place (one given twice)
void require_two(const Tensor& x, const Tensor& y, const char* what) {
  require(x.numel() == 0 || y.numel() == 0 || x.data_ptr() != y.data_ptr(), what, ": the same tensor is given twice");
}

// The calls have no forward-mode derivative: a tangent is refused, not lost
void require_no_tangent(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts) require(!t || !t->_fw_grad(0).defined(), "forward-mode derivatives are not supported");
}

// Written in place: autograd then refuses to use a value that it saved before
void changed(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();  // (inference tensors have no version, and are never saved)
}
void refuse_gradients_in_place(std::initializer_list<const Tensor*> ts, const char* what) {
  for (const Tensor* t : ts) require(!t || !at::GradMode::is_enabled() || !t->requires_grad(), what, ": in place only where no gradient is needed");
}

// at::empty without the way through the dispatcher (a call has two to four results)
Tensor fresh(c10::IntArrayRef sizes, at::ScalarType type, c10::Device dev) {
  return Tensor(at::detail::empty_cuda(sizes, type, dev, std::nullopt));
}

// Several whole-number results in one allocation, each on a 16-byte boundary
struct Carved {
  Tensor bytes;
  int64_t used = 0;
  Carved(std::initializer_list<int64_t> sizes, c10::Device dev) {
    int64_t n = 0;
    for (int64_t s : sizes) n += (s + 15) / 16 * 16;
    bytes = fresh({n}, at::kByte, dev);
  }
  Tensor take(c10::IntArrayRef sizes, at::ScalarType type) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(bytes.storage()), bytes.key_set(), c10::scalarTypeToTypeMeta(type));
    const int64_t size = c10::elementSize(type);
    t.unsafeGetTensorImpl()->set_storage_offset(used / size);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    used += (c10::multiply_integers(sizes) * size + 15) / 16 * 16;
    return t;
  }
};

// a copy in rows next to each other, on a 16-byte boundary
Tensor packed(const Tensor& t) { return t.is_contiguous() ? t.clone(at::MemoryFormat::Contiguous) : t.contiguous(); }

const Tensor* maybe(const MaybeTensor& t) { return t ? &*t : nullptr; }
int32_t* i32(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }

int32_t to_i32(int64_t v, const char* what) {
  require(v >= 0 && v <= std::numeric_limits<int32_t>::max(), what, " is out of range");
  return static_cast<int32_t>(v);
}

// tree_fwd: (out, softmax_lse)
py::tuple tree_fwd(const Tensor& q_in, const Tensor& kc, const Tensor& vc, const Tensor& mask, const Tensor& lens, const MaybeTensor& k_in,
                   const MaybeTensor& v_in, const MaybeTensor& table, const MaybeTensor& batch_idx, std::optional<double> scale, int64_t num_splits) {
  require_rows(q_in, "q", 4, q_in.scalar_type());
  require_rows(kc, "k_cache", 4, q_in.scalar_type());
  require_rows(vc, "v_cache", 4, q_in.scalar_type());
  const int64_t batch = q_in.size(0), nodes = q_in.size(1), heads = q_in.size(2), d = q_in.size(3), batch_c = kc.size(0), heads_k = kc.size(2);
  require(vc.sizes() == kc.sizes(), "k_cache and v_cache must have the same shape");
  require(kc.size(3) == d, "k_cache must have the head dimension of q");
  require(batch > 0 && nodes > 0 && batch_c > 0, "batch size, nodes and the KV cache must not be empty");
  require(d > 0 && d <= 256 && d % 8 == 0, "head dimension must be a multiple of 8, at most 256");
  require(heads_k > 0 && heads > 0 && heads % heads_k == 0, "Number of heads in key/value must divide number of heads in query");
  require(is_type(mask, at::kInt, 3) && mask.size(1) == nodes && mask.size(2) == (nodes + 31) / 32 && (mask.size(0) == batch || mask.size(0) == 1) &&
              (mask.size(2) == 1 || mask.stride(2) == 1),
          "the tree mask must be int32 words of shape (batch or 1, nodes, ceil(nodes / 32)) with contiguous last dimension");
  require(is_type(lens, at::kInt, 1) && lens.size(0) == batch && lens.is_contiguous(), "cache_seqlens must be int32, contiguous, one per sequence");
  int64_t cap = kc.size(1), page = 0;
  if (table) {
    require(!batch_idx, "Paged KVcache does not support cache_batch_idx");
    require(is_type(*table, at::kInt, 2) && table->size(0) == batch && (table->size(1) <= 1 || table->stride(1) == 1),
            "block_table must be int32 of shape (batch, pages per sequence) with contiguous last dimension");
    require(cap % 64 == 0 && cap > 0, "Paged KV cache block size must be divisible by 64");
    page = cap;
    cap = table->size(1) * page;
  } else if (batch_idx) {
    require(is_type(*batch_idx, at::kInt, 1) && batch_idx->size(0) == batch && batch_idx->is_contiguous(),
            "cache_batch_idx must be int32, contiguous, one per sequence");
  } else {
    require(batch_c >= batch, "the KV cache must hold at least `batch` sequences when cache_batch_idx is not given");
  }
  require(cap > 0, "the KV cache has no rows");
  require(k_in.has_value() == v_in.has_value(), "key and value must be given together");
  if (k_in) {
    require_rows(*k_in, "k", 4, q_in.scalar_type());
    require_rows(*v_in, "v", 4, q_in.scalar_type());
    require(has_shape(*k_in, {batch, nodes, heads_k, d}) && has_shape(*v_in, {batch, nodes, heads_k, d}),
            "k and v must have shape (batch, nodes, nheads_k, headdim)");
    require(nodes <= cap, "the tree has more nodes than the KV cache has rows");
    require_two(kc, vc, "k_cache and v_cache");
  }
  require(num_splits >= 0 && num_splits <= 128, "num_splits must be in [0, 128]");
  require(fits({batch, batch_c, cap, nodes, heads, heads / heads_k * nodes, batch * heads * nodes}), "sizes are out of range");
  require_no_tangent({&q_in, &kc, &vc, maybe(k_in), maybe(v_in)});
  require_device({&q_in, &kc, &vc, &mask, &lens, maybe(k_in), maybe(v_in), maybe(table), maybe(batch_idx)});
  require(direct(kc, true) && direct(vc, true), "k_cache / v_cache must be 16-byte aligned, with contiguous last dimension and strides that are multiples of 8");
  if (k_in)  // (what is written must not be one element in several places)
    require(direct(kc) && direct(vc), "tokens cannot be stored in a KV cache that repeats its elements");

  const c10::cuda::CUDAGuard guard(q_in.device());
  const Tensor q = direct(q_in) ? q_in : packed(q_in);
  Tensor k, v;
  Tensor out = fresh({batch, nodes, heads, d}, q.scalar_type(), q.device()), lse = fresh({batch, heads, nodes}, at::kFloat, q.device());
  FaTreeArgs t = {};
  FaKvcacheArgs& a = t.kv;
  if (k_in) {
    k = direct(*k_in, true) ? *k_in : packed(*k_in);
    v = direct(*v_in, true) ? *v_in : packed(*v_in);
    a.knew = view(k), a.vnew = view(v), a.seqlen_new = nodes;
  }
  a.q = view(q), a.kcache = view(kc), a.vcache = view(vc), a.out = view(out);
  a.softmax_lse = static_cast<float*>(lse.data_ptr());
  a.batch = batch, a.batch_cache = batch_c, a.seqlen_q = nodes, a.seqlen_cache = cap, a.heads = heads, a.heads_k = heads_k, a.head_dim = d;
  a.dtype = code(q), a.softmax_scale = scale ? *scale : 1.0 / std::sqrt((double)d);
  a.window_left = a.window_right = -1;
  a.cache_seqlens = i32(lens);
  if (batch_idx) a.cache_batch_idx = i32(*batch_idx);
  if (table) a.block_table = i32(*table), a.block_table_stride = to_i32(table->stride(0), "stride of block_table"), a.page_block_size = page;
  a.num_splits = num_splits;
  t.mask = i32(mask), t.mask_stride_b = mask.size(0) == 1 ? 0 : mask.stride(0), t.mask_stride_s = mask.stride(1);
  int64_t lse_bytes = 0, out_bytes = 0;
  const int n = fa_tree_plan(&t, sm_count(q.device()), &lse_bytes, &out_bytes);
  if (n < 0) check(1, "flash_attn_tree_with_kvcache");
  a.num_splits = n;  // what the workspaces are sized for
  Tensor workspace;
  if (n > 1) {
    workspace = fresh({(lse_bytes + out_bytes) / 4}, at::kFloat, q.device());
    a.out_accum = static_cast<float*>(workspace.data_ptr()), a.lse_accum = a.out_accum + out_bytes / 4;
  }
  int status;
  {
    const fa_stream_t st = stream_of(q);
    py::gil_scoped_release unlocked;
    status = fa_fwd_tree(&t, st);
  }
  check(status, "flash_attn_tree_with_kvcache");
  if (k_in) changed(kc), changed(vc);
  return py::make_tuple(out, lse);
}

// Rows (batch, seqlen, heads, dim), or (tokens, heads, dim) as one sequence
FaTensor rows_view(const Tensor& t) {
  if (t.dim() == 3) return FaTensor{t.data_ptr(), 0, t.stride(0), t.stride(1)};
  return FaTensor{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}
bool repeats(const Tensor& t) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.stride(i) == 0 && t.size(i) > 1) return true;
  return false;
}

// What a rotation takes beside its rows
struct Turn {
  Tensor cos, sin, positions;
  std::vector<int64_t> sections;
  bool cycled, interleaved, conjugate;
};

// (q, k) turned, k undefined without one; with slots q alone, and k and v in the caches
std::pair<Tensor, Tensor> turn_axes(const Tensor& q_in, const MaybeTensor& k_in, const MaybeTensor& v_in, const Turn& how, bool inplace, const MaybeTensor& slots,
                                    const MaybeTensor& k_cache, const MaybeTensor& v_cache) {
  const Tensor &cos_in = how.cos, &sin_in = how.sin, &positions = how.positions;
  const std::vector<int64_t>& sections = how.sections;
  require(q_in.defined() && (q_in.dim() == 3 || q_in.dim() == 4), "q must have shape (batch, seqlen, nheads, headdim) or (tokens, nheads, headdim)");
  const int64_t dims = q_in.dim(), heads = q_in.size(-2), d = q_in.size(-1);
  const int64_t batch = dims == 4 ? q_in.size(0) : 1, seqlen = q_in.size(dims - 3), tokens = batch * seqlen;
  const auto dtype = q_in.scalar_type();
  require_rows(q_in, "q", dims, dtype);
  require(d > 0 && d <= 256 && heads > 0, "Only support headdim <= 256, and at least one head");
  int64_t heads_k = 0;
  for (const MaybeTensor* t : {&k_in, &v_in}) {
    if (!*t) continue;
    require_rows(**t, t == &k_in ? "k" : "v", dims, dtype);
    heads_k = k_in ? k_in->size(-2) : 0;
    bool same = (*t)->size(-1) == d && (*t)->size(-2) == heads_k && heads_k > 0;
    for (int64_t i = 0; i + 2 < dims; ++i) same = same && (*t)->size(i) == q_in.size(i);
    require(same, "k and v must have the tokens and the head dimension of q, and one number of heads");
  }
  const int64_t axes = sections.size();
  require(axes >= 1 && axes <= 4, "sections: 1 to 4 axes");
  int64_t pairs = 0;
  for (int64_t n : sections) {
    require(n >= 0 && n <= 128, "sections: numbers of pairs");
    pairs += n;
  }
  require(pairs >= 1 && 2 * pairs <= d, "rotary_dim, twice the sum of the sections, must be in [2, headdim]");
  require(cos_in.dim() == 2 && sin_in.sizes() == cos_in.sizes() && cos_in.size(1) == pairs, "cos and sin must have shape (rows, sum of the sections)");
  require(cos_in.scalar_type() == dtype && sin_in.scalar_type() == dtype, "Input and cos/sin must have the same dtype");
  require(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong, "positions must be int32 or int64");
  const int64_t lead = dims - 2, extra = positions.dim() - lead;
  bool fit = extra == 1 ? positions.size(0) == axes : extra == 0 && axes == 1;
  for (int64_t i = 0; fit && i < lead; ++i) fit = positions.size(extra + i) == q_in.size(i);
  require(fit, "positions must have shape (axes, batch, seqlen) or (axes, tokens), as q has them");
  FaRotaryAxesArgs a = {};
  if (how.cycled) {  // axis x > 0 takes pairs x, x + axes, x + 2 axes, ...; the first axis what is left
    for (int64_t x = 1; x < axes; ++x)
      for (int64_t j = 0; j < sections[x]; ++j) {
        require(x + axes * j < pairs, "sections: an axis has more pairs than its turns");
        a.axis_of_pair[x + axes * j] = (uint8_t)x;
      }
  } else {
    int64_t at = 0;
    for (int64_t x = 0; x < axes; ++x)
      for (int64_t j = 0; j < sections[x]; ++j) a.axis_of_pair[at++] = (uint8_t)x;
  }
  if (slots) {
    require(k_in && v_in && k_cache && v_cache, "slots need k, v and both caches");
    require(slots->scalar_type() == at::kLong && slots->numel() == tokens && slots->is_contiguous(), "slots must be int64, contiguous, one per token");
    require_rows(*k_cache, "k_cache", 4, dtype);
    require_rows(*v_cache, "v_cache", 4, dtype);
    require(k_cache->sizes() == v_cache->sizes() && k_cache->size(2) == heads_k && k_cache->size(3) == d,
            "k_cache and v_cache must have shape (pages, page_block_size, nheads_k, headdim)");
    require(k_cache->stride(3) == 1 && v_cache->stride(3) == 1 && !repeats(*k_cache) && !repeats(*v_cache),
            "k_cache and v_cache must have contiguous last dimension and must not repeat elements");
  }
  for (const MaybeTensor* t : {&k_in})
    require(!inplace || (q_in.stride(-1) == 1 && !repeats(q_in) && (slots || !*t || ((*t)->stride(-1) == 1 && !repeats(**t)))),
            "in-place rotation needs a unit stride in the last dimension and elements of its own");
  if (inplace && k_in) require_two(q_in, *k_in, "q and k in place");
  if (inplace && v_in) require_two(q_in, *v_in, "q and v in place");
  if (slots) require_two(*k_cache, *v_cache, "k_cache and v_cache");
  require(fits({tokens, heads, heads_k, cos_in.size(0)}), "sizes are out of range");
  require_no_tangent({&q_in, maybe(k_in), maybe(v_in), &cos_in, &sin_in, maybe(k_cache), maybe(v_cache)});
  require_device({&q_in, maybe(k_in), maybe(v_in), &cos_in, &sin_in, &positions, maybe(slots), maybe(k_cache), maybe(v_cache)});

  const c10::cuda::CUDAGuard guard(q_in.device());
  auto unit = [](const Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); };
  const Tensor q = unit(q_in), cos = cos_in.contiguous(), sin = sin_in.contiguous();
  Tensor k, v, k_out;
  Tensor q_out = inplace ? q_in : fresh(q.sizes(), dtype, q.device());
  a.q = rows_view(q), a.q_out = rows_view(q_out);
  if (k_in) {
    k = unit(*k_in);
    a.k = rows_view(k);
    if (slots) {
      v = unit(*v_in);
      a.v = rows_view(v), a.k_out = rows_view(*k_cache), a.v_out = rows_view(*v_cache);
      a.slots = static_cast<int64_t*>(slots->data_ptr());
      a.page_block_size = to_i32(k_cache->size(1), "page size");
      a.num_slots = k_cache->size(0) * k_cache->size(1);
      if (a.page_block_size == 0) a.page_block_size = 1;
    } else {
      k_out = inplace ? *k_in : fresh(k.sizes(), dtype, k.device());
      a.k_out = rows_view(k_out);
    }
  }
  a.cos = cos.data_ptr(), a.sin = sin.data_ptr(), a.span = cos.size(0), a.pairs = pairs;
  a.positions = positions.data_ptr(), a.positions_64 = positions.scalar_type() == at::kLong;
  a.pos_stride_a = extra ? positions.stride(0) : 0;
  a.pos_stride_b = dims == 4 ? positions.stride(extra) : 0, a.pos_stride_s = positions.stride(extra + lead - 1);
  a.batch = batch, a.seqlen = seqlen, a.heads = heads, a.heads_k = heads_k, a.head_dim = d;
  a.dtype = code(q), a.interleaved = how.interleaved, a.conjugate = how.conjugate, a.axes = axes;
  int status;
  {
    const fa_stream_t st = stream_of(q);
    std::optional<py::gil_scoped_release> unlocked;
    if (PyGILState_Check()) unlocked.emplace();  // (autograd's threads come without it)
    status = fa_rotary_axes(&a, st);
  }
  check(status, slots ? "rotary_axes_to_cache" : "apply_rotary_emb_axes");
  if (inplace) changed(q_in);
  if (inplace && k_in && !slots) changed(*k_in);
  if (slots) changed(*k_cache), changed(*v_cache);
  return {q_out, k_out};
}

// The rotation as a node of autograd (natively, since the kernels of a small batch take 2 x 3 us and the host sets its time: 777 tokens forward and backward 77 us, of which
// torch takes 57 for a single multiplication and its gradient).
// Its gradient is the rotation back, so the backward is the same node with the other sign, and can itself be differentiated.
struct TurnNode : torch::autograd::Function<TurnNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const MaybeTensor& k, const Tensor& cos, const Tensor& sin,
                                                const Tensor& positions, const std::vector<int64_t>& sections, bool cycled, bool interleaved, bool conjugate) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({cos, sin, positions});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["how"] = (int64_t)(cycled | interleaved << 1 | conjugate << 2);
    const auto r = turn_axes(q, k, std::nullopt, {cos, sin, positions, sections, cycled, interleaved, conjugate}, false, std::nullopt, std::nullopt, std::nullopt);
    if (!k) return {r.first};
    return {r.first, r.second};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const auto sections = ctx->saved_data["sections"].toIntVector();
    const int64_t how = ctx->saved_data["how"].toInt();
    const bool dq = grads[0].defined(), dk = grads.size() > 1 && grads[1].defined();
    torch::autograd::variable_list out(9);
    if (!dq && !dk) return out;
    const auto r = apply(dq ? grads[0] : grads[1], dq && dk ? MaybeTensor(grads[1]) : MaybeTensor(), saved[0], saved[1], saved[2], sections, (how & 1) != 0,
                         (how & 2) != 0, (how & 4) == 0);
    if (dq) out[0] = r[0];
    if (dk) out[1] = r[dq ? 1 : 0];
    return out;
  }
};

py::object or_none(const Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }

// apply_rotary_emb_axes: (q, k)
py::tuple rotary_axes(const Tensor& q, const MaybeTensor& k, const Tensor& cos, const Tensor& sin, const Tensor& positions, const std::vector<int64_t>& sections,
                      bool cycled, bool interleaved, bool inplace) {
  if (at::GradMode::is_enabled() && (q.requires_grad() || (k && k->requires_grad()))) {
    if (inplace) refuse_gradients_in_place({&q, maybe(k)}, "apply_rotary_emb_axes");
    const auto r = TurnNode::apply(q, k, cos, sin, positions, sections, cycled, interleaved, false);
    return py::make_tuple(r[0], k ? py::cast(r[1]) : py::none());
  }
  const auto r = turn_axes(q, k, std::nullopt, {cos, sin, positions, sections, cycled, interleaved, false}, inplace, std::nullopt, std::nullopt, std::nullopt);
  return py::make_tuple(r.first, or_none(r.second));
}

// rotary_axes_to_cache: q
Tensor rotary_to_cache(const Tensor& q, const MaybeTensor& k, const MaybeTensor& v, const Tensor& cos, const Tensor& sin, const Tensor& positions,
                       const std::vector<int64_t>& sections, bool cycled, bool interleaved, bool inplace, const Tensor& slots, const MaybeTensor& k_cache,
                       const MaybeTensor& v_cache) {
  if (inplace) refuse_gradients_in_place({&q}, "rotary_axes_to_cache");
  return turn_axes(q, k, v, {cos, sin, positions, sections, cycled, interleaved, false}, inplace, slots, k_cache, v_cache).first;
}

// block table (batch, pages per sequence), stack of unused pages, their number: what reserving and releasing have in common
void require_pool(const Tensor& table, const Tensor& lens, const Tensor& free_pages, const Tensor& num_free, int64_t page) {
  require(is_type(table, at::kInt, 2) && (table.size(1) <= 1 || table.stride(1) == 1), "block_table must be int32 of shape (batch, pages per sequence) with contiguous last dimension");
  require(table.size(0) >= 1 && table.size(0) <= 16384, "the number of sequences must be in [1, 16384]");
  require(!repeats(table), "block_table must not repeat elements");
  require(is_type(lens, at::kInt, 1) && lens.size(0) == table.size(0) && lens.is_contiguous(), "cache_seqlens must be int32, contiguous, one per sequence");
  require(is_type(free_pages, at::kInt, 1) && free_pages.is_contiguous(), "free_pages must be int32, contiguous, of one dimension");
  require(is_type(num_free, at::kInt, 1) && num_free.size(0) == 2 && num_free.is_contiguous(), "num_free must be two int32: the number of free pages, and 0");
  require(page > 0 && fits({page, table.size(1), free_pages.size(0)}), "page_block_size must be positive");
}

// reserve_pages: (slots, positions, cu_seqlens, seqlens)
py::tuple reserve_pages(const Tensor& table, const Tensor& lens, const MaybeTensor& new_lens, int64_t new_len, const Tensor& free_pages,
                        const Tensor& num_free, int64_t page, int64_t total) {
  require_pool(table, lens, free_pages, num_free, page);
  const int64_t batch = table.size(0);
  if (new_lens)
    require(is_type(*new_lens, at::kInt, 1) && new_lens->size(0) == batch && new_lens->is_contiguous(), "new_lens must be an int, or int32, contiguous, one per sequence");
  require(new_len >= 0 && total >= 0 && fits({new_len, total}), "the numbers of new tokens must be in [0, 2^31)");
  require_device({&table, &lens, maybe(new_lens), &free_pages, &num_free});
  const c10::cuda::CUDAGuard guard(table.device());
  Carved all({total * 8, total * 4, (batch + 1) * 4, batch * 4}, table.device());
  Tensor slots = all.take({total}, at::kLong), positions = all.take({total}, at::kInt), cu = all.take({batch + 1}, at::kInt), seqlens = all.take({batch}, at::kInt);
  FaReserveArgs a = {};
  a.block_table = i32(table), a.table_stride = table.stride(0), a.batch = batch, a.per_seq = table.size(1), a.page_block_size = page;
  a.cache_seqlens = i32(lens), a.new_lens = new_lens ? i32(*new_lens) : nullptr, a.new_len = new_len;
  a.free_pages = i32(free_pages), a.pool = free_pages.size(0), a.num_free = i32(num_free);
  a.slots = static_cast<int64_t*>(slots.data_ptr()), a.positions = i32(positions), a.cu_seqlens = i32(cu), a.seqlens = i32(seqlens), a.total = total;
  check(fa_reserve_pages(&a, stream_of(table)), "reserve_pages");
  changed(table), changed(num_free);
  return py::make_tuple(slots, positions, cu, seqlens);
}

void release_pages(const Tensor& table, const Tensor& lens, const Tensor& keep, const Tensor& free_pages, const Tensor& num_free, int64_t page) {
  require_pool(table, lens, free_pages, num_free, page);
  require(is_type(keep, at::kInt, 1) && keep.size(0) == table.size(0) && keep.is_contiguous(), "keep_seqlens must be int32, contiguous, one per sequence");
  require_device({&table, &lens, &keep, &free_pages, &num_free});
  const c10::cuda::CUDAGuard guard(table.device());
  check(fa_release_pages(i32(table), table.stride(0), table.size(0), table.size(1), page, i32(lens), i32(keep), i32(free_pages), free_pages.size(0),
                         i32(num_free), stream_of(table)),
        "release_pages");
  changed(free_pages), changed(num_free);
}

// tree_layout: (words, positions)
py::tuple tree_layout(const Tensor& parents, const Tensor& lens) {
  require(is_type(parents, at::kInt, 2) && (parents.size(1) <= 1 || parents.stride(1) == 1), "parents must be int32 of shape (batch, nodes) with contiguous last dimension");
  const int64_t batch = parents.size(0), nodes = parents.size(1);
  require(nodes <= 8192 && fits({batch}), "a tree has at most 8192 nodes");
  require(is_type(lens, at::kInt, 1) && lens.size(0) == batch && lens.is_contiguous(), "cache_seqlens must be int32, contiguous, one per sequence");
  require_device({&parents, &lens});
  const c10::cuda::CUDAGuard guard(parents.device());
  Carved all({batch * nodes * ((nodes + 31) / 32) * 4, batch * nodes * 4}, parents.device());
  Tensor words = all.take({batch, nodes, (nodes + 31) / 32}, at::kInt), positions = all.take({batch, nodes}, at::kInt);
  check(fa_tree_layout(i32(parents), parents.stride(0), i32(lens), batch, nodes, i32(words), i32(positions), stream_of(parents)), "tree_layout");
  return py::make_tuple(words, positions);
}

Tensor pack_tree_mask(const Tensor& mask) {
  require(is_type(mask, at::kBool, 3) && mask.size(1) == mask.size(2), "a tree mask must be bool of shape (batch or 1, nodes, nodes)");
  const int64_t batch = mask.size(0), nodes = mask.size(1);
  require(fits({batch, nodes, batch * nodes}), "sizes are out of range");
  require_device({&mask});
  const c10::cuda::CUDAGuard guard(mask.device());
  Tensor words = fresh({batch, nodes, (nodes + 31) / 32}, at::kInt, mask.device());
  check(fa_pack_tree_mask(static_cast<const uint8_t*>(mask.data_ptr()), mask.stride(0), mask.stride(1), mask.stride(2), batch, nodes, i32(words), stream_of(mask)),
        "pack_tree_mask");
  return words;
}

// keep_path: lengths with the accepted nodes
Tensor keep_path(const py::object& given, const Tensor& lens, const Tensor& path, int64_t nodes, const MaybeTensor& table, const MaybeTensor& batch_idx,
                 const MaybeTensor& seqlens) {
  require(is_type(lens, at::kInt, 1) && lens.is_contiguous(), "cache_seqlens must be int32, contiguous, one per sequence");
  const int64_t batch = lens.size(0);
  require(is_type(path, at::kInt, 2) && path.size(0) == batch && (path.size(1) <= 1 || path.stride(1) == 1),
          "path must be int32 of shape (batch, longest path) with contiguous last dimension");
  require(nodes >= 0 && path.size(1) <= 12288 && fits({batch, nodes}), "a path has at most 12288 nodes");
  if (seqlens) require(is_type(*seqlens, at::kInt, 1) && seqlens->size(0) == batch && seqlens->is_contiguous(), "seqlens must be int32, contiguous, one per sequence");
  FaKeepArgs a = {};
  a.heads_k = a.head_dim = 1;
  std::vector<void*> ptrs;
  Tensor first;  // the first cache; of a stack, all of them
  int64_t at = 0;  // dimensions in front of a cache's own
  if (THPVariable_Check(given.ptr())) {
    first = THPVariable_Unpack(given.ptr());
    require(first.dim() == 5, "caches: a list of caches, or one tensor (caches, sequences or pages, rows, nheads_k, headdim)");
    at = 1;
    for (int64_t i = 0; i < first.size(0); ++i) ptrs.push_back(static_cast<char*>(first.data_ptr()) + i * first.stride(0) * first.element_size());
    require_rows(first, "the caches", 5, first.scalar_type());
  } else {
    require(PyList_Check(given.ptr()) || PyTuple_Check(given.ptr()), "caches: a list of caches, or one tensor (caches, sequences or pages, rows, nheads_k, headdim)");
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(given.ptr());
    PyObject** items = PySequence_Fast_ITEMS(given.ptr());
    for (Py_ssize_t i = 0; i < n; ++i) {
      require(THPVariable_Check(items[i]), "caches: a list of caches, or one tensor (caches, sequences or pages, rows, nheads_k, headdim)");
      const Tensor& c = THPVariable_Unpack(items[i]);
      require_rows(c, "a cache", 4, c.scalar_type());
      if (!i) first = c;
      require(c.sizes() == first.sizes() && c.strides() == first.strides() && c.scalar_type() == first.scalar_type(),
              "the caches must have one shape, dtype and layout, with contiguous last dimension");
      ptrs.push_back(c.data_ptr());
    }
  }
  const bool some = !ptrs.empty();
  {
    std::vector<void*> sorted = ptrs;
    std::sort(sorted.begin(), sorted.end());
    require(std::adjacent_find(sorted.begin(), sorted.end()) == sorted.end(), "the same cache is given twice");
  }
  if (some)
    require(first.stride(at + 3) == 1 && !repeats(first) && first.numel() > 0, "the caches must have one shape, dtype and layout, with contiguous last dimension");
  int64_t cap = 0, page = 0;
  if (table) {
    require(!batch_idx, "Paged KVcache does not support cache_batch_idx");
    require(is_type(*table, at::kInt, 2) && table->size(0) == batch && (table->size(1) <= 1 || table->stride(1) == 1),
            "block_table must be int32 of shape (batch, pages per sequence) with contiguous last dimension");
  }
  if (batch_idx)
    require(is_type(*batch_idx, at::kInt, 1) && batch_idx->size(0) == batch && batch_idx->is_contiguous(), "cache_batch_idx must be int32, contiguous, one per sequence");
  if (some) {
    const Tensor& c = first;
    page = c.size(at + 1);
    cap = table ? table->size(1) * page : page;
    require(table || batch_idx || c.size(at) >= batch, "the KV cache must hold at least `batch` sequences when cache_batch_idx is not given");
    require(fits({c.size(at), cap, c.size(at + 2) * c.size(at + 3)}), "sizes are out of range");
    a.stride_b = c.stride(at), a.stride_s = c.stride(at + 1), a.stride_h = c.stride(at + 2);
    a.batch_cache = c.size(at), a.heads_k = c.size(at + 2), a.head_dim = c.size(at + 3);
  }
  require_device({&lens, &path, maybe(table), maybe(batch_idx), maybe(seqlens), some ? &first : nullptr});
  if (!at)
    for (size_t i = 1; i < ptrs.size(); ++i) require_device({&lens, &THPVariable_Unpack(PySequence_Fast_ITEMS(given.ptr())[i])});
  const c10::cuda::CUDAGuard guard(lens.device());
  Tensor out = fresh({batch}, at::kInt, lens.device());
  a.caches = ptrs.data(), a.n_caches = to_i32(ptrs.size(), "number of caches");
  a.batch = batch, a.seqlen_cache = cap, a.cache_seqlens = i32(lens), a.new_seqlens = i32(out);
  if (batch_idx) a.cache_batch_idx = i32(*batch_idx);
  if (seqlens) a.seqlens = i32(*seqlens);
  if (table) a.block_table = i32(*table), a.table_stride = table->stride(0), a.page_block_size = page > 0 ? page : 1;
  a.path = i32(path), a.path_stride = path.stride(0), a.depth = path.size(1), a.nodes = nodes;
  check(fa_keep_path(&a, stream_of(lens)), "keep_tree_path");
  if (at && some) changed(first);
  if (!at)
    for (size_t i = 0; i < ptrs.size(); ++i) changed(THPVariable_Unpack(PySequence_Fast_ITEMS(given.ptr())[i]));
  return out;
}

}  // namespace

PYBIND11_MODULE(_torch_glue, m) {
  m.def("fwd", &fwd);
  m.def("bwd", &bwd);
  m.def("fwd_kvcache", &fwd_kvcache);
  m.def("tree_fwd", &tree_fwd);
  m.def("rotary_axes", &rotary_axes);
  m.def("rotary_to_cache", &rotary_to_cache);
  m.def("reserve_pages", &reserve_pages);
  m.def("release_pages", &release_pages);
  m.def("tree_layout", &tree_layout);
  m.def("pack_tree_mask", &pack_tree_mask);
  m.def("keep_path", &keep_path);
}
