// Host side of the calls whose kernels take a few microseconds: the token rows' sort and combine, the block
// norms and the logit steps (whallm_amd/ops.py documents them). A CPython extension against torch, host code
// only: it checks the arguments, allocates the outputs and calls the C ABI of libwhallm_moe.so. In Python
// these steps took 5 to 10 us a call, more than the kernels of a decode step.
//
// Errors: ValueError for what the call refuses, before anything is allocated or launched; WhallmError with
// wm_last_error() where the C call does.
#include <torch/extension.h>

#include <initializer_list>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/whallm_moe.h"

namespace {

using at::Tensor;
using Maybe = std::optional<Tensor>;

[[noreturn]] void refuse(const std::string& message) { throw py::value_error(message); }

std::string type_name(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kDouble: return "torch.float64";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return std::string("torch.") + c10::toString(t);
  }
}

Tensor of_type(const Tensor& t, at::ScalarType type, const char* name) {
  if (t.scalar_type() != type) refuse(std::string(name) + " must be " + type_name(type) + ", got " + type_name(t.scalar_type()));
  return t.contiguous();
}
Maybe of_type(const Maybe& t, at::ScalarType type, const char* name) {
  return t ? Maybe(of_type(*t, type, name)) : std::nullopt;
}
bool is_rows(at::ScalarType t) { return t == at::kBFloat16 || t == at::kFloat; }
Tensor rows_of(const Tensor& t, const char* name) {
  if (!is_rows(t.scalar_type()))
    refuse(std::string(name) + " must be bfloat16 or float32, got " + type_name(t.scalar_type()));
  return t.contiguous();
}
Tensor rows_like(const Tensor& t, const char* name, const Tensor& like) {
  if (t.scalar_type() != like.scalar_type())
    refuse(std::string(name) + " must be " + type_name(like.scalar_type()) + " like the other rows, got " +
           type_name(t.scalar_type()));
  return t.contiguous();
}

void* at_of(const Tensor& t) { return t.data_ptr(); }
void* at_of(const Maybe& t) { return t ? t->data_ptr() : nullptr; }
int is_f32(const Tensor& t) { return t.scalar_type() == at::kFloat; }

const Tensor* ptr(const Tensor& t) { return &t; }
const Tensor* ptr(const Maybe& t) { return t ? &*t : nullptr; }

// Refuses inputs whose gradient or tangent would be lost: these calls are not recorded by autograd. Forward mode is a
// mode of its own, on under torch.no_grad() and off in inference mode.
void no_autograd(const char* name, const char* gradients, std::initializer_list<const Tensor*> tensors) {
  const bool reverse = at::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (const Tensor* t : tensors) {
    if (!t) continue;
    if (reverse && t->requires_grad())
      refuse(std::string(name) + " is not recorded by autograd (" + gradients + "): call it under torch.no_grad()");
    if (forward && t->_fw_grad(0).defined()) refuse(std::string(name) + " has no forward-mode derivative: pass the tensor without its tangent");
  }
}

c10::Device device_of(std::initializer_list<const Tensor*> tensors) {
  std::optional<c10::Device> device;
  for (const Tensor* t : tensors) {
    if (!t) continue;
    if (!t->is_cuda()) refuse("whallm_amd ops take device (HIP) tensors");
    if (!device) device = t->device();
    else if (*device != t->device()) refuse("all tensors must be on one device");
  }
  return *device;
}

// The device made current for the call and its current stream.
struct On {
  c10::DeviceGuard guard;
  void* stream;
  explicit On(c10::Device device) : guard(device) {
    static py::object& raw = *new py::object(py::module_::import("torch._C").attr("_cuda_getCurrentRawStream"));
    stream = reinterpret_cast<void*>(raw((int)device.index()).cast<uintptr_t>());
  }
};

// Runs the C call without the interpreter's lock, as ctypes does.
template <typename Call>
void checked(const char* name, Call call) {
  int status;
  std::string message;
  {
    py::gil_scoped_release release;
    status = call();
    if (status != 0) message = wm_last_error();
  }
  if (status != 0) {
    const py::object error = py::module_::import("whallm_amd._lib").attr("WhallmError");
    PyErr_SetString(error.ptr(), (std::string(name) + ": " + message).c_str());
    throw py::error_already_set();
  }
}

// Whether two contiguous tensors have a byte in common, whichever storages hold them.
bool meet(const Tensor& a, const Tensor& b) {
  const char *p = static_cast<const char*>(a.const_data_ptr()), *q = static_cast<const char*>(b.const_data_ptr());
  return a.nbytes() > 0 && b.nbytes() > 0 && p < q + b.nbytes() && q < p + a.nbytes();
}
// The caller's `out` is written while other workgroups still read the inputs: it may be `same`, element for element, and
// lies over no other.
void own_out(const Maybe& out, const char* name, const Tensor& same, const char* same_name,
             std::initializer_list<const Tensor*> others) {
  if (!out) return;
  const bool itself = out->const_data_ptr() == same.const_data_ptr() && out->scalar_type() == same.scalar_type();
  bool apart = itself || !meet(*out, same);
  for (const Tensor* t : others) apart = apart && !(t && meet(*out, *t));
  if (!apart) refuse(std::string(name) + " must be " + same_name + " itself or share no memory with it, and none with another input");
}
// Autograd sees that `out` was written.
void changed(const Maybe& out) {
  if (out && !out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
}

Tensor empty(at::IntArrayRef shape, at::ScalarType type, c10::Device device) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(device));
}

// `n` elements of a new 1-d tensor from `first` on: a view without the dispatcher's way (0.1 us, narrow 0.5).
Tensor part(const Tensor& whole, int64_t first, int64_t n) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(whole.storage_offset() + first);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

// ---------------------------------------------------------------- token rows to experts and back

// The tokens of rows [T * k, H] in the order of `inverse`.
int64_t pair_rows(const Tensor& rows, const Tensor& inverse, int64_t k) {
  if (rows.dim() != 2 || rows.size(1) < 1) refuse("rows must be [tokens * k, hidden]");
  if (rows.size(1) > 1 << 20) refuse("hidden must be at most 1048576");
  if (rows.size(0) > INT32_MAX) refuse("tokens * k must be below 2^31");
  if (k > 64) refuse("k must be at most 64");
  if (k < 1 || rows.size(0) % k) refuse("rows must hold k rows of every token");
  if (inverse.scalar_type() != at::kInt || !inverse.is_contiguous() || inverse.numel() != rows.size(0))
    refuse("the permutation is not that of these rows");
  return rows.size(0) / k;
}

py::tuple sort_tokens(const Tensor& x_, const Tensor& indices_, int64_t experts, int64_t tile_rows) {
  no_autograd("sort_tokens", "its gradients are sort_tokens_backward's", {&x_});
  const Tensor x = rows_of(x_, "x");
  const int64_t dims = x.dim();
  bool fit = dims >= 1 && indices_.dim() == dims;
  for (int64_t i = 0; fit && i < dims - 1; ++i) fit = indices_.size(i) == x.size(i);
  if (!fit) refuse("indices must be [.., K] for x [.., H]");
  const Tensor indices = of_type(indices_, at::kInt, "indices");
  const int64_t H = x.size(-1), k = indices.size(-1);
  if (H < 1 || k < 1 || experts < 1 || tile_rows < 1) refuse("hidden, k, experts and tile_rows must be positive");
  if (k > 64 || experts > 1024 || H > 1 << 20) refuse("k must be at most 64, experts 1024 and hidden 1048576");
  if (tile_rows > INT32_MAX) tile_rows = INT32_MAX;
  const int64_t T = x.numel() / H, P = T * k;
  if (P > INT32_MAX) refuse("tokens * k must be below 2^31");
  const c10::Device device = device_of({&x, &indices});
  const On on(device);
  const int64_t max_tiles = (P + tile_rows - 1) / tile_rows + experts;
  const size_t ws_bytes = wm_sort_tokens_workspace_size((int32_t)T, (int32_t)k, (int32_t)experts);
  const Tensor rows = empty({P, H}, x.scalar_type(), device), tiles = empty({max_tiles, 2}, at::kInt, device);
  // the other lists and the workspace in one allocation
  const Tensor lists = empty({2 * P + experts + 2 + (int64_t)((ws_bytes + 3) / 4)}, at::kInt, device);
  int32_t* at = static_cast<int32_t*>(lists.data_ptr());
  int32_t *order = at, *inverse = at + P, *offsets = at + 2 * P, *count = offsets + experts + 1;
  checked("wm_sort_tokens", [&] {
    return wm_sort_tokens(at_of(x), is_f32(x), (int32_t)T, (int32_t)H, static_cast<int32_t*>(at_of(indices)), (int32_t)k,
                          (int32_t)experts, (int32_t)tile_rows, at_of(rows), order, inverse, offsets,
                          static_cast<int32_t*>(at_of(tiles)), count, count + 1, ws_bytes, on.stream);
  });
  return py::make_tuple(rows, part(lists, 0, P), part(lists, P, P), part(lists, 2 * P, experts + 1), tiles,
                        part(lists, 2 * P + experts + 1, 1));
}

Tensor sort_tokens_backward(const Tensor& drows_, const Tensor& inverse, int64_t k) {
  no_autograd("sort_tokens_backward", "it has no gradient", {&drows_});
  const Tensor drows = rows_of(drows_, "drows");
  const int64_t T = pair_rows(drows, inverse, k), H = drows.size(1);
  const c10::Device device = device_of({&drows, &inverse});
  const On on(device);
  const Tensor dx = empty({T, H}, drows.scalar_type(), device);
  checked("wm_sort_tokens_backward", [&] {
    return wm_sort_tokens_backward(at_of(drows), is_f32(drows), static_cast<int32_t*>(at_of(inverse)), (int32_t)T, (int32_t)k,
                                   (int32_t)H, at_of(dx), on.stream);
  });
  return dx;
}

// Whether `t` is [.., H] for weights [.., K].
bool fits(const Tensor& t, const Tensor& weights, int64_t H) {
  if (t.dim() != weights.dim() || t.size(-1) != H) return false;
  for (int64_t i = 0; i < t.dim() - 1; ++i)
    if (t.size(i) != weights.size(i)) return false;
  return true;
}

Tensor combine_rows(const Tensor& rows_, const Tensor& weights_, const Tensor& inverse, const Maybe& add_) {
  no_autograd("combine_rows", "its gradients are combine_rows_backward's", {&rows_, &weights_, ptr(add_)});
  const Tensor rows = rows_of(rows_, "rows"), weights = of_type(weights_, at::kFloat, "weights");
  if (weights.dim() < 1) refuse("weights must be [.., K]");
  const int64_t k = weights.size(-1), T = pair_rows(rows, inverse, k), H = rows.size(1);
  if (weights.numel() != T * k) refuse("weights must be [.., K] matching rows");
  Maybe add;
  if (add_) {
    add = rows_like(*add_, "add", rows);
    if (!fits(*add, weights, H)) refuse("add must be [.., H] matching weights");
  }
  const c10::Device device = device_of({&rows, &weights, &inverse, ptr(add)});
  const On on(device);
  at::DimVector shape(weights.sizes().begin(), weights.sizes().end());
  shape.back() = H;
  const Tensor y = empty(shape, rows.scalar_type(), device);
  checked("wm_combine_rows", [&] {
    return wm_combine_rows(at_of(rows), is_f32(rows), static_cast<float*>(at_of(weights)), static_cast<int32_t*>(at_of(inverse)),
                           (int32_t)T, (int32_t)k, (int32_t)H, at_of(add), at_of(y), on.stream);
  });
  return y;
}

std::tuple<Tensor, Tensor> combine_rows_backward(const Tensor& dy_, const Tensor& rows_, const Tensor& weights_,
                                                 const Tensor& inverse, const Tensor& offsets) {
  no_autograd("combine_rows_backward", "it has no gradient", {&dy_, &rows_, &weights_});
  const Tensor rows = rows_of(rows_, "rows"), dy = rows_like(dy_, "dy", rows), weights = of_type(weights_, at::kFloat, "weights");
  if (weights.dim() < 1) refuse("weights must be [.., K]");
  const int64_t k = weights.size(-1), T = pair_rows(rows, inverse, k), H = rows.size(1);
  if (weights.numel() != T * k || !fits(dy, weights, H)) refuse("dy must be [.., H] and weights [.., K] matching rows");
  if (offsets.scalar_type() != at::kInt || !offsets.is_contiguous() || offsets.numel() < 1)
    refuse("the permutation's offsets must be contiguous int32");
  const c10::Device device = device_of({&dy, &rows, &weights, &inverse, &offsets});
  const On on(device);
  const Tensor drows = at::empty_like(rows), dweights = at::empty_like(weights);
  checked("wm_combine_rows_backward", [&] {
    return wm_combine_rows_backward(at_of(dy), at_of(rows), is_f32(rows), static_cast<float*>(at_of(weights)),
                                    static_cast<int32_t*>(at_of(inverse)),
                                    static_cast<int32_t*>(at_of(offsets)) + offsets.numel() - 1, (int32_t)T, (int32_t)k, (int32_t)H,
                                    at_of(drows), static_cast<float*>(at_of(dweights)), on.stream);
  });
  return {drows, dweights};
}

// ---------------------------------------------------------------- norms around a block

struct NormForm {
  wm_block_norm_form c = {};
  Tensor y;
  Maybe post, pre, gate;
  int64_t H, T;
};

NormForm norm_form(const Tensor& residual, const Tensor& y, const Maybe& post, const Maybe& pre, const Maybe& gate,
                   bool gate_sigmoid, double scale, double eps, double weight_offset, bool post_norm) {
  NormForm f;
  if (!is_rows(residual.scalar_type()))
    refuse("residual must be float32 or bfloat16, got " + type_name(residual.scalar_type()));
  if (residual.dim() < 1 || residual.size(-1) < 1 || residual.size(-1) > 16384)
    refuse("residual must be [.., H] with H from 1 to 16384");
  f.H = residual.size(-1);
  f.T = residual.numel() / f.H;
  if (f.T > INT32_MAX) refuse("tokens must be below 2^31");
  f.y = of_type(y, at::kBFloat16, "y");
  if (f.y.sizes() != residual.sizes()) refuse("y must match residual");
  if (post && !post_norm) refuse("post_weight needs post_norm");
  if (!(eps >= 0)) refuse("eps must not be negative");
  f.post = of_type(post, at::kBFloat16, "post_weight");
  f.pre = of_type(pre, at::kBFloat16, "pre_weight");
  for (const Maybe* w : {&f.post, &f.pre})
    if (*w && ((*w)->dim() != 1 || (*w)->size(0) != f.H)) refuse("weights must be [H]");
  if (gate) {
    if (!is_rows(gate->scalar_type())) refuse("gate must be float32 or bfloat16, got " + type_name(gate->scalar_type()));
    bool lead = gate->dim() == residual.dim();
    for (int64_t i = 0; lead && i < residual.dim() - 1; ++i) lead = gate->size(i) == residual.size(i);
    if (gate->dim() == 1 && gate->size(0) == f.H) f.c.gate_kind = 2;
    else if (lead && gate->size(-1) == 1) f.c.gate_kind = 1;
    else if (lead && gate->size(-1) == f.H) f.c.gate_kind = 3;
    else refuse("gate must be [H], [.., 1] or [.., H]");
    f.gate = gate->contiguous();
    f.c.gate_fp32 = is_f32(*gate);
  }
  f.c.post_weight = at_of(f.post);
  f.c.pre_weight = at_of(f.pre);
  f.c.gate = at_of(f.gate);
  f.c.weight_offset = (float)weight_offset;
  f.c.scale = (float)scale;
  f.c.eps = (float)eps;
  f.c.post_norm = post_norm;
  f.c.gate_sigmoid = gate_sigmoid;
  f.c.residual_fp32 = is_f32(residual);
  return f;
}

std::tuple<Tensor, Tensor> block_norm(const Tensor& residual_, const Tensor& y, const Maybe& post, const Maybe& pre,
                                      const Maybe& gate, bool gate_sigmoid, double scale, double eps, double weight_offset,
                                      bool post_norm, const Maybe& out) {
  no_autograd("block_norm", "its gradients are block_norm_backward's", {&residual_, &y, ptr(post), ptr(pre), ptr(gate), ptr(out)});
  const NormForm f = norm_form(residual_, y, post, pre, gate, gate_sigmoid, scale, eps, weight_offset, post_norm);
  if (out && (out->scalar_type() != residual_.scalar_type() || out->sizes() != residual_.sizes() || !out->is_contiguous()))
    refuse("residual_out must be a contiguous tensor shaped and typed like residual");
  const Tensor residual = residual_.contiguous();
  own_out(out, "residual_out", residual, "residual", {&f.y, ptr(f.post), ptr(f.pre), ptr(f.gate)});
  const c10::Device device = device_of({&residual, &f.y, ptr(f.post), ptr(f.pre), ptr(f.gate), ptr(out)});
  const On on(device);
  const Tensor residual_out = out ? *out : at::empty_like(residual), x = at::empty_like(f.y);
  checked("wm_block_norm", [&] {
    return wm_block_norm(&f.c, at_of(residual), at_of(f.y), (int32_t)f.T, (int32_t)f.H, at_of(residual_out), at_of(x), on.stream);
  });
  changed(out);
  return {x, residual_out};
}

py::tuple block_norm_backward(const Tensor& dx_, const Maybe& dresidual_, const Tensor& residual_out_, const Tensor& y,
                              const Maybe& post, const Maybe& pre, const Maybe& gate, bool gate_sigmoid, double scale, double eps,
                              double weight_offset, bool post_norm) {
  no_autograd("block_norm_backward", "it has no gradient",
              {&dx_, ptr(dresidual_), &residual_out_, &y, ptr(post), ptr(pre), ptr(gate)});
  const NormForm f = norm_form(residual_out_, y, post, pre, gate, gate_sigmoid, scale, eps, weight_offset, post_norm);
  const Tensor dx = of_type(dx_, at::kBFloat16, "dx"), residual_out = residual_out_.contiguous();
  if (dx.sizes() != residual_out.sizes()) refuse("dx must match residual_out");
  Maybe dresidual;
  if (dresidual_) {
    if (dresidual_->scalar_type() != residual_out.scalar_type() || dresidual_->sizes() != residual_out.sizes())
      refuse("dresidual must be shaped and typed like residual_out");
    dresidual = dresidual_->contiguous();
  }
  const c10::Device device = device_of({&dx, ptr(dresidual), &residual_out, &f.y, ptr(f.post), ptr(f.pre), ptr(f.gate)});
  const On on(device);
  const Tensor dr = at::empty_like(residual_out), dy = at::empty_like(f.y);
  Maybe dpost, dpre, dgate;
  const bool channel = f.c.gate_kind == 2;
  const int64_t columns = (f.post ? 1 : 0) + (f.pre ? 1 : 0) + channel;  // fp32 [H] each, in one allocation
  if (columns) {
    const Tensor sums = empty({columns * f.H}, at::kFloat, device);
    int64_t at = 0;
    if (f.post) dpost = part(sums, at, f.H), at += f.H;
    if (f.pre) dpre = part(sums, at, f.H), at += f.H;
    if (channel) dgate = part(sums, at, f.H);
  }
  if (f.gate && !channel) dgate = empty(f.gate->sizes(), f.c.gate_kind == 3 ? f.gate->scalar_type() : at::kFloat, device);
  const size_t ws_bytes = wm_block_norm_backward_workspace_size((int32_t)f.T, (int32_t)f.H);
  const Tensor ws = empty({(int64_t)ws_bytes}, at::kByte, device);
  checked("wm_block_norm_backward", [&] {
    return wm_block_norm_backward(&f.c, at_of(dx), at_of(dresidual), at_of(residual_out), at_of(f.y), (int32_t)f.T, (int32_t)f.H,
                                  at_of(dr), at_of(dy), static_cast<float*>(at_of(dpost)), static_cast<float*>(at_of(dpre)),
                                  at_of(dgate), at_of(ws), ws_bytes, on.stream);
  });
  return py::make_tuple(dr, dy, dpost, dpre, dgate);
}

// ---------------------------------------------------------------- logits to acceptance

Maybe row_values(const Maybe& t, int64_t rows, at::ScalarType type, const char* name) {
  if (!t) return std::nullopt;
  Tensor v = of_type(*t, type, name);
  if (v.dim() != 1 || v.size(0) != rows) refuse(std::string(name) + " must be [rows]");
  return v;
}

// [rows, n], or [1, n] for a list that all rows share; `stride` elements lie between rows.
Maybe row_lists(const Maybe& t, int64_t rows, at::ScalarType type, const char* name, int64_t& stride) {
  if (!t) return std::nullopt;
  Tensor v = of_type(*t, type, name);
  if (v.dim() != 2 || (v.size(0) != rows && v.size(0) != 1))
    refuse(std::string(name) + " must be [rows, n], or [1, n] for all rows");
  stride = v.size(0) == 1 ? 0 : v.size(1);
  return v;
}

Tensor process_logits(const Tensor& logits_, const Maybe& history_, const Maybe& lengths_, const Maybe& prompt_lengths_,
                      const Maybe& repetition_, const Maybe& frequency_, const Maybe& presence_, const Maybe& bias_ids_,
                      const Maybe& bias_values_, const Maybe& mask_, const Maybe& temperature_, bool log_probs, const Maybe& out_) {
  no_autograd("process_logits", "it has no gradient",
              {&logits_, ptr(repetition_), ptr(frequency_), ptr(presence_), ptr(bias_values_), ptr(temperature_), ptr(out_)});
  const Tensor logits = rows_of(logits_, "logits");
  if (logits.dim() != 2 || logits.size(1) < 1) refuse("logits must be [rows, vocab]");
  const int64_t R = logits.size(0), V = logits.size(1);
  if (R > INT32_MAX || V > 1 << 22) refuse("logits must have at most 2147483647 rows of at most 4194304 values");
  wm_logit_rules r = {};
  Maybe lengths = row_values(lengths_, R, at::kInt, "lengths"), prompts = row_values(prompt_lengths_, R, at::kInt, "prompt_lengths");
  const Maybe repetition = row_values(repetition_, R, at::kFloat, "repetition"),
              frequency = row_values(frequency_, R, at::kFloat, "frequency"),
              presence = row_values(presence_, R, at::kFloat, "presence"),
              temperature = row_values(temperature_, R, at::kFloat, "temperature");
  Maybe history = row_lists(history_, R, at::kInt, "history", r.history_stride);
  if (!history && (lengths || prompts)) refuse("lengths need a history");
  if (history && history->size(1) == 0) history = lengths = prompts = std::nullopt;
  if (history && history->size(1) > (1 << 20) - 1) refuse("history must hold at most 1048575 tokens a row");
  if (bias_ids_.has_value() != bias_values_.has_value()) refuse("bias_ids and bias_values go together");
  if (bias_ids_ && bias_ids_->sizes() != bias_values_->sizes()) refuse("bias_ids and bias_values must have one shape");
  Maybe bias_ids = row_lists(bias_ids_, R, at::kInt, "bias_ids", r.bias_stride),
        bias_values = of_type(bias_values_, at::kFloat, "bias_values");
  if (bias_ids && bias_ids->size(1) == 0) bias_ids = bias_values = std::nullopt;
  if (bias_ids && bias_ids->size(1) > 2047) refuse("bias_ids must hold at most 2047 tokens a row");
  const Maybe mask = row_lists(mask_, R, at::kInt, "mask", r.mask_stride);
  if (mask && mask->size(1) != (V + 31) / 32) refuse("mask must hold a bit for every token, 32 in a word");
  if (out_ && (out_->scalar_type() != at::kFloat || out_->sizes() != logits.sizes() || !out_->is_contiguous()))
    refuse("out must be a contiguous float32 tensor shaped like logits");
  own_out(out_, "out", logits, "logits",
          {ptr(history), ptr(lengths), ptr(prompts), ptr(repetition), ptr(frequency), ptr(presence), ptr(bias_ids),
           ptr(bias_values), ptr(mask), ptr(temperature)});
  const c10::Device device = device_of({&logits, ptr(history), ptr(lengths), ptr(prompts), ptr(repetition), ptr(frequency),
                                        ptr(presence), ptr(bias_ids), ptr(bias_values), ptr(mask), ptr(temperature), ptr(out_)});
  const On on(device);
  r.history = static_cast<int32_t*>(at_of(history));
  r.history_len = history ? (int32_t)history->size(1) : 0;
  r.biases = bias_ids ? (int32_t)bias_ids->size(1) : 0;
  r.lengths = static_cast<int32_t*>(at_of(lengths));
  r.prompt_lengths = static_cast<int32_t*>(at_of(prompts));
  r.repetition = static_cast<float*>(at_of(repetition));
  r.frequency = static_cast<float*>(at_of(frequency));
  r.presence = static_cast<float*>(at_of(presence));
  r.bias_ids = static_cast<int32_t*>(at_of(bias_ids));
  r.bias_values = static_cast<float*>(at_of(bias_values));
  r.mask = at_of(mask);
  r.temperature = static_cast<float*>(at_of(temperature));
  const Tensor out = out_ ? *out_ : empty({R, V}, at::kFloat, device);
  const size_t ws_bytes = log_probs ? wm_process_logits_workspace_size((int32_t)R, (int32_t)V) : 0;
  Maybe ws;
  if (log_probs) ws = empty({(int64_t)ws_bytes}, at::kByte, device);
  checked("wm_process_logits", [&] {
    return wm_process_logits(at_of(logits), is_f32(logits), (int32_t)R, (int32_t)V, &r, log_probs, static_cast<float*>(at_of(out)),
                             at_of(ws), ws_bytes, on.stream);
  });
  changed(out_);
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("sort_tokens", &sort_tokens);
  m.def("sort_tokens_backward", &sort_tokens_backward);
  m.def("combine_rows", &combine_rows);
  m.def("combine_rows_backward", &combine_rows_backward);
  m.def("block_norm", &block_norm);
  m.def("block_norm_backward", &block_norm_backward);
  m.def("process_logits", &process_logits);
}
