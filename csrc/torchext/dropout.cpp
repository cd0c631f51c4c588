// Counter-based dropout as a differentiable torch operator (ops/masking.py): the host side of
// every call -- output, view walked, launch -- and its autograd node, without Python in either
// direction: a forward and a backward pass cost the host 53 us where torch's own dropout and addition
// cost it 61 and an addition alone 40 (as Python functions they cost 120 where this costs 47).
// Device tensors go to tpi_dropout (csrc/hip/dropout.hip); host tensors are computed here, to the
// same bits.
#include <ATen/Parallel.h>
#include <torch/extension.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/library.h>

#include <vector>

#include "../common/float16.h"
#include "../common/philox.h"
#include "../hip/tpi_hip.h"
#include "torchext.h"

namespace tpi {

namespace {

inline float load(const void* base, int64_t at, int type) {
  if (type == TPI_F32) return ((const float*)base)[at];
  const uint16_t h = ((const uint16_t*)base)[at];
  return type == TPI_F16 ? tpi_f16_to_f32(h) : tpi_bf16_to_f32(h);
}

inline void store(void* base, int64_t at, int type, float v) {
  if (type == TPI_F32) ((float*)base)[at] = v;
  else ((uint16_t*)base)[at] = type == TPI_F16 ? tpi_f32_to_f16(v) : tpi_f32_to_bf16(v);
}

void dropout_range(const tpi_dropout_args& a, uint64_t seed, uint64_t draw, uint64_t lo,
                   uint64_t hi) {
  int64_t index[TPI_MAX_DIMS];
  uint64_t rest = lo;
  for (int d = a.ndim - 1; d >= 0; --d) {
    index[d] = (int64_t)(rest % (uint64_t)a.sizes[d]);
    rest /= (uint64_t)a.sizes[d];
  }
  const tpi_keep keep = tpi_keep_below(a.threshold);
  uint64_t block = ~0ull;
  uint32_t kept = 0;
  for (uint64_t e = lo; e < hi; ++e) {
    int64_t x = 0, r = 0, o = 0;
    uint64_t n = a.first;
    for (int d = 0; d < a.ndim; ++d) {
      x += index[d] * a.sx[d];
      r += index[d] * a.sr[d];
      o += index[d] * a.so[d];
      n += (uint64_t)(index[d] * a.si[d]);
    }
    if (n >> 3 != block) {
      block = n >> 3;
      kept = tpi_draw_block(block, draw, seed, keep);
    }
    float v = 0.0f;
    if (kept >> (n & 7) & 1) v = load((const void*)a.x, x, a.in_type) * a.scale;
    if (a.residual) v = v + load((const void*)a.residual, r, a.out_type);
    store((void*)a.out, o, a.out_type, v);
    for (int d = a.ndim - 1; d >= 0 && ++index[d] == a.sizes[d]; --d) index[d] = 0;
  }
}

void dropout_host(const tpi_dropout_args& a) {
  uint64_t seed = a.seed, draw = a.draw, total = 1;
  if (a.state) {
    seed = ((const uint64_t*)a.state)[0];
    draw = ((const uint64_t*)a.state)[1] + a.draw;
  }
  if (a.used) {
    ((uint64_t*)a.used)[0] = seed;
    ((uint64_t*)a.used)[1] = draw;
  }
  for (int d = 0; d < a.ndim; ++d) total *= (uint64_t)a.sizes[d];
  at::parallel_for(0, (int64_t)total, 1 << 15, [&](int64_t lo, int64_t hi) {
    dropout_range(a, seed, draw, (uint64_t)lo, (uint64_t)hi);
  });
}

int type_of(at::ScalarType t) {
  return t == at::kFloat ? TPI_F32 : t == at::kHalf ? TPI_F16 : TPI_BF16;
}

// What names a mask and places a tensor in it.  Numbers without a sign go through torch as the signed
// ones of their bits.
struct Mask : torch::CustomClassHolder {
  int64_t threshold;
  double scale;
  int64_t seed, number;
  std::optional<at::Tensor> state;  // {seed, number} on the device
  int64_t first;
  std::vector<int64_t> strides;  // of the whole tensor's indexes; empty: x is the whole tensor
  Mask(int64_t threshold, double scale, int64_t seed, int64_t number,
       const std::optional<at::Tensor>& state, int64_t first, at::IntArrayRef strides)
      : threshold(threshold), scale(scale), seed(seed), number(number), state(state), first(first),
        strides(strides.vec()) {}
};

// Views walked together, as dimensions that every operand has a stride for: those of size 1
// dropped, those merged that all operands walk as one.
int merge(at::IntArrayRef shape, const int64_t* const (&strides)[4], tpi_dropout_args& a) {
  int n = 0;
  int64_t* const to[4] = {a.sx, a.sr, a.so, a.si};
  for (size_t d = 0; d < shape.size(); ++d) {
    const int64_t size = shape[d];
    if (size == 1) continue;
    bool one = n > 0;
    for (int k = 0; one && k < 4; ++k) one = to[k][n - 1] == strides[k][d] * size;
    if (one) {
      a.sizes[n - 1] *= size;
    } else {
      TORCH_CHECK_VALUE(n < TPI_MAX_DIMS, "dropout: tensors with more than ", TPI_MAX_DIMS,
                        " (merged) dims are not supported");
      a.sizes[n++] = size;
    }
    for (int k = 0; k < 4; ++k) to[k][n - 1] = strides[k][d];
  }
  if (n == 0) {
    a.sizes[n++] = 1;
    for (int k = 0; k < 4; ++k) to[k][0] = 1;
  }
  return n;
}

// Where a tensor's first element is.  Not every tensor has memory for its elements: a wrapper
// (DTensor, jagged, fake) has none of its own, a storage may have been shrunk or freed; their
// address is null, or what lies behind it is not theirs.
uint64_t address(const at::Tensor& t) {
  TORCH_CHECK_TYPE(t.layout() == at::kStrided && !t.is_nested(),
                   "dropout of a nested or sparse tensor is not supported");
  uint64_t elements = (uint64_t)t.storage_offset() + 1;
  for (int64_t d = 0; d < t.dim(); ++d) elements += (uint64_t)((t.size(d) - 1) * t.stride(d));
  const void* p = t.const_data_ptr();
  TORCH_CHECK_VALUE(p && elements * t.element_size() <= t.storage().nbytes(),
                    "dropout needs tensors with memory of their own for all elements (of a "
                    "distributed tensor, its local part)");
  return (uint64_t)p;
}

at::Tensor empty_out(const at::Tensor& x, const std::optional<at::Tensor>& residual,
                     at::ScalarType dtype) {
  TORCH_CHECK_TYPE(x.layout() == at::kStrided && !x.is_nested(),
                   "dropout of a nested or sparse tensor is not supported");
  return at::empty_like(residual ? *residual : x, x.options().dtype(dtype));
}

#define TPI_DROPOUT_ARGS                                                                       \
  const at::Tensor &x, const std::optional<at::Tensor>&residual, at::ScalarType dtype,         \
      int64_t threshold, double scale, int64_t seed, int64_t number,                           \
      const std::optional<at::Tensor>&state, int64_t first, at::IntArrayRef strides,           \
      const std::optional<at::Tensor>&used

bool two_words(const std::optional<at::Tensor>& t, const at::Tensor& x) {
  return !t || (t->scalar_type() == at::kLong && t->numel() == 2 && t->is_contiguous() &&
                t->device() == x.device());
}

bool type_ok(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

// What ops.dropout has checked; a traced program may be run on other tensors.
void check_args(TPI_DROPOUT_ARGS) {
  const at::ScalarType type = x.scalar_type();
  TORCH_CHECK_TYPE(type_ok(type) && type_ok(dtype) &&
                       (type == dtype || type == at::kFloat || dtype == at::kFloat) &&
                       (!residual || (residual->scalar_type() == dtype &&
                                      (type == dtype || dtype == at::kFloat))),
                   "dropout: unsupported types");
  TORCH_CHECK_VALUE(!residual || (residual->sizes() == x.sizes() && residual->device() == x.device()),
                    "dropout: the residual must have x's shape and device");
  TORCH_CHECK_VALUE(threshold >= 0 && threshold <= 1ll << 32 && number >= 0 && first >= 0,
                    "dropout: a number is out of range");
  TORCH_CHECK_VALUE(strides.empty() || (int64_t)strides.size() == x.dim(),
                    "dropout: a stride of the whole tensor for each dimension");
  TORCH_CHECK_VALUE(two_words(state, x) && two_words(used, x),
                    "dropout: a draw's state must be two contiguous int64 on x's device");
}

// The operator itself, on the host and the device.
at::Tensor dropout_kernel(TPI_DROPOUT_ARGS) {
  check_args(x, residual, dtype, threshold, scale, seed, number, state, first, strides, used);
  at::Tensor out = empty_out(x, residual, dtype);
  const int64_t n = x.numel();
  if (n == 0) return out;  // nor will the backward pass read `used`
  tpi_dropout_args a{};
  a.x = address(x);
  a.residual = residual ? address(*residual) : 0;
  a.out = address(out);
  a.state = state ? address(*state) : 0;
  a.used = used ? address(*used) : 0;
  a.seed = (uint64_t)seed;
  a.draw = (uint64_t)number;
  a.first = (uint64_t)first;
  a.threshold = (uint64_t)threshold;
  a.scale = (float)scale;
  a.in_type = type_of(x.scalar_type());
  a.out_type = type_of(dtype);
  if (strides.empty() && x.is_contiguous() && out.is_contiguous() &&
      (!residual || residual->is_contiguous())) {
    a.ndim = 1;
    a.sizes[0] = n;
    a.sx[0] = a.sr[0] = a.so[0] = a.si[0] = 1;
  } else {
    std::vector<int64_t> index = strides.vec();
    if (index.empty()) {
      index.resize(x.dim());
      int64_t step = 1;
      for (int64_t d = x.dim() - 1; d >= 0; --d) {
        index[d] = step;
        step *= x.size(d);
      }
    }
    const int64_t* const walked[4] = {x.strides().data(),
                                      residual ? residual->strides().data() : out.strides().data(),
                                      out.strides().data(), index.data()};
    a.ndim = merge(x.sizes(), walked, a);
  }
  if (x.is_cpu()) {
    dropout_host(a);
    return out;
  }
  const c10::DeviceGuard guard(x.device());
  hip_check(hip_api().dropout(&a, current_stream(x.device().index())), "dropout");
  return out;
}

at::Tensor dropout_meta(TPI_DROPOUT_ARGS) { return empty_out(x, residual, dtype); }

// The operator as torch knows it: whatever a program does to its operators (tracing, wrapped
// tensors, differentiation) finds it there.
const auto& dropout_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("tpi::dropout", "")
                             .typed<at::Tensor(TPI_DROPOUT_ARGS)>();
  return op;
}

at::Tensor call(const at::Tensor& x, const std::optional<at::Tensor>& residual,
                at::ScalarType dtype, const Mask& mask, const std::optional<at::Tensor>& used) {
  return dropout_op().call(x, residual, dtype, mask.threshold, mask.scale, mask.seed, mask.number,
                           mask.state, mask.first, mask.strides, used);
}

// A gradient has whatever layout the rest of the graph gave it.  One of more dimensions than a launch
// walks may not merge into those where the forward pass's operands did; laid out in order, it
// does wherever they did.
at::Tensor walkable(const at::Tensor& t) { return t.dim() > TPI_MAX_DIMS ? t.contiguous() : t; }

// The gradient of a dropped element is 0, of a kept one the scale times the output's: the
// operator itself, applied to the gradient (so it can be differentiated again).
struct Dropout : torch::autograd::Function<Dropout> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                            const std::optional<at::Tensor>& residual, at::ScalarType dtype,
                            const c10::intrusive_ptr<Mask>& mask,
                            std::optional<at::Tensor> used) {
    c10::intrusive_ptr<Mask> again = mask;
    if (mask->state && x.requires_grad()) {
      // the state may have moved on by the time the backward pass runs
      if (!used) used = at::empty({2}, mask->state->options());
      again = c10::make_intrusive<Mask>(*mask);
      again->state = used;
      again->number = 0;
    }
    ctx->saved_data["mask"] = c10::IValue::make_capsule(again);
    ctx->saved_data["type"] = (int64_t)x.scalar_type();
    ctx->saved_data["residual"] = residual && residual->requires_grad();
    ctx->saved_data["x"] = x.requires_grad();
    const at::AutoDispatchBelowADInplaceOrView below;
    return call(x, residual, dtype, *mask, used);
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const at::Tensor& grad = grads[0];
    at::Tensor dx, dr;
    if (grad.defined() && ctx->saved_data["x"].toBool())
      dx = call(walkable(grad.resolve_neg()), std::nullopt,
                (at::ScalarType)ctx->saved_data["type"].toInt(),
                *c10::static_intrusive_pointer_cast<Mask>(ctx->saved_data["mask"].toCapsule()),
                std::nullopt);
    if (ctx->saved_data["residual"].toBool()) dr = grad;
    return {dx, dr, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// The tangent that forward mode carries with a tensor; undefined: none.
at::Tensor tangent(const std::optional<at::Tensor>& t) {
  return t && t->defined() ? t->_fw_grad(/*level=*/0) : at::Tensor();
}

at::Tensor dropout_autograd(TPI_DROPOUT_ARGS) {
  const at::Tensor tx = tangent(x), tr = tangent(residual);
  const bool forward =
      (tx.defined() || tr.defined()) && c10::AutogradState::get_tls_state().get_fw_grad_mode();
  const bool backward =
      at::GradMode::is_enabled() && (x.requires_grad() || (residual && residual->requires_grad()));
  if (!forward && !backward) {
    const at::AutoDispatchBelowADInplaceOrView below;
    return dropout_op().call(x, residual, dtype, threshold, scale, seed, number, state, first, strides,
                             used);
  }
  const auto mask = c10::make_intrusive<Mask>(threshold, scale, seed, number, state, first, strides);
  if (forward) {
    // linear in both: the tangent is the operator, applied to x's, plus the residual's
    std::optional<at::Tensor> added, turned;
    if (residual) added = tr.defined() ? residual->_fw_primal(0) : *residual;
    if (tr.defined()) turned = tr;
    const at::Tensor out = call(tx.defined() ? x._fw_primal(0) : x, added, dtype, *mask, used);
    return at::_make_dual(out, tx.defined() ? call(tx, turned, dtype, *mask, std::nullopt) : tr.clone(),
                          0);
  }
  return Dropout::apply(x, residual, dtype, mask, used);
}

at::Tensor dropout(const at::Tensor& x, const std::optional<at::Tensor>& residual,
                   uint64_t threshold, double scale, uint64_t seed, uint64_t number,
                   const std::optional<at::Tensor>& state, uint64_t first,
                   const std::vector<int64_t>& strides) {
  // views that are negated lazily (the imaginary part of a conjugate) are written out
  std::optional<at::Tensor> added;
  if (residual) added = residual->resolve_neg();
  return dropout_op().call(x.resolve_neg(), added, added ? added->scalar_type() : x.scalar_type(),
                           (int64_t)threshold, scale, (int64_t)seed, (int64_t)number, state,
                           (int64_t)first, strides, std::nullopt);
}

TORCH_LIBRARY(tpi, m) {
  m.def("dropout(Tensor x, Tensor? residual, ScalarType dtype, int threshold, float scale, int seed, "
        "int number, Tensor? state, int first, int[] strides, Tensor(a!)? used=None) -> Tensor");
}
TORCH_LIBRARY_IMPL(tpi, CPU, m) { m.impl("dropout", &dropout_kernel); }
TORCH_LIBRARY_IMPL(tpi, CUDA, m) { m.impl("dropout", &dropout_kernel); }
TORCH_LIBRARY_IMPL(tpi, Meta, m) { m.impl("dropout", &dropout_meta); }
TORCH_LIBRARY_IMPL(tpi, Autograd, m) { m.impl("dropout", &dropout_autograd); }

}  // namespace

void bind_dropout(py::module_& m) {
  m.def("dropout", &dropout, py::call_guard<py::gil_scoped_release>());
  m.def("surroundings", [] {
    const bool traced =
        torch::jit::tracer::isTracing() ||
        c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value();
    return (torch::autograd::get_current_graph_task_id() >= 0 ? 1 : 0) | (traced ? 2 : 0);
  }, "bit 0: the caller runs inside a backward pass; bit 1: what it does is being recorded");
}

}  // namespace tpi
