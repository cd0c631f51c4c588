// Counter-based dropout as a differentiable torch operator (ops/masking.py): the host side of
// every call -- output, view walked, launch -- and its autograd node, without Python in either
// direction: a forward and a backward pass cost the host 47 us (120 as Python functions; torch's own
// dropout and addition 55, an addition alone 34).
// Device tensors go to tpi_dropout (csrc/hip/dropout.hip); host tensors are computed here, to the
// same bits.
#include <ATen/Parallel.h>
#include <torch/extension.h>

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

// What names a mask and places a tensor in it.
struct Mask : torch::CustomClassHolder {
  uint64_t seed, number, first, threshold;
  float scale;
  std::vector<int64_t> strides;  // of the whole tensor's indexes; empty: x is the whole tensor
  at::Tensor state;              // {seed, number} on the device, or undefined
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

at::Tensor dropout_pass(const at::Tensor& x, const at::Tensor& residual, at::ScalarType out_type,
                        const Mask& mask, const at::Tensor& used) {
  TORCH_CHECK_TYPE(x.layout() == at::kStrided && !x.is_nested(),
                   "dropout of a nested or sparse tensor is not supported");
  at::Tensor out = at::empty_like(residual.defined() ? residual : x, x.options().dtype(out_type));
  const int64_t n = x.numel();
  if (n == 0) return out;  // nor will the backward pass read `used`
  TORCH_CHECK(!x._is_zerotensor() && !(residual.defined() && residual._is_zerotensor()),
              "dropout of a tensor without storage");
  tpi_dropout_args a{};
  a.x = address(x);
  a.residual = residual.defined() ? address(residual) : 0;
  a.out = address(out);
  a.state = mask.state.defined() ? address(mask.state) : 0;
  a.used = used.defined() ? address(used) : 0;
  a.seed = mask.seed;
  a.draw = mask.number;
  a.first = mask.first;
  a.threshold = mask.threshold;
  a.scale = mask.scale;
  a.in_type = type_of(x.scalar_type());
  a.out_type = type_of(out_type);
  if (mask.strides.empty() && x.is_contiguous() && out.is_contiguous() &&
      (!residual.defined() || residual.is_contiguous())) {
    a.ndim = 1;
    a.sizes[0] = n;
    a.sx[0] = a.sr[0] = a.so[0] = a.si[0] = 1;
  } else {
    std::vector<int64_t> index = mask.strides;
    if (index.empty()) {
      index.resize(x.dim());
      int64_t step = 1;
      for (int64_t d = x.dim() - 1; d >= 0; --d) {
        index[d] = step;
        step *= x.size(d);
      }
    }
    const int64_t* const strides[4] = {x.strides().data(),
                                       residual.defined() ? residual.strides().data()
                                                          : out.strides().data(),
                                       out.strides().data(), index.data()};
    a.ndim = merge(x.sizes(), strides, a);
  }
  if (x.is_cpu()) {
    dropout_host(a);
    return out;
  }
  const c10::DeviceGuard guard(x.device());
  hip_check(hip_api().dropout(&a, current_stream(x.device().index())), "dropout");
  return out;
}

at::Tensor run(const at::Tensor& x, const at::Tensor& residual, at::ScalarType out_type,
               const c10::intrusive_ptr<Mask>& mask);

// The gradient of a dropped element is 0, of a kept one the scale times the output's: the
// operator itself, applied to the gradient (so it can be differentiated again).
struct Dropout : torch::autograd::Function<Dropout> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                            const std::optional<at::Tensor>& added, int64_t out_type,
                            const c10::intrusive_ptr<Mask>& mask) {
    const at::Tensor residual = added.value_or(at::Tensor());
    at::Tensor used;
    c10::intrusive_ptr<Mask> again = mask;
    if (mask->state.defined() && x.requires_grad()) {
      // the state may have moved on by the time the backward pass runs
      used = at::empty({2}, mask->state.options());
      again = c10::make_intrusive<Mask>(*mask);
      again->state = used;
      again->number = 0;
    }
    ctx->saved_data["mask"] = c10::IValue::make_capsule(again);
    ctx->saved_data["type"] = (int64_t)x.scalar_type();
    ctx->saved_data["residual"] = residual.defined() && residual.requires_grad();
    ctx->saved_data["x"] = x.requires_grad();
    return dropout_pass(x, residual, (at::ScalarType)out_type, *mask, used);
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const at::Tensor& grad = grads[0];
    at::Tensor dx, dr;
    if (grad.defined() && ctx->saved_data["x"].toBool())
      dx = run(grad.resolve_neg(), at::Tensor(), (at::ScalarType)ctx->saved_data["type"].toInt(),
               c10::static_intrusive_pointer_cast<Mask>(ctx->saved_data["mask"].toCapsule()));
    if (ctx->saved_data["residual"].toBool()) dr = grad;
    return {dx, dr, at::Tensor(), at::Tensor()};
  }
};

at::Tensor run(const at::Tensor& x, const at::Tensor& residual, at::ScalarType out_type,
               const c10::intrusive_ptr<Mask>& mask) {
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || (residual.defined() && residual.requires_grad())))
    return Dropout::apply(x, residual.defined() ? std::optional<at::Tensor>(residual) : std::nullopt,
                          (int64_t)out_type, mask);
  return dropout_pass(x, residual, out_type, *mask, at::Tensor());
}

at::Tensor dropout(const at::Tensor& x, const std::optional<at::Tensor>& residual,
                   uint64_t threshold, double scale, uint64_t seed, uint64_t number,
                   const std::optional<at::Tensor>& state, uint64_t first,
                   std::vector<int64_t> strides) {
  auto mask = c10::make_intrusive<Mask>();
  mask->seed = seed;
  mask->number = number;
  mask->first = first;
  mask->threshold = threshold;
  mask->scale = (float)scale;
  mask->strides = std::move(strides);
  if (state) mask->state = *state;
  // views that are negated lazily (the imaginary part of a conjugate) are written out
  return run(x.resolve_neg(), residual ? residual->resolve_neg() : at::Tensor(),
             residual ? residual->scalar_type() : x.scalar_type(), mask);
}

}  // namespace

void bind_dropout(py::module_& m) {
  m.def("dropout", &dropout, py::call_guard<py::gil_scoped_release>());
}

}  // namespace tpi
