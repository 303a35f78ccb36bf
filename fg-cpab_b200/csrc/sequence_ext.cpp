// The sequence-network operators in C++ over the C ABI of libcpab_b200: the
// autograd nodes of gated_scan and rms_norm, and the calls without a gradient
// (gated_scan_step, rms_norm_quantized, adamw).  Part of _cpab_ext, for the
// reason torch_ext.cpp gives: a step's host time.  The Python twins
// (cpab/pytorch/recurrence.py, cpab/pytorch/norm.py, cpab/_native.py) issue the
// same C ABI calls with the same arguments.
#include "ext_common.h"

namespace {

// ---- gated_scan --------------------------------------------------------------

// x and gate as the kernels read them: [B, T, D] with the channels adjacent.
// Without a gate, x is [B, T, 2 D], the inputs' channels before the gates'.
struct ScanInput {
  Tensor x, gate;   // as given, channels adjacent
  int64_t B, T, D;
  int dtype;
  const void *xp, *gp;
  int64_t xb, xt, gb, gt;
};

ScanInput scan_input(const Tensor &x, const Tensor &gate) {
  ScanInput s;
  s.dtype = dtype_of(x, "x");
  s.x = channels_adjacent(x);
  s.B = x.size(0), s.T = x.size(1);
  const int64_t e = x.element_size();
  s.xp = s.x.const_data_ptr(), s.xb = s.x.stride(0), s.xt = s.x.stride(1);
  if (gate.defined()) {
    s.D = x.size(2);
    s.gate = channels_adjacent(gate);
    s.gp = s.gate.const_data_ptr(), s.gb = s.gate.stride(0), s.gt = s.gate.stride(1);
  } else {
    s.D = x.size(2) / 2;
    s.gp = static_cast<const char *>(s.xp) + s.D * e, s.gb = s.xb, s.gt = s.xt;
  }
  return s;
}

void check_scan(const Tensor &x, const Tensor &gate, const Tensor &h0, const Tensor &lengths) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (no CPU path)");
  dtype_of(x, "x");
  TORCH_CHECK_VALUE(x.dim() == 3, "x must be [B, T, D], got ", x.sizes());
  if (gate.defined()) require(gate, x, x.scalar_type(), x.sizes(), "gate");
  else TORCH_CHECK_VALUE(x.size(2) % 2 == 0, "x without a gate must be [B, T, 2 D], got ", x.sizes());
  const int64_t D = gate.defined() ? x.size(2) : x.size(2) / 2;
  if (h0.defined()) require(h0, x, at::kFloat, {x.size(0), D}, "h0");
  if (lengths.defined()) require(lengths, x, at::kInt, {x.size(0)}, "lengths");
}

Tensor scan_workspace(const ScanInput &s) {
  return at::empty({cpab_b200_gated_scan_workspace(s.dtype, s.B, s.T, s.D)}, s.x.options().dtype(at::kFloat));
}

struct ScanOutput {
  Tensor h, last, states;
};

ScanOutput scan_forward(const ScanInput &s, const Tensor &h0, const Tensor &lengths, bool keep) {
  ScanOutput o;
  const auto f32 = s.x.options().dtype(at::kFloat);
  o.h = at::empty({s.B, s.T, s.D}, s.x.options());
  o.last = at::empty({s.B, s.D}, f32);
  if (keep) {
    const int64_t c = cpab_b200_gated_scan_chunk();
    o.states = at::empty({s.B, (s.T + c - 1) / c, s.D}, f32);
  }
  const Tensor start = h0.defined() ? h0.contiguous() : h0;
  const Tensor len = lengths.defined() ? lengths.contiguous() : lengths;
  const Tensor work = scan_workspace(s);
  check(cpab_b200_gated_scan(s.dtype, s.xp, s.xb, s.xt, s.gp, s.gb, s.gt, s.B, s.T, s.D,
                             static_cast<const int32_t *>(ptr(len)), fptr(start), ptr_mut(o.h),
                             fptr_mut(o.last), fptr_mut(o.states), fptr_mut(work), stream_of(s.x)));
  return o;
}

class ScanFunction : public torch::autograd::Function<ScanFunction> {
 public:
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const MaybeTensor &gate_,
                               const MaybeTensor &h0_, const MaybeTensor &lengths_) {
    const Tensor gate = given(gate_), h0 = given(h0_), lengths = given(lengths_);
    const c10::cuda::CUDAGuard guard(x.device());
    const ScanInput s = scan_input(x, gate);
    const ScanOutput o = scan_forward(s, h0, lengths, true);
    ctx->save_for_backward({s.x, s.gate, o.states, lengths});
    // (edges are counted over the given tensors only, so not by position here)
    ctx->saved_data["want_h0"] = h0.defined() && h0.requires_grad();
    ctx->set_materialize_grads(false);
    return {o.h, o.last};
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    once("gated_scan");
    const auto saved = ctx->get_saved_variables();
    const Tensor x = saved[0], gate = saved[1], states = saved[2], lengths = saved[3];
    if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const c10::cuda::CUDAGuard guard(x.device());
    const ScanInput s = scan_input(x, gate);
    const Tensor dh = grads[0].defined() ? grads[0].contiguous() : Tensor();
    const Tensor dlast = grads[1].defined() ? grads[1].contiguous() : Tensor();
    const Tensor len = lengths.defined() ? lengths.contiguous() : lengths;
    const Tensor dx = at::empty({s.B, s.T, gate.defined() ? s.D : 2 * s.D}, x.options());
    const Tensor dgate = gate.defined() ? at::empty({s.B, s.T, s.D}, x.options()) : Tensor();
    void *dgp = gate.defined() ? ptr_mut(dgate)
                               : static_cast<char *>(ptr_mut(dx)) + s.D * x.element_size();
    const Tensor &dg = gate.defined() ? dgate : dx;
    const Tensor dh0 = ctx->saved_data["want_h0"].toBool()
                           ? at::empty({s.B, s.D}, x.options().dtype(at::kFloat)) : Tensor();
    const Tensor work = scan_workspace(s);
    check(cpab_b200_gated_scan_backward(
        s.dtype, s.xp, s.xb, s.xt, s.gp, s.gb, s.gt, s.B, s.T, s.D,
        static_cast<const int32_t *>(ptr(len)), fptr(states), ptr(dh), fptr(dlast), ptr_mut(dx),
        dx.stride(0), dx.stride(1), dgp, dg.stride(0), dg.stride(1), fptr_mut(dh0), fptr_mut(work), stream_of(x)));
    return {dx, dgate, dh0, Tensor()};
  }
};

std::tuple<Tensor, Tensor> gated_scan(const Tensor &x, const MaybeTensor &gate_, const MaybeTensor &h0_,
                                      const MaybeTensor &lengths_) {
  const Tensor gate = given(gate_), h0 = given(h0_), lengths = given(lengths_);
  check_scan(x, gate, h0, lengths);
  if (needs_grad({&x, &gate, &h0})) {
    const variable_list r = ScanFunction::apply(x, gate_, h0_, lengths_);
    return {r[0], r[1]};
  }
  const c10::cuda::CUDAGuard guard(x.device());
  const ScanOutput o = scan_forward(scan_input(x, gate), h0, lengths, false);
  return {o.h, o.last};
}

Tensor gated_scan_step(const Tensor &x, const MaybeTensor &gate_, const Tensor &state,
                       const MaybeTensor &slots_) {
  const Tensor gate = given(gate_), slots = given(slots_);
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (no CPU path)");
  TORCH_CHECK(!has_tangent({&x, &gate, &state}), "gated_scan_step has no gradient, of forward mode neither");
  const int dtype = dtype_of(x, "x");
  TORCH_CHECK_VALUE(x.dim() == 2, "x must be [B, D], got ", x.sizes());
  if (gate.defined()) require(gate, x, x.scalar_type(), x.sizes(), "gate");
  else TORCH_CHECK_VALUE(x.size(1) % 2 == 0, "x without a gate must be [B, 2 D], got ", x.sizes());
  const int64_t B = x.size(0), D = gate.defined() ? x.size(1) : x.size(1) / 2;
  TORCH_CHECK_VALUE(state.dim() == 2 && (slots.defined() || state.size(0) == B),
                    "state must be [rows, D] (rows = B without slots), got ", state.sizes());
  require(state, x, at::kFloat, {state.size(0), D}, "state");
  TORCH_CHECK_VALUE(state.is_contiguous(), "state must be contiguous (it is updated in place)");
  if (slots.defined()) require(slots, x, at::kInt, {B}, "slots");
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor xc = channels_adjacent(x), gc = gate.defined() ? channels_adjacent(gate) : gate;
  const Tensor sl = slots.defined() ? slots.contiguous() : slots;
  const Tensor h = at::empty({B, D}, x.options());
  written(state);
  const void *gp = gate.defined() ? ptr(gc) : static_cast<const char *>(ptr(xc)) + D * x.element_size();
  check(cpab_b200_gated_scan_step(dtype, ptr(xc), xc.stride(0), gp, gate.defined() ? gc.stride(0) : xc.stride(0),
                                  B, D, static_cast<const int32_t *>(ptr(sl)), state.size(0), fptr_mut(state),
                                  ptr_mut(h), stream_of(x)));
  return h;
}

// ---- rms_norm ------------------------------------------------------------------

void check_norm(const Tensor &x, const Tensor &weight, const Tensor &residual) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (no CPU path)");
  dtype_of(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x must be [..., D] with D > 0, got ", x.sizes());
  TORCH_CHECK_TYPE(weight.scalar_type() == at::kFloat || weight.scalar_type() == x.scalar_type(),
                   "weight must be float32 or of x's type, got ", weight.scalar_type());
  require(weight, x, weight.scalar_type(), {x.size(-1)}, "weight");
  if (residual.defined()) {
    TORCH_CHECK_TYPE(residual.scalar_type() == at::kFloat || residual.scalar_type() == x.scalar_type(),
                     "residual must be float32 or of x's type, got ", residual.scalar_type());
    require(residual, x, residual.scalar_type(), x.sizes(), "residual");
  }
}

struct NormOutput {
  Tensor y, sum, rstd;
};

NormOutput norm_forward(const Tensor &x, const Tensor &weight, const Tensor &residual, double eps, bool keep) {
  const Tensor xr = rows_of(x), rr = residual.defined() ? rows_of(residual) : Tensor();
  const Tensor w = weight.contiguous();
  const Tensor &stream = residual.defined() ? residual : x;
  NormOutput o;
  o.y = at::empty(x.sizes(), x.options());
  if (residual.defined()) o.sum = at::empty(x.sizes(), residual.options());
  if (keep) o.rstd = at::empty({xr.size(0)}, x.options().dtype(at::kFloat));
  check(cpab_b200_rms_norm(dtype_of(x, "x"), dtype_of(stream, "residual"), dtype_of(w, "weight"), ptr(xr),
                           xr.stride(0), ptr(rr), rr.defined() ? rr.stride(0) : 0, ptr(w), xr.size(0),
                           xr.size(1), (float)eps, ptr_mut(o.y), ptr_mut(o.sum), fptr_mut(o.rstd),
                           stream_of(x)));
  return o;
}

class NormFunction : public torch::autograd::Function<NormFunction> {
 public:
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight,
                               const MaybeTensor &residual_, double eps) {
    const Tensor residual = given(residual_);
    const c10::cuda::CUDAGuard guard(x.device());
    const NormOutput o = norm_forward(x, weight, residual, eps, true);
    ctx->save_for_backward({residual.defined() ? o.sum : x, weight, o.rstd});
    ctx->saved_data["x_type"] = (int64_t)x.scalar_type();
    ctx->set_materialize_grads(false);
    if (residual.defined()) return {o.y, o.sum};
    return {o.y};
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    once("rms_norm");
    const auto saved = ctx->get_saved_variables();
    const Tensor sum = saved[0], weight = saved[1], rstd = saved[2];
    const auto x_type = static_cast<at::ScalarType>(ctx->saved_data["x_type"].toInt());
    const bool residual = grads.size() > 1;
    const Tensor gs = residual && grads[1].defined() ? grads[1].contiguous() : Tensor();
    if (!grads[0].defined()) {  // only the sum is used
      if (!gs.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
      return {gs.to(x_type), Tensor(), gs, Tensor()};
    }
    const c10::cuda::CUDAGuard guard(sum.device());
    const Tensor gy = grads[0].contiguous(), rows = rows_of(sum), w = weight.contiguous();
    const int64_t n = rows.size(0), D = rows.size(1);
    const bool mixed = sum.scalar_type() != x_type;
    const Tensor dx = at::empty(sum.sizes(), sum.options().dtype(x_type));
    const Tensor dres = mixed ? at::empty(sum.sizes(), sum.options()) : Tensor();
    const Tensor dw = ctx->needs_input_grad(1) ? at::empty(weight.sizes(), weight.options()) : Tensor();
    const int dt = dtype_of(dx, "x");
    const Tensor work = dw.defined()
        ? at::empty({cpab_b200_rms_norm_workspace(dt, n, D)}, sum.options().dtype(at::kFloat)) : Tensor();
    check(cpab_b200_rms_norm_backward(dt, dtype_of(sum, "residual"), dtype_of(w, "weight"), ptr(rows),
                                      rows.stride(0), ptr(w), fptr(rstd), n, D, ptr(gy), ptr(gs), ptr_mut(dx),
                                      ptr_mut(dres), fptr_mut(work), ptr_mut(dw), stream_of(sum)));
    return {dx, dw, residual ? (mixed ? dres : dx) : Tensor(), Tensor()};
  }
};

std::vector<Tensor> rms_norm(const Tensor &x, const Tensor &weight, const MaybeTensor &residual_,
                             double eps) {
  const Tensor residual = given(residual_);
  check_norm(x, weight, residual);
  if (needs_grad({&x, &weight, &residual})) return NormFunction::apply(x, weight, residual_, eps);
  const c10::cuda::CUDAGuard guard(x.device());
  const NormOutput o = norm_forward(x, weight, residual, eps, false);
  if (residual.defined()) return {o.y, o.sum};
  return {o.y};
}

std::vector<Tensor> rms_norm_quantized(const Tensor &x, const Tensor &weight, const MaybeTensor &residual_,
                                       double eps) {
  const Tensor residual = given(residual_);
  check_norm(x, weight, residual);
  TORCH_CHECK(!has_tangent({&x, &weight, &residual}),
              "rms_norm_quantized has no gradient, of forward mode neither");
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor xr = rows_of(x), rr = residual.defined() ? rows_of(residual) : Tensor();
  const Tensor w = weight.contiguous();
  const Tensor &stream = residual.defined() ? residual : x;
  const Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
  const Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  const Tensor sum = residual.defined() ? at::empty(x.sizes(), residual.options()) : Tensor();
  check(cpab_b200_rms_norm_quantized(dtype_of(x, "x"), dtype_of(stream, "residual"), dtype_of(w, "weight"),
                                     ptr(xr), xr.stride(0), ptr(rr), rr.defined() ? rr.stride(0) : 0, ptr(w),
                                     xr.size(0), xr.size(1), (float)eps, static_cast<uint8_t *>(ptr_mut(q)),
                                     fptr_mut(scale), ptr_mut(sum), stream_of(x)));
  if (residual.defined()) return {q, scale, sum};
  return {q, scale};
}

// ---- adamw ---------------------------------------------------------------------

// counts[g] tensors of group g one after another in the lists; hyper holds a
// group's (lr, beta1, beta2, eps, weight_decay); lr_tensors a group's learning
// rate on the device (None: hyper's).  scales is empty where every state has
// 32 bits.
void adamw(const pybind11::list &params, const pybind11::list &grads, const pybind11::list &exp_avgs,
           const pybind11::list &exp_avg_sqs, const pybind11::list &scales, const pybind11::list &steps,
           const std::vector<int64_t> &counts, const std::vector<double> &hyper,
           const std::vector<MaybeTensor> &lr_tensors, int64_t seed, const Tensor &workspace) {
  const size_t n = params.size();
  TORCH_CHECK_VALUE(grads.size() == n && exp_avgs.size() == n && exp_avg_sqs.size() == n && steps.size() == n &&
                        (scales.empty() || scales.size() == n),
                    "adamw: lists of different lengths");
  if (n == 0) return;
  const at::Device device = item(params, 0, "adamw: parameter")->device();
  TORCH_CHECK(device.is_cuda(), "params must be CUDA tensors (no CPU path)");
  for (const MaybeTensor &lr : lr_tensors)
    TORCH_CHECK(!lr.has_value() || (lr->device() == device && lr->scalar_type() == at::kFloat && lr->numel() == 1),
                "adamw: a learning rate on the device must be one float32 on the parameters' device, ", device);
  const c10::cuda::CUDAGuard guard(device);
  std::vector<cpab_adamw_tensor> list(n);
  std::vector<Tensor> copies;  // gradients laid out as their parameters
  size_t k = 0;
  for (size_t g = 0; g < counts.size(); ++g) {
    for (int64_t i = 0; i < counts[g]; ++i, ++k) {
      const Tensor &p = *item(params, k, "adamw: parameter"), &m = *item(exp_avgs, k, "adamw: first moment");
      const Tensor &v = *item(exp_avg_sqs, k, "adamw: second moment"), &step = *item(steps, k, "adamw: step");
      const Tensor *grad = item(grads, k, "adamw: gradient");
      const bool eight = m.scalar_type() == at::kFloat8_e4m3fn;
      TORCH_CHECK(p.device() == device && grad->device() == device && m.device() == device &&
                      v.device() == device && step.device() == device,
                  "adamw: tensor ", k, ": all tensors must be on one device");
      TORCH_CHECK_TYPE(grad->scalar_type() == p.scalar_type(), "adamw: tensor ", k, ": gradient of type ",
                       grad->scalar_type(), " for a parameter of type ", p.scalar_type());
      TORCH_CHECK_TYPE(v.scalar_type() == m.scalar_type() && (eight || m.scalar_type() == at::kFloat),
                       "adamw: tensor ", k, ": states must be float32, or both float8_e4m3fn");
      TORCH_CHECK_TYPE(step.scalar_type() == at::kFloat && step.numel() == 1,
                       "adamw: tensor ", k, ": step must be one float32");
      TORCH_CHECK_VALUE(grad->sizes() == p.sizes() && m.sizes() == p.sizes() && v.sizes() == p.sizes(),
                        "adamw: tensor ", k, ": parameter, gradient and states must have one shape");
      const bool plain = p.is_contiguous();
      TORCH_CHECK_VALUE(plain ? m.is_contiguous() && v.is_contiguous()
                              : p.is_non_overlapping_and_dense() && m.strides() == p.strides() &&
                                    v.strides() == p.strides(),
                        "adamw: tensor ", k, ": parameter and states must be dense and laid out alike");
      if (!(plain ? grad->is_contiguous() : grad->strides() == p.strides())) {
        copies.push_back(at::empty_like(p));
        copies.back().copy_(*grad);
      }
      const bool copied = !(plain ? grad->is_contiguous() : grad->strides() == p.strides());
      float *sc = nullptr;
      if (eight) {
        const int64_t blocks = (p.numel() + 255) / 256;
        const Tensor *t = scales.empty() ? nullptr : item(scales, k, "adamw: scales", true);
        TORCH_CHECK_VALUE(t != nullptr && t->device() == device && t->scalar_type() == at::kFloat &&
                              t->is_contiguous() && t->numel() == 2 * blocks,
                          "adamw: tensor ", k, ": 8-bit states need float32 scales [", blocks, ", 2]");
        sc = fptr_mut(*t);
        written(*t);
      }
      for (const Tensor *t : {&p, &m, &v, &step}) written(*t);
      cpab_adamw_tensor &t = list[k];
      t.param = ptr_mut(p), t.grad = ptr(copied ? copies.back() : *grad), t.exp_avg = ptr_mut(m);
      t.exp_avg_sq = ptr_mut(v), t.scales = sc, t.step = fptr_mut(step), t.numel = p.numel();
      t.lr_device = lr_tensors[g].has_value() ? fptr(*lr_tensors[g]) : nullptr;
      t.dtype = dtype_of(p, "a parameter"), t.state_bits = eight ? 8 : 32;
      t.lr = hyper[5 * g], t.beta1 = hyper[5 * g + 1], t.beta2 = hyper[5 * g + 2], t.eps = hyper[5 * g + 3];
      t.weight_decay = hyper[5 * g + 4];
    }
  }
  check(cpab_b200_adamw(list.data(), (int)n, (uint32_t)seed, static_cast<int32_t *>(ptr_mut(workspace)),
                        stream_of(*item(params, 0, "adamw: parameter"))));
}

}  // namespace

void bind_sequence(pybind11::module &m) {
  m.def("gated_scan", &gated_scan, "x, gate or None, h0 or None, lengths or None -> h, last state");
  m.def("gated_scan_step", &gated_scan_step, "x, gate or None, state (in place), slots or None -> h");
  m.def("rms_norm", &rms_norm, "x, weight, residual or None, eps -> [y] or [y, sum]");
  m.def("rms_norm_quantized", &rms_norm_quantized, "x, weight, residual or None, eps -> [q, scale(, sum)]");
  m.def("adamw", &adamw,
        "params, grads, exp_avgs, exp_avg_sqs, scales, steps, counts, hyper, lr tensors, seed, workspace");
}
