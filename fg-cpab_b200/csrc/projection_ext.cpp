// 8-bit projections and orthogonalised steps in C++ over the C ABI of
// libcpab_b200: quantize_blocks, matmul_quantized, the autograd node of
// linear_quantized, orthogonalize and muon.  Part of _cpab_ext, for the reason
// torch_ext.cpp gives: a call's host time.  The Python twins
// (cpab/pytorch/projection.py, cpab/_native.py) issue the same C ABI calls with
// the same arguments.
#include "ext_common.h"

namespace {

constexpr at::ScalarType kCodes = at::kFloat8_e4m3fn, kScales = at::kFloat8_e8m0fnu;

int64_t round_to(int64_t n, int64_t unit) { return (n + unit - 1) / unit * unit; }

// ---- codes ---------------------------------------------------------------------

// Codes [*lead, K] whose rows begin on multiples of 16 bytes, and scales
// [*lead, ceil(K / 128)] whose rows begin on multiples of 4.
struct Codes {
  Tensor q, scale;
  int64_t q_row = 0, scale_row = 0;
};

Tensor padded(at::IntArrayRef lead, int64_t n, int64_t pitch, at::ScalarType type, const Tensor &like) {
  std::vector<int64_t> shape(lead.begin(), lead.end());
  shape.push_back(pitch);
  const Tensor t = at::empty(shape, like.options().dtype(type));
  return n == pitch ? t : t.narrow(-1, 0, n);
}

Codes new_codes(at::IntArrayRef lead, int64_t K, const Tensor &like) {
  Codes c;
  const int64_t blocks = (K + 127) / 128;
  c.q_row = round_to(K, 16), c.scale_row = round_to(blocks, 4);
  c.q = padded(lead, K, c.q_row, kCodes, like);
  c.scale = padded(lead, blocks, c.scale_row, kScales, like);
  return c;
}

void check_quantize(const Tensor &x) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (no CPU path)");
  dtype_of(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x must be [..., K] with K > 0, got ", x.sizes());
}

// Codes as the library takes them: a place in somebody's memory.
struct Place {
  uint8_t *q = nullptr, *scale = nullptr;
  int64_t q_row = 0, scale_row = 0;
};
Place place_of(const Codes &c) {
  return {static_cast<uint8_t *>(ptr_mut(c.q)), static_cast<uint8_t *>(ptr_mut(c.scale)), c.q_row, c.scale_row};
}

// Codes of several matrices in one tensor of bytes.
class Slab {
 public:
  // A place for R rows of K codes, from a multiple of 256 bytes; filled in by allocate().
  size_t add(int64_t R, int64_t K) {
    Place p;
    p.q_row = round_to(K, 16), p.scale_row = round_to((K + 127) / 128, 4);
    starts_.push_back({bytes_, bytes_ + round_to(R * p.q_row, 256)});
    places_.push_back(p);
    bytes_ = starts_.back().second + round_to(R * p.scale_row, 256);
    return places_.size() - 1;
  }
  void allocate(const Tensor &like) { place(at::empty({bytes_}, like.options().dtype(at::kByte))); }
  void place(const Tensor &bytes) {
    memory = bytes;
    auto *base = static_cast<uint8_t *>(ptr_mut(memory));
    for (size_t i = 0; i < places_.size(); ++i)
      places_[i].q = base + starts_[i].first, places_[i].scale = base + starts_[i].second;
  }
  const Place &operator[](size_t i) const { return places_[i]; }
  Tensor memory;

 private:
  std::vector<Place> places_;
  std::vector<std::pair<int64_t, int64_t>> starts_;
  int64_t bytes_ = 0;
};

// x's codes by rows and of its transpose (null: not wanted), and the sums of its columns.
Tensor quantize(const Tensor &x, const Place *rows, const Place *turned, const at::ScalarType *sum_type) {
  const Tensor xr = rows_of(x);
  const int64_t R = xr.size(0), K = xr.size(1);
  Tensor sums;
  Tensor work;
  if (sum_type != nullptr) {
    sums = at::empty({K}, x.options().dtype(*sum_type));
    work = at::empty({cpab_b200_quantize_blocks_workspace(R, K)}, x.options().dtype(at::kFloat));
  }
  const Place none;
  const Place &r = rows != nullptr ? *rows : none, &t = turned != nullptr ? *turned : none;
  check(cpab_b200_quantize_blocks(dtype_of(x, "x"), ptr(xr), xr.stride(0), R, K, r.q, r.q_row, r.scale, r.scale_row, t.q,
                                  t.q_row, t.scale, t.scale_row, sums.defined() ? dtype_of(sums, "bias") : CPAB_F32,
                                  ptr_mut(sums), fptr_mut(work), stream_of(x)));
  return sums;
}

std::vector<Tensor> quantize_blocks(const Tensor &x, bool transposed) {
  check_quantize(x);
  TORCH_CHECK(!has_tangent({&x}), "quantize_blocks has no gradient, of forward mode neither");
  TORCH_CHECK_VALUE(!transposed || x.dim() == 2, "x must be [R, K] for its transpose, got ", x.sizes());
  const c10::cuda::CUDAGuard guard(x.device());
  const Codes rows = new_codes(x.sizes().slice(0, x.dim() - 1), x.size(-1), x);
  const Place r = place_of(rows);
  if (!transposed) {
    quantize(x, &r, nullptr, nullptr);
    return {rows.q, rows.scale};
  }
  const Codes turned = new_codes({x.size(1)}, x.size(0), x);
  const Place t = place_of(turned);
  quantize(x, &r, &t, nullptr);
  return {rows.q, rows.scale, turned.q, turned.scale};
}

// ---- products --------------------------------------------------------------------

// Codes [..., K] with their scales as the library reads them.
struct Operand {
  Tensor q, scale;
  int64_t rows, K;
  cpab_quantized c;
  bool loose = false;  // codes whose rows do not begin on multiples of 16 bytes
};

Operand operand(const Tensor &q, const Tensor &scale, const char *name) {
  TORCH_CHECK_TYPE(q.scalar_type() == kCodes, name, " must be float8_e4m3fn, got ", q.scalar_type());
  TORCH_CHECK_VALUE(q.dim() >= 1 && q.size(-1) > 0, name, " must be [..., K] with K > 0, got ", q.sizes());
  const bool per_row = scale.scalar_type() == at::kFloat;
  TORCH_CHECK_TYPE(per_row || scale.scalar_type() == kScales, name,
                   "'s scale must be float8_e8m0fnu (for each 128 codes) or float32 (for each row), got ",
                   scale.scalar_type());
  Operand o;
  o.K = q.size(-1);
  const int64_t blocks = (o.K + 127) / 128;
  std::vector<int64_t> want(q.sizes().begin(), q.sizes().end() - 1);
  if (!per_row) want.push_back(blocks);
  TORCH_CHECK_VALUE(scale.sizes() == at::IntArrayRef(want), name, "'s scale must have shape ", want, ", got ",
                    scale.sizes());
  o.q = q.dim() == 2 ? q : q.reshape({-1, o.K});
  o.rows = o.q.size(0);
  if (o.K > 1 && o.q.stride(1) != 1) {
    const Tensor copy = padded({o.rows}, o.K, round_to(o.K, 16), kCodes, q);
    copy.copy_(o.q);
    o.q = copy;
  }
  o.loose = (o.rows > 1 && (o.q.stride(0) % 16 != 0 || o.q.stride(0) < o.K)) ||
            reinterpret_cast<uintptr_t>(o.q.const_data_ptr()) % 16 != 0;
  int64_t scale_row = 0;
  if (per_row) {
    o.scale = scale.reshape({-1}).contiguous();
  } else {
    o.scale = scale.dim() == 2 ? scale : scale.reshape({-1, blocks});
    if ((blocks > 1 && o.scale.stride(1) != 1) || (o.rows > 1 && o.scale.stride(0) < blocks))
      o.scale = o.scale.contiguous();
    scale_row = o.rows > 1 ? o.scale.stride(0) : round_to(blocks, 4);
  }
  o.c = {static_cast<const uint8_t *>(ptr(o.q)), o.rows > 1 ? o.q.stride(0) : round_to(o.K, 16), ptr(o.scale), scale_row};
  return o;
}

// Copies loose codes to where the products can read them, both operands' at once.
void lay_out(Operand &x, Operand &w) {
  const uint8_t *src[2];
  uint8_t *dst[2];
  int64_t row[2], rows[2], bytes = 0;
  Operand *which[2];
  int n = 0;
  const int64_t pitch = round_to(x.K, 16);
  for (Operand *o : {&x, &w})
    if (o->loose) which[n] = o, src[n] = o->c.codes, row[n] = o->q.stride(0), rows[n] = o->rows, bytes += pitch * o->rows, ++n;
  if (n == 0) return;
  const Tensor copy = at::empty({bytes}, x.q.options().dtype(at::kByte));
  auto *at = static_cast<uint8_t *>(ptr_mut(copy));
  for (int i = 0; i < n; ++i) {
    dst[i] = at, which[i]->c.codes = at, which[i]->c.row = pitch, which[i]->q = copy;
    at += pitch * rows[i];
  }
  check(cpab_b200_lay_out_codes(n, src, row, rows, dst, x.K, stream_of(x.q)));
}

Operand operand(const Place &p, int64_t rows, int64_t K) {
  Operand o;
  o.rows = rows, o.K = K;
  o.c = {p.q, p.q_row, p.scale, p.scale_row};
  return o;
}

Tensor product(const Operand &x, const Operand &w, const Tensor &bias, at::IntArrayRef lead, at::ScalarType type,
               const Tensor &like) {
  std::vector<int64_t> shape(lead.begin(), lead.end());
  shape.push_back(w.rows);
  const Tensor y = at::empty(shape, like.options().dtype(type));
  const int dt = dtype_of(y, "dtype");
  const int64_t floats = cpab_b200_matmul_quantized_workspace(x.rows, w.rows, x.K);
  const Tensor work = floats > 0 ? at::empty({floats}, like.options().dtype(at::kFloat)) : Tensor();
  check(cpab_b200_matmul_quantized(dt, &x.c, &w.c, x.rows, w.rows, x.K, bias.defined() ? dtype_of(bias, "bias") : dt,
                                   ptr(bias), ptr_mut(y), w.rows, fptr_mut(work), stream_of(like)));
  return y;
}

Tensor matmul_quantized(const Tensor &q, const Tensor &scale, const Tensor &weight, const Tensor &weight_scale,
                        const MaybeTensor &bias_, at::ScalarType type) {
  const Tensor bias = given(bias_);
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor (no CPU path)");
  TORCH_CHECK_TYPE(type == at::kFloat || type == at::kHalf || type == at::kBFloat16,
                   "dtype must be float32, float16 or bfloat16, got ", type);
  TORCH_CHECK_VALUE(weight.dim() == 2, "weight must be [N, K], got ", weight.sizes());
  TORCH_CHECK(weight.device() == q.device(), "weight is on ", weight.device(), ", q on ", q.device());
  for (const Tensor *t : {&scale, &weight_scale})
    TORCH_CHECK(t->device() == q.device(), "a scale is on ", t->device(), ", the codes on ", q.device());
  TORCH_CHECK(!has_tangent({&scale, &weight_scale, &bias}), "matmul_quantized has no gradient, of forward mode neither");
  const c10::cuda::CUDAGuard guard(q.device());
  Operand x = operand(q, scale, "q"), w = operand(weight, weight_scale, "weight");
  TORCH_CHECK_VALUE(w.K == x.K, "weight must be [N, ", x.K, "], got ", weight.sizes());
  Tensor b;
  if (bias.defined()) {
    TORCH_CHECK_TYPE(bias.scalar_type() == at::kFloat || bias.scalar_type() == type,
                     "bias must be float32 or of the result's type, got ", bias.scalar_type());
    require(bias, q, bias.scalar_type(), {w.rows}, "bias");
    b = bias.contiguous();
  }
  const Tensor kept_q = x.q, kept_w = w.q;  // (until their copies are asked for)
  lay_out(x, w);
  return product(x, w, b, q.sizes().slice(0, q.dim() - 1), type, q);
}

// ---- linear_quantized ---------------------------------------------------------------

void check_linear(const Tensor &x, const Tensor &weight, const Tensor &bias) {
  check_quantize(x);
  TORCH_CHECK_VALUE(weight.dim() == 2, "weight must be [N, K], got ", weight.sizes());
  TORCH_CHECK_TYPE(weight.scalar_type() == at::kFloat || weight.scalar_type() == x.scalar_type(),
                   "weight must be float32 or of x's type, got ", weight.scalar_type());
  require(weight, x, weight.scalar_type(), {weight.size(0), x.size(-1)}, "weight");
  if (bias.defined()) {
    TORCH_CHECK_TYPE(bias.scalar_type() == at::kFloat || bias.scalar_type() == x.scalar_type(),
                     "bias must be float32 or of x's type, got ", bias.scalar_type());
    require(bias, x, bias.scalar_type(), {weight.size(0)}, "bias");
  }
}

// What the backward keeps, in one tensor: the codes of x's transpose (for the
// weight's gradient) and of the weight's (for x's).
struct Kept {
  Slab slab;
  size_t x = 0, w = 0;
  Kept(int64_t M, int64_t N, int64_t K, bool keep_x, bool keep_w) {
    if (keep_x) x = slab.add(K, M);
    if (keep_w) w = slab.add(K, N);
  }
};

Tensor linear_forward(const Tensor &x, const Tensor &weight, const Tensor &bias, bool keep_x, bool keep_w, Tensor *kept) {
  const int64_t K = x.size(-1), N = weight.size(0), M = x.numel() / K;
  Slab s;
  const size_t xq = s.add(M, K), wq = s.add(N, K);
  s.allocate(x);
  Kept k(M, N, K, keep_x, keep_w);
  if (keep_x || keep_w) k.slab.allocate(x);
  *kept = k.slab.memory;
  quantize(x, &s[xq], keep_x ? &k.slab[k.x] : nullptr, nullptr);
  quantize(weight, &s[wq], keep_w ? &k.slab[k.w] : nullptr, nullptr);
  return product(operand(s[xq], M, K), operand(s[wq], N, K), bias.defined() ? bias.contiguous() : bias,
                 x.sizes().slice(0, x.dim() - 1), x.scalar_type(), x);
}

class LinearFunction : public torch::autograd::Function<LinearFunction> {
 public:
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const MaybeTensor &bias_) {
    const Tensor bias = given(bias_);
    const c10::cuda::CUDAGuard guard(x.device());
    const bool want_x = x.requires_grad(), want_w = weight.requires_grad();
    Tensor kept;
    const Tensor y = linear_forward(x, weight, bias, want_w, want_x, &kept);
    ctx->save_for_backward({kept});
    ctx->saved_data["facts"] = std::vector<int64_t>{
        want_x, want_w, bias.defined() && bias.requires_grad(), (int64_t)x.scalar_type(), (int64_t)weight.scalar_type(),
        (int64_t)(bias.defined() ? bias.scalar_type() : at::kFloat), x.size(-1)};
    return y;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    once("linear_quantized");
    const Tensor &dy = grads[0];
    if (!dy.defined()) return {Tensor(), Tensor(), Tensor()};
    const auto facts = ctx->saved_data["facts"].toIntVector();
    const bool want_x = facts[0], want_w = facts[1], want_b = facts[2];
    const auto x_type = (at::ScalarType)facts[3], w_type = (at::ScalarType)facts[4], b_type = (at::ScalarType)facts[5];
    const int64_t K = facts[6], N = dy.size(-1), M = N > 0 ? dy.numel() / N : 0;
    const c10::cuda::CUDAGuard guard(dy.device());
    if (N == 0) {
      std::vector<int64_t> shape(dy.sizes().begin(), dy.sizes().end());
      shape.back() = K;
      return {want_x ? at::zeros(shape, dy.options()) : Tensor(),
              want_w ? at::zeros({0, K}, dy.options().dtype(w_type)) : Tensor(),
              want_b ? at::zeros({0}, dy.options().dtype(b_type)) : Tensor()};
    }
    Kept kept(M, N, K, want_w, want_x);
    if (want_x || want_w) kept.slab.place(ctx->get_saved_variables()[0]);
    Slab s;
    size_t rows = 0, turned = 0;
    if (want_x) rows = s.add(M, N);
    if (want_w) turned = s.add(N, M);
    if (want_x || want_w) s.allocate(dy);
    const Tensor db = quantize(dy, want_x ? &s[rows] : nullptr, want_w ? &s[turned] : nullptr, want_b ? &b_type : nullptr);
    Tensor dx, dw;
    if (want_x)
      dx = product(operand(s[rows], M, N), operand(kept.slab[kept.w], K, N), Tensor(), dy.sizes().slice(0, dy.dim() - 1),
                   x_type, dy);
    if (want_w)
      dw = M == 0 ? at::zeros({N, K}, dy.options().dtype(w_type))
                  : product(operand(s[turned], N, M), operand(kept.slab[kept.x], K, M), Tensor(), {N}, w_type, dy);
    return {dx, dw, db};
  }
};

Tensor linear_quantized(const Tensor &x, const Tensor &weight, const MaybeTensor &bias_) {
  const Tensor bias = given(bias_);
  check_linear(x, weight, bias);
  if (needs_grad({&x, &weight, &bias})) return LinearFunction::apply(x, weight, bias_);
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor kept;
  return linear_forward(x, weight, bias, false, false, &kept);
}

// ---- orthogonalised steps ---------------------------------------------------------------

Tensor orthogonalize(const Tensor &x, int64_t steps, const std::vector<double> &coefficients, double eps) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (no CPU path)");
  const int dtype = dtype_of(x, "x");
  TORCH_CHECK(!has_tangent({&x}), "orthogonalize has no gradient, of forward mode neither");
  TORCH_CHECK_VALUE(x.dim() >= 2, "x must be [..., m, n], got ", x.sizes());
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor xc = x.contiguous();
  const int64_t m = x.size(-2), n = x.size(-1), batch = x.numel() > 0 ? x.numel() / (m * n) : 0;
  const Tensor out = at::empty(x.sizes(), x.options());
  const Tensor work = at::empty({cpab_b200_orthogonalize_workspace(dtype, batch, m, n)}, x.options().dtype(at::kByte));
  check(cpab_b200_orthogonalize(dtype, ptr(xc), batch, m, n, (int)steps, coefficients.data(), eps, ptr_mut(out),
                                ptr_mut(work), stream_of(x)));
  return out;
}

void muon(const pybind11::list &params, const pybind11::list &grads, const pybind11::list &momenta, double lr,
          const MaybeTensor &lr_device_, double momentum, bool nesterov, double weight_decay, int64_t steps,
          const std::vector<double> &coefficients, double eps, int64_t adjust) {
  const size_t n = params.size();
  const Tensor lr_device = given(lr_device_);
  TORCH_CHECK_VALUE(grads.size() == n && momenta.size() == n, "muon: lists of different lengths");
  if (n == 0) return;
  const Tensor &first = *item(params, 0, "muon: parameter");
  const at::Device device = first.device();
  TORCH_CHECK(device.is_cuda(), "params must be CUDA tensors (no CPU path)");
  TORCH_CHECK(!lr_device.defined() || (lr_device.device() == device && lr_device.scalar_type() == at::kFloat &&
                                       lr_device.numel() == 1),
              "muon: a learning rate on the device must be one float32 on the parameters' device, ", device);
  std::vector<cpab_muon_tensor> list(n);
  std::vector<Tensor> copies;  // contiguous gradients
  for (size_t k = 0; k < n; ++k) {
    const Tensor &p = *item(params, k, "muon: parameter"), &g = *item(grads, k, "muon: gradient");
    const Tensor &m = *item(momenta, k, "muon: momentum");
    TORCH_CHECK(p.device() == device && g.device() == device && m.device() == device, "muon: tensor ", k,
                ": all tensors must be on one device");
    TORCH_CHECK_TYPE(g.scalar_type() == p.scalar_type(), "muon: tensor ", k, ": gradient of type ", g.scalar_type(),
                     " for a parameter of type ", p.scalar_type());
    TORCH_CHECK_TYPE(m.scalar_type() == at::kFloat, "muon: tensor ", k, ": momentum must be float32, got ", m.scalar_type());
    TORCH_CHECK_VALUE(p.dim() == 2 && g.sizes() == p.sizes() && m.sizes() == p.sizes(), "muon: tensor ", k,
                      ": parameter, gradient and momentum must be matrices of one shape, got ", p.sizes());
    TORCH_CHECK_VALUE(p.is_contiguous() && m.is_contiguous(), "muon: tensor ", k,
                      ": parameter and momentum must be contiguous");
    const Tensor *grad = &g;
    if (!g.is_contiguous()) {
      copies.push_back(g.contiguous());
      grad = &copies.back();
    }
    list[k] = {ptr_mut(p), ptr(*grad), fptr_mut(m), p.size(0), p.size(1), dtype_of(p, "a parameter")};
  }
  const c10::cuda::CUDAGuard guard(device);
  for (size_t k = 0; k < n; ++k)
    for (const Tensor *t : {item(params, k, "muon: parameter"), item(momenta, k, "muon: momentum")}) written(*t);
  const Tensor work = at::empty({cpab_b200_muon_workspace(list.data(), (int)n)}, first.options().dtype(at::kByte));
  check(cpab_b200_muon(list.data(), (int)n, lr, fptr(lr_device), momentum, nesterov, weight_decay, (int)steps,
                       coefficients.data(), eps, (int)adjust, ptr_mut(work), stream_of(first)));
}

}  // namespace

void bind_projection(pybind11::module &m) {
  m.def("quantize_blocks", &quantize_blocks, "x, transposed -> [q, scale(, qt, scale_t)]");
  m.def("matmul_quantized", &matmul_quantized, "q, scale, weight, weight scale, bias or None, type -> y");
  m.def("linear_quantized", &linear_quantized, "x, weight, bias or None -> y");
  m.def("orthogonalize", &orthogonalize, "x, steps, coefficients, eps -> matrices");
  m.def("muon", &muon,
        "params, grads, momenta, lr, lr tensor or None, momentum, nesterov, weight decay, steps, coefficients, eps, "
        "adjust");
}
