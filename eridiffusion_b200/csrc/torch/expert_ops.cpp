// Token-routed experts and products on 4-bit weights as autograd nodes: router, plan, dispatch, combine, the product grouped by
// expert and the product on codes. Shapes, types and devices are checked by ops/functional.py; nothing here reads a value back
// from the device. A backward pass that is recorded itself (create_graph) runs on nodes and operations that have gradients; operands are
// laid out before a node takes them, so that what it saves is what autograd knows.
#include "eri_ops.h"

#include <c10/cuda/CUDAGuard.h>

#include <limits>

namespace eri_ops {

namespace {

using c10::cuda::CUDAGuard;

// Rows that a kernel reads through a pointer and a row stride (a multiple of 8 elements), copied when they are not laid out so.
struct Rows {
  Tensor t;
  long long ld;
};
Rows rows_of(const Tensor& t) {
  if (rows_ok(t) && t.stride(0) >= t.size(1)) return {t, (long long)t.stride(0)};
  return {contig16(t), (long long)t.size(1)};
}
bool recorded() { return at::GradMode::is_enabled(); }       // inside a backward pass
const int* ints(const Tensor& t) { return t.defined() ? (const int*)t.data_ptr() : nullptr; }

// ------------------------------------------------------------------------------------------- router
struct ExpertRoute : torch::autograd::Function<ExpertRoute> {
  // The backward kernel's formulas (a row that may choose nothing has weights and gradients of zero).
  static Tensor gradient(const Tensor& s, const Tensor& allowed, const Tensor& idx, const Tensor& dw, bool normalize) {
    Tensor f = s.to(at::kFloat);
    if (allowed.defined()) f = f.masked_fill(allowed.logical_not(), -std::numeric_limits<float>::infinity());
    const Tensor top = f.gather(1, idx), first = top.detach().narrow(1, 0, 1);
    const Tensor m = first.masked_fill(first == -std::numeric_limits<float>::infinity(), 0.f);
    const Tensor z = (top - m).exp(), all = normalize ? z : (f - m).exp(), sum = all.sum(1, true), total = sum.masked_fill(sum == 0, 1.f);
    const Tensor w = z / total, dot = (w * dw).sum(1, true), none = at::zeros(s.sizes(), f.options());
    Tensor ds = normalize ? none.scatter(1, idx, w * (dw - dot)) : all / total * (none.scatter(1, idx, dw) - dot);
    if (allowed.defined()) ds = ds.masked_fill(allowed.logical_not(), 0.f);
    return ds.to(s.scalar_type());
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& s, const OptT& allowed_o, int64_t k, bool normalize) {
    const Tensor allowed = opt(allowed_o);
    const CUDAGuard guard(s.device());
    const int64_t T = s.size(0), E = s.size(1);
    const long long ld = s.is_contiguous() ? E : s.stride(0);
    Tensor idx = at::empty({T, k}, s.options().dtype(at::kLong)), w = empty_f32({T, k}, s);
    check(L.eri_expert_route_fwd(s.data_ptr(), ld, ptr(allowed), idx.data_ptr(), (float*)w.data_ptr(), (int)T, (int)E, (int)k, normalize,
                                 s.scalar_type() == at::kBFloat16, stream()), "expert_route_fwd");
    if (ctx) {
      ctx->save_for_backward({s, allowed, idx, w});
      ctx->saved_data["m"] = std::vector<int64_t>{k, normalize, ld};
      ctx->mark_non_differentiable({idx});
      ctx->set_materialize_grads(false);
    }
    return {idx, w};
  }
  static variable_list backward(AutogradContext* ctx, variable_list gout) {
    variable_list out(4);
    if (!gout[1].defined()) return out;
    auto sv = ctx->get_saved_variables();
    const Tensor &s = sv[0], &allowed = sv[1], &idx = sv[2], &w = sv[3];
    const auto m = ctx->saved_data["m"].toIntVector();
    const CUDAGuard guard(s.device());
    if (recorded()) {
      out[0] = gradient(s, allowed, idx, gout[1], m[1]);
      return out;
    }
    const Tensor dw = contig(gout[1]);
    Tensor ds = at::empty({s.size(0), s.size(1)}, s.options());
    check(L.eri_expert_route_bwd(s.data_ptr(), m[2], ptr(allowed), idx.data_ptr(), (const float*)w.data_ptr(),
                                 (const float*)dw.data_ptr(), ds.data_ptr(), (int)s.size(0), (int)s.size(1), (int)m[0], (int)m[1],
                                 s.scalar_type() == at::kBFloat16, stream()), "expert_route_bwd");
    out[0] = ds;
    return out;
  }
};

// ------------------------------------------------------------------------------------------- dispatch / combine
Tensor scatter(const Tensor& x_, const Tensor& rows, const Tensor& offsets) {
  const Rows x = rows_of(x_);
  const int64_t T = rows.size(0), k = rows.size(1), D = x.t.size(1), E = offsets.size(0) - 1;
  Tensor xs = empty_bf16({T * k, D}, x.t);
  check(L.eri_expert_scatter(x.t.data_ptr(), x.ld, ints(rows), ints(offsets) + E, xs.data_ptr(), (int)T, (int)k, (int)(T * k), (int)D,
                             stream()), "expert_scatter");
  return xs;
}
Tensor gather(const Tensor& y_, const Tensor& rows, const Tensor& w) {
  const Rows y = rows_of(y_);
  const int64_t T = rows.size(0), k = rows.size(1), D = y.t.size(1);
  Tensor out = empty_bf16({T, D}, y.t);
  check(L.eri_expert_gather(y.t.data_ptr(), y.ld, ints(rows), (const float*)ptr(w), out.data_ptr(), (int)T, (int)k, (int)(T * k), (int)D,
                            stream()), "expert_gather");
  return out;
}

struct ExpertDispatch : torch::autograd::Function<ExpertDispatch> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& rows, const Tensor& offsets) {
    const CUDAGuard guard(x.device());
    if (ctx) ctx->save_for_backward({rows, offsets});
    return scatter(x, rows, offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list gout) {
    auto sv = ctx->get_saved_variables();
    const Tensor &rows = sv[0], &offsets = sv[1];
    const CUDAGuard guard(rows.device());
    if (recorded()) return {expert_combine(gout[0], at::ones(rows.sizes(), rows.options().dtype(at::kFloat)), rows, offsets), Tensor(), Tensor()};
    return {gather(gout[0], rows, Tensor()), Tensor(), Tensor()};
  }
};

struct ExpertCombine : torch::autograd::Function<ExpertCombine> {
  // dy and dw in operations that have gradients; choices without a row go to one of their own behind the others.
  static Tensor nobody(const Tensor& rows) { return (rows < 0).logical_or(rows >= rows.numel()); }
  static Tensor gradient_rows(const Tensor& dout, const Tensor& w, const Tensor& rows) {
    const int64_t n = rows.numel(), D = dout.size(1);
    const Tensor dy = (w.unsqueeze(-1) * dout.to(at::kFloat).unsqueeze(1)).to(dout.scalar_type()).reshape({n, D});
    const Tensor to = rows.masked_fill(nobody(rows), n).flatten().to(at::kLong);
    return at::zeros({n + 1, D}, dout.options()).index_copy(0, to, dy).narrow(0, 0, n);
  }
  static Tensor gradient_weights(const Tensor& dout, const Tensor& y, const Tensor& rows) {
    const Tensor yt = y.index_select(0, rows.masked_fill(nobody(rows), 0).flatten()).view({rows.size(0), rows.size(1), y.size(1)}).to(at::kFloat);
    return (dout.to(at::kFloat).unsqueeze(1) * yt.masked_fill(nobody(rows).unsqueeze(-1), 0.f)).sum(-1);
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& w, const Tensor& rows, const Tensor& offsets) {
    const CUDAGuard guard(y.device());
    if (ctx) ctx->save_for_backward({w.requires_grad() ? y : Tensor(), w, rows, offsets});
    return gather(y, rows, w);
  }
  static variable_list backward(AutogradContext* ctx, variable_list gout) {
    auto sv = ctx->get_saved_variables();
    const Tensor &w = sv[1], &rows = sv[2], &offsets = sv[3];
    const CUDAGuard guard(rows.device());
    if (recorded())
      return {ctx->needs_input_grad(0) ? gradient_rows(gout[0], w, rows) : Tensor(),
              ctx->needs_input_grad(1) ? gradient_weights(gout[0], sv[0], rows) : Tensor(), Tensor(), Tensor()};
    const Rows d = rows_of(gout[0]), y = ctx->needs_input_grad(1) ? rows_of(sv[0]) : d;       // y: for dw alone
    const int64_t T = rows.size(0), k = rows.size(1), D = d.t.size(1), E = offsets.size(0) - 1;
    Tensor dy, dw;
    if (ctx->needs_input_grad(0)) dy = empty_bf16({T * k, D}, d.t);
    if (ctx->needs_input_grad(1)) dw = empty_f32({T, k}, d.t);
    if (dy.defined() || dw.defined())
      check(L.eri_expert_gather_bwd(d.t.data_ptr(), d.ld, y.t.data_ptr(), y.ld, ints(rows), (const float*)w.data_ptr(), ints(offsets) + E,
                                    mptr(dy), (float*)mptr(dw), (int)T, (int)k, (int)(T * k), (int)D, stream()), "expert_gather_bwd");
    return {dy, dw, Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------------------- grouped product
enum { kFwd = 0, kDx = 1, kDw = 2 };

// dw[e] = dy^T x over the rows of expert e, in `out` or added to it.
void weight_gradient(const Tensor& x_, const Tensor& dy_, const Tensor& offsets, const Tensor& out, bool accum) {
  const Rows x = rows_of(x_), dy = rows_of(dy_);
  const int64_t R = x.t.size(0), E = out.size(0), N = out.size(1), K = out.size(2);
  if (R > 0)
    check(L.eri_expert_gemm(kDw, x.t.data_ptr(), x.ld, dy.t.data_ptr(), dy.ld, nullptr, ints(offsets), out.data_ptr(), (int)R, (int)E, (int)N,
                            (int)K, 0, accum, extent(out), stream()), "expert_gemm_dw");
  else if (!accum)
    out.zero_();
}
// The same as a node, for backward passes that are recorded.
struct ExpertWeightGradient : torch::autograd::Function<ExpertWeightGradient> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& dy, const Tensor& offsets) {
    const CUDAGuard guard(x.device());
    ctx->save_for_backward({dy.requires_grad() ? x : Tensor(), x.requires_grad() ? dy : Tensor(), offsets});
    Tensor out = empty_bf16({offsets.size(0) - 1, dy.size(1), x.size(1)}, x);
    weight_gradient(x, dy, offsets, out, false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gout) {
    auto sv = ctx->get_saved_variables();
    const Tensor &x = sv[0], &dy = sv[1], &offsets = sv[2];
    Tensor gx, gdy;
    if (ctx->needs_input_grad(0)) gx = expert_linear(dy, gout[0].transpose(1, 2), offsets, 0, false);
    if (ctx->needs_input_grad(1)) gdy = expert_linear(x, gout[0], offsets, 0, false);
    return {gx, gdy, Tensor()};
  }
};

struct ExpertLinear : torch::autograd::Function<ExpertLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& w, const Tensor& offsets, int64_t columns, bool accum) {
    const CUDAGuard guard(x_.device());
    const Rows x = rows_of(x_);
    const int64_t R = x.t.size(0), E = w.size(0), N = w.size(1), K = w.size(2);
    Tensor y = empty_bf16({R, N}, x.t);
    if (R > 0)
      check(L.eri_expert_gemm(kFwd, x.t.data_ptr(), x.ld, nullptr, 0, w.data_ptr(), ints(offsets), y.data_ptr(), (int)R, (int)E, (int)N,
                              (int)K, (int)columns, 0, extent(y), stream()), "expert_gemm");
    if (ctx) {
      ctx->save_for_backward({w.requires_grad() ? x_ : Tensor(), w, offsets});       // a frozen weight leaves nothing to do with x
      ctx->saved_data["m"] = std::vector<int64_t>{columns, accum};
    }
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gout) {
    auto sv = ctx->get_saved_variables();
    const Tensor &x = sv[0], &w = sv[1], &offsets = sv[2];
    const auto m = ctx->saved_data["m"].toIntVector();
    const CUDAGuard guard(w.device());
    const int64_t E = w.size(0), N = w.size(1), K = w.size(2);
    Tensor dx, dw;
    if (recorded()) {
      if (ctx->needs_input_grad(0)) dx = expert_linear(gout[0], w.transpose(1, 2), offsets, m[0], false);
      if (ctx->needs_input_grad(1)) dw = ExpertWeightGradient::apply(x, gout[0], offsets);
      return {dx, dw, Tensor(), Tensor(), Tensor()};
    }
    const Rows dy = rows_of(gout[0]);
    if (ctx->needs_input_grad(0)) {
      const int64_t R = dy.t.size(0);
      dx = empty_bf16({R, K}, dy.t);
      if (R > 0)
        check(L.eri_expert_gemm(kDx, dy.t.data_ptr(), dy.ld, nullptr, 0, w.data_ptr(), ints(offsets), dx.data_ptr(), (int)R, (int)E,
                                (int)N, (int)K, (int)m[0], 0, extent(dx), stream()), "expert_gemm_dx");
    }
    if (ctx->needs_input_grad(1)) {
      const bool acc = has_grad_buffer(w, at::kBFloat16, m[1]) && al16(w.grad());
      Tensor out = acc ? w.grad() : empty_bf16({E, N, K}, w);
      weight_gradient(x, dy.t, offsets, out, acc);
      if (!acc) dw = out;
    }
    return {dx, dw, Tensor(), Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------------------- 4-bit codes
// dx = dy W on the codes.
Tensor codes_gradient(const Tensor& dy_, const Tensor& codes, const Tensor& scale, const Tensor& offsets, int E, int N, int K, int block, bool nf4) {
  const CUDAGuard guard(codes.device());
  const Tensor dy = contig16(dy_);
  const int R = (int)dy.size(0);
  Tensor dx = empty_bf16({R, K}, dy);
  if (R > 0) {
    Tensor work = empty_f32({L.eri_linear_4bit_planes(R, N, K, block, offsets.defined()), R, K}, dy);
    check(L.eri_linear_4bit_dgrad(dy.data_ptr(), N, codes.data_ptr(), (const float*)scale.data_ptr(), ints(offsets), (float*)work.data_ptr(),
                                  dx.data_ptr(), R, E, N, K, block, nf4, stream()), "linear_4bit_dgrad");
  }
  return dx;
}
// The same as a node, for backward passes that are recorded.
struct Linear4bitGradient : torch::autograd::Function<Linear4bitGradient> {
  static Tensor forward(AutogradContext* ctx, const Tensor& dy, const Tensor& codes, const Tensor& scale, const OptT& offsets_o, int64_t E,
                        int64_t N, int64_t K, int64_t block, bool nf4) {
    ctx->save_for_backward({codes, scale, opt(offsets_o)});
    ctx->saved_data["m"] = std::vector<int64_t>{E, N, block, nf4};
    return codes_gradient(dy, codes, scale, opt(offsets_o), (int)E, (int)N, (int)K, (int)block, nf4);
  }
  static variable_list backward(AutogradContext* ctx, variable_list gout) {
    auto sv = ctx->get_saved_variables();
    const auto m = ctx->saved_data["m"].toIntVector();
    variable_list out(9);
    out[0] = *linear_4bit(gout[0], sv[0], sv[1], wrap(sv[2]), OptT(), m[0], m[1], m[2], m[3]);
    return out;
  }
};

struct Linear4bit : torch::autograd::Function<Linear4bit> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& codes, const Tensor& scale, const OptT& offsets_o,
                        const OptT& bias_o, int64_t E, int64_t N, int64_t block, bool nf4) {
    const Tensor offsets = opt(offsets_o), bias = opt(bias_o);
    const CUDAGuard guard(x_.device());
    const Rows x = rows_of(x_);
    const int64_t R = x.t.size(0), K = x.t.size(1);
    Tensor y = empty_bf16({R, N}, x.t);
    if (R > 0)
      check(L.eri_linear_4bit(x.t.data_ptr(), x.ld, codes.data_ptr(), (const float*)scale.data_ptr(), ints(offsets), ptr(bias), y.data_ptr(),
                              (int)R, (int)E, (int)N, (int)K, (int)block, nf4, stream()), "linear_4bit");
    if (ctx) {
      ctx->save_for_backward({codes, scale, offsets});
      ctx->saved_data["m"] = std::vector<int64_t>{R, K, E, N, block, nf4, bias.defined()};
    }
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gout) {
    auto sv = ctx->get_saved_variables();
    const Tensor &codes = sv[0], &scale = sv[1], &offsets = sv[2];
    const auto m = ctx->saved_data["m"].toIntVector();
    const CUDAGuard guard(codes.device());
    Tensor dx, db;
    if (ctx->needs_input_grad(0))
      dx = recorded() ? Linear4bitGradient::apply(gout[0], codes, scale, wrap(offsets), m[2], m[3], m[1], m[4], (bool)m[5])
                      : codes_gradient(gout[0], codes, scale, offsets, (int)m[2], (int)m[3], (int)m[1], (int)m[4], m[5]);
    // an absent optional argument has no edge; a bias comes without offsets
    if (m[6] && ctx->needs_input_grad(3)) db = gout[0].sum(0);
    return {dx, Tensor(), Tensor(), Tensor(), db, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

}  // namespace

namespace {
void same_device(const char* what, const Tensor& a, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK_VALUE(!t->defined() || t->device() == a.device(), what, ": tensors on different devices: ", a.device(), " and ", t->device());
}
void check_plan(const char* what, const Tensor& rows, const Tensor& offsets) {
  TORCH_CHECK_VALUE(rows.scalar_type() == at::kInt && rows.is_contiguous() && offsets.scalar_type() == at::kInt && offsets.is_contiguous() &&
                        offsets.dim() == 1 && offsets.size(0) > 1, what, ": not a plan of expert_plan");
}
// Offsets as the kernels take them; rows are fewer than 2^31, so a wider offset is one behind them all.
Tensor int32(const Tensor& t) { return contig(t.scalar_type() == at::kInt ? t : t.clamp(0, std::numeric_limits<int>::max()).to(at::kInt)); }
}  // namespace

// Whether ts are the slices whole[0], whole[1], .. and record no gradients.
bool are_slices(const Tensor& whole, const std::vector<Tensor>& ts) {
  if (whole.size(0) != (int64_t)ts.size()) return false;
  const char* at = (const char*)whole.data_ptr();
  for (const Tensor& t : ts) {
    if (t.data_ptr() != at || t.sizes() != whole.sizes().slice(1) || t.scalar_type() != whole.scalar_type() || !t.is_contiguous() ||
        t.requires_grad() || t.device() != whole.device())
      return false;
    at += t.numel() * t.element_size();
  }
  return true;
}

std::vector<Tensor> expert_route(const Tensor& scores, const OptT& allowed_, int64_t k, bool normalize) {
  const Tensor allowed = contig(opt(allowed_));
  same_device("expert_route", scores, {&allowed});
  const bool grad = any_grad({&scores});
  const Tensor s = scores.stride(1) == 1 && scores.stride(0) >= scores.size(1) ? scores : scores.contiguous();
  if (grad) return ExpertRoute::apply(s, wrap(allowed), k, normalize);
  return ExpertRoute::forward(nullptr, s, wrap(allowed), k, normalize);
}

std::vector<Tensor> expert_plan(const Tensor& idx_, int64_t experts) {
  const CUDAGuard guard(idx_.device());
  const Tensor idx = contig(idx_);
  const auto o = idx.options().dtype(at::kInt);
  const int64_t n = idx.numel();
  Tensor offsets = at::empty({experts + 1}, o), rows = at::empty(idx.sizes(), o);
  check(L.eri_expert_plan(idx.data_ptr(), idx.scalar_type() == at::kLong, (int)n, (int)experts, (int*)offsets.data_ptr(),
                          (int*)rows.data_ptr(), stream()), "expert_plan");
  return {offsets, rows};
}

Tensor expert_dispatch(const Tensor& x, const Tensor& rows, const Tensor& offsets) {
  same_device("expert_dispatch", x, {&rows, &offsets});
  check_plan("expert_dispatch", rows, offsets);
  if (any_grad({&x})) return ExpertDispatch::apply(x, rows, offsets);
  return ExpertDispatch::forward(nullptr, x, rows, offsets);
}

Tensor expert_combine(const Tensor& y_, const Tensor& w_, const Tensor& rows, const Tensor& offsets) {
  same_device("expert_combine", y_, {&w_, &rows, &offsets});
  check_plan("expert_combine", rows, offsets);
  const bool grad = any_grad({&y_, &w_});
  const Tensor y = rows_of(y_).t, w = contig(w_.scalar_type() == at::kFloat ? w_ : w_.to(at::kFloat));
  if (grad) return ExpertCombine::apply(y, w, rows, offsets);
  return ExpertCombine::forward(nullptr, y, w, rows, offsets);
}

Tensor expert_linear(const Tensor& x_, const Tensor& w_, const Tensor& offsets_, int64_t columns, bool accum) {
  same_device("expert_linear", x_, {&w_, &offsets_});
  const bool grad = any_grad({&x_, &w_});
  const Tensor offsets = int32(offsets_), x = rows_of(x_).t, w = contig16(w_);
  if (grad) return ExpertLinear::apply(x, w, offsets, columns, accum);
  return ExpertLinear::forward(nullptr, x, w, offsets, columns, accum);
}

// Nothing where the codes are not laid out for the kernel, or were made in inference mode and a gradient is asked for.
OptT linear_4bit(const Tensor& x, const Tensor& codes, const Tensor& scale_, const OptT& offsets_, const OptT& bias_, int64_t experts,
                 int64_t N, int64_t block, bool nf4) {
  const Tensor bias = contig(opt(bias_));
  Tensor offsets = opt(offsets_);
  same_device("linear_4bit", x, {&codes, &scale_, &offsets, &bias});
  const int64_t weights = experts * N * x.size(-1);
  TORCH_CHECK_VALUE(codes.numel() * 2 == weights && scale_.numel() * block == weights, "linear_4bit: ", codes.numel(), " bytes of codes and ",
                    scale_.numel(), " scales for ", weights, " weights in blocks of ", block);
  if (codes.scalar_type() != at::kByte || !codes.is_contiguous() || !al16(codes)) return OptT();
  if (offsets.defined()) offsets = int32(offsets);
  const Tensor scale = contig(scale_.scalar_type() == at::kFloat ? scale_ : scale_.to(at::kFloat));
  const int64_t K = x.size(-1);
  const Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, K});
  const bool grad = any_grad({&x2, &bias});
  if (grad && (codes.is_inference() || scale.is_inference())) return OptT();       // they cannot be kept for the backward pass
  Tensor y = grad ? Linear4bit::apply(x2, codes, scale, wrap(offsets), wrap(bias), experts, N, block, nf4)
                  : Linear4bit::forward(nullptr, x2, codes, scale, wrap(offsets), wrap(bias), experts, N, block, nf4);
  if (x.dim() == 2) return y;
  auto shape = x.sizes().vec();
  shape.back() = N;
  return y.view(shape);
}

}  // namespace eri_ops
