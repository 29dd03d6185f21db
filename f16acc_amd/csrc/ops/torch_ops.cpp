// The operators' torch side: argument checks, allocation, autograd and the
// launch through the C ABI (include/f16acc_ops.h), in C++.  In Python the same
// steps took longer than the kernels of most calls: routing 1001 tokens of 60
// experts forward and backward 98 us, of which the kernels run 8.
//
// Everything runs on the current stream of the operands' device and allocates
// through torch's allocator; nothing synchronises and nothing is kept between
// calls.  A failed check raises ValueError, a failed launch RuntimeError, and a call that
// something records or differentiates forward NotImplementedError.

#include "torch_common.h"
#include "torch_fp4.h"

namespace {

// ---------------------------------------------------------------------------
// Quantisation
// ---------------------------------------------------------------------------

struct Rows {
  Tensor q, s;  // [rows, up(K, 128)], zero padded; [blocks, rows]
};

// Row blocks of x, and of x transposed, from one pass.
std::pair<Rows, Rows> quant_both(const Tensor& x, bool rows, bool cols) {
  const int64_t M = x.size(0), K = x.size(1);
  Rows r, c;
  if (rows) r = {empty({M, up(K, kBlock)}, x, kF8), empty({blocks(K), M}, x, at::kFloat)};
  if (cols) c = {empty({K, up(M, kBlock)}, x, kF8), empty({blocks(M), K}, x, at::kFloat)};
  const On on(x);
  check_rc(f16acc_quant_both(x.const_data_ptr(), type_of(x), M, K, x.stride(0), x.stride(1), bytes(r.q),
                             up(K, kBlock), floats(r.s), M, bytes(c.q), up(M, kBlock), floats(c.s), K, on.stream));
  return {r, c};
}

Rows quant_rows(const Tensor& x) { return quant_both(x, true, false).first; }

struct Squares {
  Tensor q, s, qt;  // [N, up(K, 128)], [blocks(N), blocks(K)], transposed values [K, up(N, 128)]
};
Squares quant_weight(const Tensor& w, bool transposed) {
  const int64_t N = w.size(0), K = w.size(1);
  Squares r{empty({N, up(K, kBlock)}, w, kF8), empty({blocks(N), blocks(K)}, w, at::kFloat), {}};
  if (transposed) r.qt = empty({K, up(N, kBlock)}, w, kF8);
  const On on(w);
  check_rc(f16acc_quant_weight(w.const_data_ptr(), type_of(w), N, K, w.stride(0), w.stride(1), bytes(r.q),
                               up(K, kBlock), floats(r.s), blocks(K), bytes(r.qt), up(N, kBlock), on.stream));
  return r;
}

std::tuple<Tensor, Tensor> quantize(const Tensor& x, bool transposed) {
  check_call("quantize", {&x});
  check_float("quantize", x);
  REQUIRE(x.dim() >= 1 && (!transposed || x.dim() == 2), "quantize needs ",
        transposed ? "a 2-d tensor to transpose" : "one dimension or more", ", got ", x.sizes());
  at::NoGradGuard no_grad;
  const Tensor x2 = rows_of(x.detach());
  if (transposed) {
    const Rows c = quant_both(x2, false, true).second;
    return {c.q.narrow(1, 0, x2.size(0)), c.s.t()};
  }
  const Rows r = quant_rows(x2);
  return {r.q.narrow(1, 0, x2.size(1)).view(x.sizes()), r.s.t().view(with_last(x, r.s.size(0)))};
}

std::tuple<Tensor, Tensor> quantize_weight(const Tensor& w) {
  check_call("quantize_weight", {&w});
  check_float("quantize_weight", w);
  REQUIRE(w.dim() >= 2, "quantize_weight needs [..., N, K], got ", w.sizes());
  at::NoGradGuard no_grad;
  const int64_t N = w.size(-2), K = w.size(-1);
  std::vector<int64_t> qs(w.sizes().begin(), w.sizes().end()), ss = qs;
  qs.back() = up(K, kBlock);
  ss.back() = blocks(K);
  ss[ss.size() - 2] = blocks(N);
  const Tensor q = empty(qs, w, kF8), s = empty(ss, w, at::kFloat);
  if (w.numel() == 0) return {q.narrow(-1, 0, K), s};
  const Tensor w3 = w.detach().reshape({-1, N, K});
  const On on(w);
  for (int64_t i = 0; i < w3.size(0); ++i) {
    const Tensor wi = w3[i];
    check_rc(f16acc_quant_weight(wi.const_data_ptr(), type_of(w), N, K, wi.stride(0), wi.stride(1),
                                 bytes(q) + i * N * qs.back(), qs.back(), floats(s) + i * blocks(N) * blocks(K),
                                 blocks(K), nullptr, 0, on.stream));
  }
  return {q.narrow(-1, 0, K), s};
}


// An e4m3 operand [..., rows, K] with rows as the products read them: itself, or a copy
// whose rows are 16-byte aligned and zero from K to the next multiple of 16.
Operand packed(const Tensor& q) {
  const int64_t d = q.dim(), rows = q.size(-2), K = q.size(-1), ld = rows > 1 ? q.stride(-2) : up(K, 16);
  bool as_it_is = K % 16 == 0 && (q.stride(-1) == 1 || K <= 1) && ld >= K && ld % 16 == 0 && ld <= kMaxRow &&
                  (uintptr_t)q.const_data_ptr() % 16 == 0;
  for (int64_t i = 0; i < d - 2; ++i) as_it_is = as_it_is && q.stride(i) % 16 == 0;
  if (as_it_is) return {q, ld};
  std::vector<int64_t> sizes(q.sizes().begin(), q.sizes().end());
  sizes.back() = up(K, 16);
  const Tensor out = empty(sizes, q, kF8);
  const Tensor src = d == 2 ? q : q.reshape({-1, K});  // (leading dimensions that do not merge are copied)
  const On on(q);
  check_rc(f16acc_pack8(bytes(src), bytes(out), src.size(0), K, src.stride(0), src.stride(1), up(K, 16), on.stream));
  return {out, up(K, 16)};
}

// Scales ([rows], [blocks of K]) as the products read them.
Tensor near(const Tensor& s) {
  return s.stride(0) <= kMaxRow / 4 ? s : s.clone(at::MemoryFormat::Contiguous);
}

// ---------------------------------------------------------------------------
// Products
// ---------------------------------------------------------------------------

// out [M, N] from x [M, K] and w [N, K]; sx and sw are ([m], [kb]) and ([n or n / 128], [kb]) indexed.
void product(const Tensor& x, int64_t ldx, const Tensor& sx, const Tensor& w, int64_t ldw, const Tensor& sw,
             bool row_scales, int64_t K, const Tensor& out, const Maybe& bias = {}, int tile = -1, int splits = 0) {
  const int64_t M = out.size(0), N = out.size(1);
  const size_t n = f16acc_mm_fp8_workspace(M, N, K, row_scales, tile, splits);
  Tensor ws;
  if (n) ws = empty({(int64_t)n}, out, at::kByte);
  const On on(out);
  check_rc(f16acc_mm_fp8(bytes(x), ldx, floats(sx), sx.stride(0), sx.stride(1), bytes(w), ldw, floats(sw),
                         sw.stride(0), sw.stride(1), row_scales, data(bias), out.data_ptr(), out.stride(0),
                         out.stride(1), M, N, K, type_of(out), tile, splits, bytes(ws), n, on.stream));
}

Tensor mm(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale, at::ScalarType out_dtype,
          const Maybe& bias, const Maybe& out_, int tile, int splits) {
  check_call("fp8.mm", {&a, &a_scale, &b, &b_scale});
  for (const Tensor* t : {&a, &a_scale, &b, &b_scale}) check_device("fp8.mm", a, *t);
  REQUIRE(a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(0), "fp8.mm needs (M, K) @ (K, N), got ", a.sizes(), " @ ",
        b.sizes());
  const int64_t M = a.size(0), K = a.size(1), N = b.size(1);
  REQUIRE(a.scalar_type() == kF8 && b.scalar_type() == kF8 && a_scale.scalar_type() == at::kFloat &&
            b_scale.scalar_type() == at::kFloat,
        "fp8.mm needs float8_e4m3fn operands and float32 scales");
  REQUIRE(a_scale.sizes() == at::IntArrayRef({M, blocks(K)}), "a_scale must be ", at::IntArrayRef({M, blocks(K)}),
        ", got ", a_scale.sizes());
  const bool row_scales = N > 1 && b_scale.sizes() == at::IntArrayRef({blocks(K), N});
  REQUIRE(row_scales || b_scale.sizes() == at::IntArrayRef({blocks(K), blocks(N)}), "b_scale must be ",
        at::IntArrayRef({blocks(K), blocks(N)}), " or ", at::IntArrayRef({blocks(K), N}), ", got ", b_scale.sizes());
  REQUIRE(is_type(out_dtype), "fp8.mm writes torch.float16, bfloat16 or float32, not ", out_dtype);
  Maybe b_;
  if (out_) {
    check_device("fp8.mm_tile", a, *out_);
    REQUIRE(out_->sizes() == at::IntArrayRef({M, N}), "out must be ", at::IntArrayRef({M, N}), ", got ", out_->sizes());
    REQUIRE(at::has_internal_overlap(*out_) != at::MemOverlap::Yes, "out must not share memory between its elements");
  }
  if (bias) {
    check_device("fp8.mm_tile", a, *bias);
    REQUIRE(bias->sizes() == at::IntArrayRef({N}) && bias->scalar_type() == out_dtype, "bias must be ", out_dtype, " [", N,
            "], got ", bias->scalar_type(), " ", bias->sizes());
    b_ = bias->contiguous();
  }
  const Tensor out = out_ ? *out_ : empty({M, N}, a, out_dtype);
  if (M == 0 || N == 0) return out;
  if (K == 0) return b_ ? out.copy_(b_->expand({M, N})) : out.zero_();
  const Operand x = packed(a), w = packed(b.t());
  product(x.q, x.ld, near(a_scale), w.q, w.ld, near(b_scale.t()), row_scales, K, out, b_, tile, splits);
  return out;
}

// y = x w^T + bias; dx = dy w, dw = dy^T x, each from operands quantised along its own
// contraction: x and dy in blocks of 128 channels and of 128 tokens, w in
// squares, which serve both of its products.
// The result is no view: autograd forbids changing a view that a function returned in place.
Tensor train_forward(const Tensor& x, const Tensor& w, const Maybe& bias, bool need_x, bool need_w, Rows* cols,
                     Squares* sq) {
  const Tensor x2 = rows_of(x);
  auto [r, c] = quant_both(x2, true, need_w);
  *cols = c;
  *sq = quant_weight(w, need_x);
  const Tensor y = empty(with_last(x, w.size(0)), x, x.scalar_type());
  product(r.q, r.q.size(1), r.s.t(), sq->q, sq->q.size(1), sq->s, false, x2.size(1),
          y.view({x2.size(0), w.size(0)}), bias);
  return y;
}

struct Train : torch::autograd::Function<Train> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& bias) {
    Rows cols;
    Squares sq;
    const Tensor y = train_forward(x, w, bias, x.requires_grad(), w.requires_grad(), &cols, &sq);
    ctx->save_for_backward({cols.q, cols.s, sq.qt, sq.s});
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["dtype"] = (int64_t)w.scalar_type();
    ctx->saved_data["need"] = (int64_t)x.requires_grad() + 2 * (int64_t)w.requires_grad() +
                              4 * (int64_t)(bias && bias->requires_grad());
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_derivative_only();
    const auto saved = ctx->get_saved_variables();
    const Tensor &qt = saved[0], &st = saved[1], &wqt = saved[2], &ws = saved[3];
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const int64_t need = ctx->saved_data["need"].toInt(), K = shape.back();
    const Tensor dy = rows_of(check_grad("fp8.linear", grads[0]));
    const int64_t M = dy.size(0), N = dy.size(1);
    Rows r, c;
    if (need & 3) std::tie(r, c) = quant_both(dy, need & 1, need & 2);
    Tensor dx, dw, db;
    if (need & 1) {
      dx = empty({M, K}, dy, dy.scalar_type());
      product(r.q, r.q.size(1), r.s.t(), wqt, wqt.size(1), ws.t(), false, N, dx);
      dx = dx.view(shape);
    }
    if (need & 2) {
      dw = empty({N, K}, dy, (at::ScalarType)ctx->saved_data["dtype"].toInt());
      product(c.q, c.q.size(1), c.s.t(), qt, qt.size(1), st.t(), true, M, dw);
    }
    if (need & 4) db = column_sums(dy);
    return {dx, dw, db};
  }
};

Tensor stored(const Tensor& x, const Tensor& w_, const Tensor& w_scale_, const Maybe& bias) {
  const Tensor x2 = rows_of(x), w_scale = near(w_scale_);
  const int64_t M = x2.size(0), K = x2.size(1), N = w_.size(0);
  // rows of any alignment go as they are (the library copies them where it has to)
  const bool rows = (K <= 1 || w_.stride(1) == 1) && (N <= 1 || w_.stride(0) >= K);
  const Operand w = rows ? Operand{w_, N > 1 ? w_.stride(0) : up(K, 16)} : packed(w_);
  Tensor y = empty(with_last(x, N), x, x.scalar_type());
  const size_t n = f16acc_linear_fp8_workspace(M, N, K, bytes(w.q), w.ld);
  const Tensor ws = empty({(int64_t)n}, x, at::kByte);
  const On on(x);
  check_rc(f16acc_linear_fp8(x2.const_data_ptr(), type_of(x), x2.stride(0), x2.stride(1), bytes(w.q), w.ld,
                             floats(w_scale), w_scale.stride(0), w_scale.stride(1), data(bias), y.data_ptr(), M, N, K,
                             bytes(ws), n, on.stream));
  return y;
}

// linear on a stored 8-bit weight, with the gradients of x and the bias.
struct Stored : torch::autograd::Function<Stored> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& w_scale,
                        const Maybe& bias) {
    ctx->save_for_backward({w, w_scale});
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["need"] = (int64_t)x.requires_grad() + 2 * (int64_t)(bias && bias->requires_grad());
    return stored(x, w, w_scale, bias);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_derivative_only();
    const auto saved = ctx->get_saved_variables();
    const Tensor &w = saved[0], &w_scale = saved[1];
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const int64_t need = ctx->saved_data["need"].toInt(), N = w.size(0), K = w.size(1);
    const Tensor dy = rows_of(check_grad("fp8.linear", grads[0]));
    Tensor dx, db;
    if (need & 1) {
      const Rows r = quant_rows(dy);
      const Operand wt = packed(w.t());
      dx = empty({dy.size(0), K}, dy, dy.scalar_type());
      product(r.q, r.q.size(1), r.s.t(), wt.q, wt.ld, near(w_scale.t()), false, N, dx);
      dx = dx.view(shape);
    }
    if (need & 2) db = column_sums(dy);
    return {dx, {}, {}, db};
  }
};

Tensor linear(const Tensor& x, const Tensor& w, const Maybe& w_scale, const Maybe& bias) {
  check_call("fp8.linear", {&x, &w, maybe(w_scale), maybe(bias)});
  check_float("fp8.linear", x);
  check_device("fp8.linear", x, w);
  if (w_scale) check_device("fp8.linear", x, *w_scale);
  if (bias) check_device("fp8.linear", x, *bias);
  REQUIRE(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1), "fp8.linear needs [..., K] and [N, K], got ",
        x.sizes(), " and ", w.sizes());
  const int64_t N = w.size(0), K = w.size(1);
  REQUIRE(!bias || (bias->sizes() == at::IntArrayRef({N}) && bias->scalar_type() == x.scalar_type()), "bias must be ",
        x.scalar_type(), " [", N, "], got ", bias->scalar_type(), " ", bias->sizes());
  if (!w_scale) {
    REQUIRE(is_type(w.scalar_type()), "fp8.linear needs w_scale for a ", w.scalar_type(), " weight");
  } else {
    REQUIRE(w.scalar_type() == kF8 && w_scale->scalar_type() == at::kFloat &&
              w_scale->sizes() == at::IntArrayRef({blocks(N), blocks(K)}),
          "fp8.linear needs a float8_e4m3fn weight with float32 ", at::IntArrayRef({blocks(N), blocks(K)}),
          " scales, got ", w.scalar_type(), " with ", w_scale->scalar_type(), " ", w_scale->sizes());
  }
  if (x.numel() == 0 || N == 0) {  // nothing to multiply: torch gives the empty (or zero) result and its gradients
    const Tensor y = at::matmul(x, w.to(x.scalar_type()).t());
    return bias ? y + *bias : y;
  }
  const bool grad = c10::GradMode::is_enabled();
  Maybe b;
  if (bias) b = bias->contiguous();
  if (!w_scale) {
    if (grad && (x.requires_grad() || w.requires_grad() || (b && b->requires_grad()))) return Train::apply(x, w, b);
    Rows cols;
    Squares sq;
    return train_forward(x, w, b, false, false, &cols, &sq);
  }
  if (grad && (x.requires_grad() || (b && b->requires_grad()))) return Stored::apply(x, w, *w_scale, b);
  return stored(x, w, *w_scale, b);
}

// ---------------------------------------------------------------------------
// Mixture of experts
// ---------------------------------------------------------------------------

struct RouteOptions {
  int64_t k, groups, top;
  bool sigmoid, renormalize;
  double scale;
};

std::tuple<Tensor, Tensor> route_forward(const Tensor& logits, const Maybe& bias, const RouteOptions& o) {
  const Tensor x = rows_of(logits);
  const int64_t T = x.size(0), E = x.size(1);
  const auto sizes = with_last(logits, o.k);
  Tensor weights = empty(sizes, x, at::kFloat), ids = empty(sizes, x, at::kInt);
  const On on(x);
  check_rc(f16acc_route(x.const_data_ptr(), type_of(x), T, x.stride(0), x.stride(1), (int)E, (int)o.k, o.sigmoid,
                        (const float*)data(bias), (int)o.groups, (int)o.top, o.renormalize, (float)o.scale,
                        floats(weights), (int*)ids.data_ptr(), on.stream));
  return {weights, ids};
}

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Maybe& bias, const RouteOptions& o) {
    auto [weights, ids] = route_forward(logits, bias, o);
    ctx->mark_non_differentiable({ids});
    ctx->save_for_backward({logits, ids});
    ctx->saved_data["o"] = (int64_t)o.k * 4 + o.sigmoid * 2 + o.renormalize;
    ctx->saved_data["scale"] = o.scale;
    return {weights, ids};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_derivative_only();
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &ids = saved[1];
    const int64_t o = ctx->saved_data["o"].toInt();
    Tensor dx = empty(logits.sizes(), logits, logits.scalar_type());
    if (!grads[0].defined()) return {dx.zero_(), {}, {}};
    const Tensor x = rows_of(logits), dw = rows_of(check_grad("route", grads[0]));
    const On on(x);
    check_rc(f16acc_route_grad(x.const_data_ptr(), type_of(x), x.size(0), x.stride(0), x.stride(1), (int)x.size(1),
                               (int)(o >> 2), (o >> 1) & 1, o & 1, (float)ctx->saved_data["scale"].toDouble(),
                               (const int*)ids.const_data_ptr(), floats(dw), dw.stride(0), dw.stride(1),
                               dx.data_ptr(), on.stream));
    return {dx, {}, {}};
  }
};

// The options of a routing over E experts, checked.
RouteOptions route_options(int64_t E, int64_t k, const std::string& scoring, int64_t groups, int64_t top,
                           bool renormalize, double scale) {
  REQUIRE(scoring == "softmax" || scoring == "sigmoid", "scoring must be 'softmax' or 'sigmoid', not '", scoring, "'");
  REQUIRE(1 <= E && E <= 1024, "route needs 1 to 1024 experts, got ", E);
  REQUIRE(1 <= groups && groups <= 64 && E % groups == 0 && 1 <= top && top <= groups, E, " experts in ", groups,
        " groups of which ", top, " stay: not equal groups, or over 64");
  REQUIRE(1 <= k && k <= 64 && k <= E / groups * top,
        "k must be 1 to 64 and at most the experts of the groups that stay, got ", k);
  return {k, groups, top, scoring == "sigmoid", renormalize, scale};
}

Maybe route_bias(const char* name, const Tensor& like, const Maybe& bias, int64_t E) {
  if (!bias) return {};
  check_device(name, like, *bias);
  REQUIRE(bias->scalar_type() == at::kFloat && bias->sizes() == at::IntArrayRef({E}), "bias must be float32 [", E,
        "], got ", bias->scalar_type(), " ", bias->sizes());
  return bias->detach().contiguous();
}

std::tuple<Tensor, Tensor> route(const Tensor& logits, int64_t k, const std::string& scoring, const Maybe& bias,
                                 int64_t groups, int64_t top, bool renormalize, double scale) {
  check_call("route", {&logits, maybe(bias)});
  check_float("route", logits);
  REQUIRE(logits.dim() >= 1, "route needs [..., E] logits");
  const RouteOptions o = route_options(logits.size(-1), k, scoring, groups, top, renormalize, scale);
  const Maybe b = route_bias("route", logits, bias, logits.size(-1));
  if (c10::GradMode::is_enabled() && logits.requires_grad()) {
    const variable_list r = Route::apply(logits, b, o);
    return {r[0], r[1]};
  }
  return route_forward(logits, b, o);
}

// The experts' weights, checked: w1 [E, 2, I, D], w2 [E, D, I] and their scales.
void check_experts(const char* name, const Tensor& x, const Tensor& w1, const Tensor& s1, const Tensor& w2,
                   const Tensor& s2) {
  const bool dims = x.dim() >= 1 && w1.dim() == 4 && w1.size(1) == 2 && w2.dim() == 3;
  const int64_t E = dims ? w1.size(0) : 0, I = dims ? w1.size(2) : 0, D = dims ? w1.size(3) : 0;
  REQUIRE(dims && x.size(-1) == D && w2.sizes() == at::IntArrayRef({E, D, I}) && 1 <= E && E <= 1024 && D > 0 && I > 0,
        name, " needs x [..., D], w1 [E, 2, I, D] and w2 [E, D, I] (E 1 to 1024, D and I positive), got ", x.sizes(),
        ", ", w1.sizes(), ", ", w2.sizes());
  REQUIRE(w1.scalar_type() == kF8 && w2.scalar_type() == kF8, name, " needs float8_e4m3fn weights");
  REQUIRE(s1.scalar_type() == at::kFloat && s1.sizes() == at::IntArrayRef({E, 2, blocks(I), blocks(D)}),
        "w1_scale must be float32 ", at::IntArrayRef({E, 2, blocks(I), blocks(D)}), ", got ", s1.scalar_type(), " ",
        s1.sizes());
  REQUIRE(s2.scalar_type() == at::kFloat && s2.sizes() == at::IntArrayRef({E, blocks(D), blocks(I)}),
        "w2_scale must be float32 ", at::IntArrayRef({E, blocks(D), blocks(I)}), ", got ", s2.scalar_type(), " ",
        s2.sizes());
}

void check_no_grad(const char* name, std::initializer_list<const Tensor*> tensors) {
  bool grown = false;
  for (const Tensor* t : tensors) grown = grown || (t && t->requires_grad());
  REQUIRE(!c10::GradMode::is_enabled() || !grown, name,
        " has no backward pass: call it under torch.no_grad() or torch.inference_mode()");
}

// The experts' weights as the kernels read them, and how many tokens go into one call: the kernels address
// rows of the quantised tokens and hidden values by 31 bits, more tokens go in parts.
struct ExpertRows {
  Operand w1, w2;
  int64_t part;
  // any: rows of any alignment go as they are
  ExpertRows(int64_t T, int64_t k, const Tensor& q1, const Tensor& q2, bool any) {
    const int64_t D = q1.size(3), I = q1.size(2);
    auto rows = [&](const Tensor& w) {
      return any && (w.size(-1) <= 1 || w.stride(-1) == 1) ? Operand{w, w.stride(-2)} : packed(w);
    };
    w1 = rows(q1), w2 = rows(q2);
    const int64_t most = 0x7fff0000 / std::max(up(D, kBlock), k * up(I, kBlock));
    part = std::min(T, std::max<int64_t>(most, 1));
  }
};

Tensor experts(const Tensor& x, const Tensor& weights, const Tensor& ids, const Tensor& w1, const Tensor& s1,
               const Tensor& w2, const Tensor& s2) {
  check_call("experts", {&x, &weights, &ids, &w1, &s1, &w2, &s2});
  check_float("experts", x);
  for (const Tensor* t : {&weights, &ids, &w1, &s1, &w2, &s2}) check_device("experts", x, *t);
  check_experts("experts", x, w1, s1, w2, s2);
  REQUIRE(ids.dim() == x.dim() && ids.sizes() == weights.sizes() && ids.size(-1) >= 1 &&
            ids.sizes().slice(0, ids.dim() - 1) == x.sizes().slice(0, x.dim() - 1),
        "weights and ids must be [..., k] over x's tokens, got ", weights.sizes(), " and ", ids.sizes(), " for ",
        x.sizes());
  REQUIRE(weights.scalar_type() == at::kFloat && (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong),
        "experts needs float32 weights and int32 or int64 ids, got ", weights.scalar_type(), " and ",
        ids.scalar_type());
  check_no_grad("experts", {&x, &weights, &w1, &s1, &w2, &s2});
  const int64_t E = w1.size(0), I = w1.size(2), D = w1.size(3), k = ids.size(-1);
  const Tensor x2 = rows_of(x), wt = rows_of(weights);
  const int64_t T = x2.size(0);
  Tensor y = empty(x.sizes(), x, x.scalar_type());
  if (T == 0) return y;
  Tensor i32 = rows_of(ids);
  if (i32.scalar_type() == at::kLong) i32 = i32.clamp(-1, E).to(at::kInt);  // (a cast alone would wrap)
  i32 = i32.contiguous();
  const ExpertRows p(T, k, w1, w2,
                     f16acc_experts_any_rows(x2.const_data_ptr(), type_of(x), T, x2.stride(0), x2.stride(1), (int)k));
  const size_t n = f16acc_experts_workspace(p.part, (int)k, (int)E, D, I);
  const Tensor ws = empty({(int64_t)n}, x, at::kByte);
  const On on(x);
  for (int64_t t = 0; t < T; t += p.part) {
    const int64_t tokens = std::min(p.part, T - t);
    check_rc(f16acc_experts((const char*)x2.const_data_ptr() + t * x2.stride(0) * x2.element_size(), type_of(x),
                            tokens, x2.stride(0), x2.stride(1), floats(wt) + t * wt.stride(0), wt.stride(0),
                            wt.stride(1), (const int*)i32.const_data_ptr() + t * k, (int)k, (int)E, D, I,
                            bytes(p.w1.q), p.w1.q.stride(0), p.w1.q.stride(1), p.w1.ld, floats(s1), s1.stride(0),
                            s1.stride(1), s1.stride(2), s1.stride(3), bytes(p.w2.q), p.w2.q.stride(0), p.w2.ld,
                            floats(s2), s2.stride(0), s2.stride(1), s2.stride(2),
                            (char*)y.data_ptr() + t * D * y.element_size(), bytes(ws), n, on.stream));
  }
  return y;
}

Tensor layer(const Tensor& x, const Tensor& router, int64_t k, const Tensor& w1, const Tensor& s1, const Tensor& w2,
             const Tensor& s2, const std::string& scoring, const Maybe& bias, int64_t groups, int64_t top,
             bool renormalize, double scale) {
  check_call("layer", {&x, &router, &w1, &s1, &w2, &s2, maybe(bias)});
  check_float("layer", x);
  for (const Tensor* t : {&router, &w1, &s1, &w2, &s2}) check_device("layer", x, *t);
  check_experts("layer", x, w1, s1, w2, s2);
  const int64_t E = w1.size(0), I = w1.size(2), D = w1.size(3);
  REQUIRE(is_type(router.scalar_type()) && router.sizes() == at::IntArrayRef({E, D}),
          "router must be torch.float16, bfloat16 or float32 ", at::IntArrayRef({E, D}), ", got ",
          router.scalar_type(), " ", router.sizes());
  const RouteOptions o = route_options(E, k, scoring, groups, top, renormalize, scale);
  const Maybe b = route_bias("layer", x, bias, E);
  check_no_grad("layer", {&x, &router, &w1, &s1, &w2, &s2, maybe(bias)});
  const Tensor x2 = rows_of(x);
  const int64_t T = x2.size(0);
  Tensor y = empty(x.sizes(), x, x.scalar_type());
  if (T == 0) return y;
  const ExpertRows p(T, k, w1, w2, f16acc_layer_any_rows(T, (int)k, D, I));
  const size_t n = f16acc_layer_workspace(p.part, (int)k, (int)E, D, I);
  const Tensor ws = empty({(int64_t)n}, x, at::kByte);
  const On on(x);
  for (int64_t t = 0; t < T; t += p.part) {
    const int64_t tokens = std::min(p.part, T - t);
    check_rc(f16acc_layer((const char*)x2.const_data_ptr() + t * x2.stride(0) * x2.element_size(), type_of(x), tokens,
                          x2.stride(0), x2.stride(1), router.const_data_ptr(), type_of(router), router.stride(0),
                          router.stride(1), (int)E, (int)k, o.sigmoid, (const float*)data(b), (int)o.groups, (int)o.top,
                          o.renormalize, (float)o.scale, D, I, bytes(p.w1.q), p.w1.q.stride(0), p.w1.q.stride(1),
                          p.w1.ld, floats(s1), s1.stride(0), s1.stride(1), s1.stride(2), s1.stride(3), bytes(p.w2.q),
                          p.w2.q.stride(0), p.w2.ld, floats(s2), s2.stride(0), s2.stride(1), s2.stride(2),
                          (char*)y.data_ptr() + t * D * y.element_size(), bytes(ws), n, on.stream));
  }
  return y;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.attr("torch_version") = TORCH_VERSION;  // the module uses torch's C++ types, which change between versions
  m.attr("abi_version") = f16acc_ops_abi_version();
  typedef py::call_guard<py::gil_scoped_release> Free;  // other threads run during checks, allocation and launch
  m.def("quantize", &quantize, Free());
  m.def("quantize_weight", &quantize_weight, Free());
  m.def("mm", [](const Tensor& a, const Tensor& sa, const Tensor& b, const Tensor& sb, py::object dtype,
                 const Maybe& bias, const Maybe& out, int tile, int splits) {
    REQUIRE(THPDtype_Check(dtype.ptr()), "fp8.mm writes torch.float16, bfloat16 or float32");
    const at::ScalarType type = ((THPDtype*)dtype.ptr())->scalar_type;
    py::gil_scoped_release free;
    return mm(a, sa, b, sb, type, bias, out, tile, splits);
  });
  m.def("linear", &linear, Free());
  m.def("route", &route, Free());
  m.def("experts", &experts, Free());
  m.def("layer", &layer, Free());
  m.def("fp4_quantize", &quantize4, Free());
  m.def("fp4_dequantize", [](const Tensor& q, const Tensor& s, py::object dtype) {
    REQUIRE(THPDtype_Check(dtype.ptr()), "fp4.dequantize gives torch.float16, bfloat16 or float32");
    const at::ScalarType type = ((THPDtype*)dtype.ptr())->scalar_type;
    py::gil_scoped_release free;
    return dequantize4(q, s, type);
  });
  m.def("fp4_mm", [](const Tensor& a, const Tensor& sa, const Tensor& b, const Tensor& sb, py::object dtype,
                     const Maybe& bias, const Maybe& out, int tile, int splits) {
    REQUIRE(THPDtype_Check(dtype.ptr()), "fp4.mm writes torch.float16, bfloat16 or float32");
    const at::ScalarType type = ((THPDtype*)dtype.ptr())->scalar_type;
    py::gil_scoped_release free;
    return mm4(a, sa, b, sb, type, bias, out, tile, splits);
  });
  m.def("fp4_linear", &linear4, Free());
}
