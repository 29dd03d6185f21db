// The torch side of the microscaled 4-bit operators (f16acc_amd.fp4).
#pragma once

#include "torch_common.h"

namespace {

constexpr int64_t kMx = 32;
constexpr auto kF4 = at::ScalarType::Float4_e2m1fn_x2;  // two values
constexpr auto kE8 = at::ScalarType::Float8_e8m0fnu;
int64_t pairs(int64_t v) { return (v + 1) / 2; }
int64_t mx_blocks(int64_t v) { return (v + kMx - 1) / kMx; }

// A 4-bit operand, or scales, as [rows, last dimension], as bytes where torch may have to copy them (it has
// few functions for their types).
Tensor rows4(const Tensor& t) { return t.dim() == 2 ? t : rows_of(t.detach().view(at::kByte)); }

// An operand of a product: bytes of strides (r, c); the scales' dword of (row, quad of blocks) at row * row + quad * quad
// bytes, or, where quad is 0, the byte of (row, block) at row * row + block * block.
struct Operand4 {
  const uint8_t *q, *s;
  int64_t r, c, row, block, quad;
};

// What quantising gives: rows of 64 bytes a quad, then the scales in the products' order, in one allocation.
struct Quantised4 {
  Tensor held;
  int64_t rows, quads;
  Quantised4() : rows(0), quads(0) {}
  Quantised4(int64_t rows, int64_t cols, const Tensor& like)
      : held(empty({rows * blocks(cols) * 68}, like, at::kByte)), rows(rows), quads(blocks(cols)) {}
  Quantised4(const Tensor& held, int64_t rows, int64_t cols) : held(held), rows(rows), quads(blocks(cols)) {}
  uint8_t* q() const { return bytes(held); }
  uint8_t* s() const { return held.defined() ? bytes(held) + rows * quads * 64 : nullptr; }
  Operand4 operand() const { return {q(), s(), 64 * quads, 1, 4, 1, 4 * rows}; }
};

// A matrix to quantise along its rows (q) and columns (qt), either perhaps undefined.
f16acc_fp4_matrix matrix4(const Tensor& x, const Quantised4& q, const Quantised4& qt) {
  return {x.const_data_ptr(), x.size(0), x.size(1), x.stride(0), x.stride(1), q.q(), 64 * q.quads, q.s(), 4, 4 * q.rows,
          qt.q(), 64 * qt.quads, qt.s(), 4, 4 * qt.rows};
}
void quant4(const f16acc_fp4_matrix* a, const f16acc_fp4_matrix* b, const Tensor& x) {
  const On on(x);
  check_rc(f16acc_fp4_quant(a, b, type_of(x), on.stream));
}

std::tuple<Tensor, Tensor> quantize4(const Tensor& x, bool transposed) {
  check_call("fp4.quantize", {&x});
  check_float("fp4.quantize", x);
  REQUIRE(x.dim() >= 1 && (!transposed || x.dim() == 2), "fp4.quantize needs ",
          transposed ? "a 2-d tensor to transpose" : "one dimension or more", ", got ", x.sizes());
  at::NoGradGuard no_grad;
  const Tensor x2 = rows_of(x.detach());
  const int64_t M = x2.size(0), K = x2.size(1), R = transposed ? K : M, C = transposed ? M : K;
  const int64_t ld = 64 * blocks(C), lds = 4 * blocks(C);
  const Tensor q = empty({R, ld}, x, kF4), s = empty({R, lds}, x, kE8);
  f16acc_fp4_matrix m{x2.const_data_ptr(), M, K, x2.stride(0), x2.stride(1)};
  if (transposed)
    m.qt = bytes(q), m.ldqt = ld, m.st = bytes(s), m.st_row = lds, m.st_quad = 4;
  else
    m.q = bytes(q), m.ldq = ld, m.s = bytes(s), m.s_row = lds, m.s_quad = 4;
  quant4(&m, nullptr, x);
  // the rows without their padding, with x's leading dimensions
  auto trimmed = [&](const Tensor& t, int64_t last) {
    if (transposed) return t.narrow(1, 0, last);
    std::vector<int64_t> strides(x.dim(), 1);
    for (int64_t i = x.dim() - 2, step = t.size(1); i >= 0; --i) strides[i] = step, step *= std::max<int64_t>(x.size(i), 1);
    return t.as_strided(with_last(x, last), strides);
  };
  return {trimmed(q, pairs(C)), trimmed(s, mx_blocks(C))};
}

Tensor dequantize4(const Tensor& q, const Tensor& s, at::ScalarType dtype) {
  check_call("fp4.dequantize", {&q, &s});
  for (const Tensor* t : {&q, &s}) check_device("fp4.dequantize", q, *t);
  REQUIRE(q.scalar_type() == kF4 && s.scalar_type() == kE8,
          "fp4.dequantize needs float4_e2m1fn_x2 values and float8_e8m0fnu scales, got ", q.scalar_type(), " and ",
          s.scalar_type());
  REQUIRE(is_type(dtype), "fp4.dequantize gives torch.float16, bfloat16 or float32, not ", dtype);
  REQUIRE(q.dim() >= 1, "fp4.dequantize needs one dimension or more");
  const int64_t C = 2 * q.size(-1);
  REQUIRE(s.sizes() == at::IntArrayRef(with_last(q, mx_blocks(C))), "scale must be ",
          at::IntArrayRef(with_last(q, mx_blocks(C))), ", got ", s.sizes());
  at::NoGradGuard no_grad;
  const Tensor out = empty(with_last(q, C), q, dtype), q2 = rows4(q), s2 = rows4(s);
  const On on(q);
  check_rc(f16acc_fp4_values(bytes(q2), q2.stride(0), q2.stride(1), bytes(s2), s2.stride(0), s2.stride(1), q2.size(0),
                             C, out.data_ptr(), type_of(out), on.stream));
  return out;
}

Operand4 stored4(const Tensor& q, const Tensor& s) {
  return {bytes(q), bytes(s), q.stride(0), q.stride(1), s.stride(0), s.stride(1), 0};
}

// out [M, N] from x [M, K] and w [N, K].
void product4(const Operand4& x, const Operand4& w, int64_t K, const Tensor& out, const Maybe& bias = {}, int tile = -1,
              int splits = 0) {
  const int64_t M = out.size(0), N = out.size(1);
  const size_t n = f16acc_mm_fp4_workspace(x.q, x.r, x.c, x.quad, w.q, w.r, w.c, w.quad, M, N, K, tile, splits);
  Tensor ws;
  if (n) ws = empty({(int64_t)n}, out, at::kByte);
  const On on(out);
  check_rc(f16acc_mm_fp4(x.q, x.r, x.c, x.s, x.row, x.block, x.quad, w.q, w.r, w.c, w.s, w.row, w.block, w.quad,
                         data(bias), out.data_ptr(), out.stride(0), out.stride(1), M, N, K, type_of(out), tile, splits,
                         bytes(ws), n, on.stream));
}

Tensor mm4(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale, at::ScalarType out_dtype,
           const Maybe& bias, const Maybe& out_, int tile, int splits) {
  check_call("fp4.mm", {&a, &a_scale, &b, &b_scale});
  for (const Tensor* t : {&a, &a_scale, &b, &b_scale}) check_device("fp4.mm", a, *t);
  REQUIRE(a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(0), "fp4.mm needs (M, K / 2) @ (K / 2, N), got ",
          a.sizes(), " @ ", b.sizes());
  const int64_t M = a.size(0), P = a.size(1), K = 2 * P, N = b.size(1);
  REQUIRE(a.scalar_type() == kF4 && b.scalar_type() == kF4 && a_scale.scalar_type() == kE8 &&
              b_scale.scalar_type() == kE8,
          "fp4.mm needs float4_e2m1fn_x2 operands and float8_e8m0fnu scales");
  REQUIRE(a_scale.sizes() == at::IntArrayRef({M, mx_blocks(K)}), "a_scale must be ",
          at::IntArrayRef({M, mx_blocks(K)}), ", got ", a_scale.sizes());
  REQUIRE(b_scale.sizes() == at::IntArrayRef({mx_blocks(K), N}), "b_scale must be ",
          at::IntArrayRef({mx_blocks(K), N}), ", got ", b_scale.sizes());
  REQUIRE(is_type(out_dtype), "fp4.mm writes torch.float16, bfloat16 or float32, not ", out_dtype);
  Maybe b_;
  if (out_) {
    check_device("fp4.mm_tile", a, *out_);
    REQUIRE(out_->sizes() == at::IntArrayRef({M, N}), "out must be ", at::IntArrayRef({M, N}), ", got ", out_->sizes());
    REQUIRE(at::has_internal_overlap(*out_) != at::MemOverlap::Yes, "out must not share memory between its elements");
  }
  if (bias) {
    check_device("fp4.mm_tile", a, *bias);
    REQUIRE(bias->sizes() == at::IntArrayRef({N}) && bias->scalar_type() == out_dtype, "bias must be ", out_dtype,
            " [", N, "], got ", bias->scalar_type(), " ", bias->sizes());
    b_ = bias->contiguous();
  }
  const Tensor out = out_ ? *out_ : empty({M, N}, a, out_dtype);
  if (M == 0 || N == 0) return out;
  if (K == 0) return b_ ? out.copy_(b_->expand({M, N})) : out.zero_();
  const Operand4 bt{bytes(b), bytes(b_scale), b.stride(1), b.stride(0), b_scale.stride(1), b_scale.stride(0), 0};
  product4(stored4(a, a_scale), bt, K, out, b_, tile, splits);
  return out;
}

// y = x w^T + bias; dx = dy w, dw = dy^T x, each from operands quantised along its own contraction.
Tensor train_forward4(const Tensor& x, const Tensor& w, const Maybe& bias, bool need_x, bool need_w, Quantised4* xt,
                      Quantised4* wt) {
  const Tensor x2 = rows_of(x);
  const int64_t M = x2.size(0), K = x2.size(1), N = w.size(0);
  const Quantised4 xr(M, K, x), wr(N, K, x);
  if (need_w) *xt = Quantised4(K, M, x);
  if (need_x) *wt = Quantised4(K, N, x);
  const f16acc_fp4_matrix a = matrix4(x2, xr, *xt), b = matrix4(w, wr, *wt);
  if (x.scalar_type() == w.scalar_type()) {
    quant4(&a, &b, x);
  } else {
    quant4(&a, nullptr, x);
    quant4(&b, nullptr, w);
  }
  const Tensor y = empty(with_last(x, N), x, x.scalar_type());
  product4(xr.operand(), wr.operand(), K, y.view({M, N}), bias);
  return y;
}

struct Train4 : torch::autograd::Function<Train4> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& bias) {
    Quantised4 xt, wt;
    const Tensor y = train_forward4(x, w, bias, x.requires_grad(), w.requires_grad(), &xt, &wt);
    ctx->save_for_backward({xt.held, wt.held});
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["dtype"] = (int64_t)w.scalar_type() * 8 + (int64_t)x.requires_grad() +
                               2 * (int64_t)w.requires_grad() + 4 * (int64_t)(bias && bias->requires_grad());
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_derivative_only();
    const auto saved = ctx->get_saved_variables();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const int64_t need = ctx->saved_data["dtype"].toInt(), K = shape.back();
    const Tensor dy = rows_of(check_grad("fp4.linear", grads[0]));
    const int64_t M = dy.size(0), N = dy.size(1);
    Quantised4 r, c;
    if (need & 1) r = Quantised4(M, N, dy);
    if (need & 2) c = Quantised4(N, M, dy);
    if (need & 3) {
      const f16acc_fp4_matrix m = matrix4(dy, r, c);
      quant4(&m, nullptr, dy);
    }
    Tensor dx, dw, db;
    if (need & 1) {
      dx = empty(shape, dy, dy.scalar_type());
      product4(r.operand(), Quantised4(saved[1], K, N).operand(), N, dx.view({M, K}));
    }
    if (need & 2) {
      dw = empty({N, K}, dy, (at::ScalarType)(need >> 3));
      product4(c.operand(), Quantised4(saved[0], K, M).operand(), M, dw);
    }
    if (need & 4) db = column_sums(dy);
    return {dx, dw, db};
  }
};

// Bytes [rows, pairs] of any strides as rows.
Operand packed4(const Tensor& q) {
  const int64_t rows = q.size(0), n = q.size(1);
  const Tensor out = empty({rows, up(n, 16)}, q, at::kByte);
  const On on(q);
  check_rc(f16acc_pack8(bytes(q), bytes(out), rows, n, q.stride(0), q.stride(1), up(n, 16), on.stream));
  return {out, up(n, 16)};
}

Tensor stored_linear4(const Tensor& x, const Tensor& q, const Tensor& s, const Maybe& bias) {
  const Tensor x2 = rows_of(x);
  const int64_t M = x2.size(0), K = x2.size(1), N = q.size(0), P = pairs(K);
  // rows of any alignment go as they are (the library copies them where it has to)
  const bool rows = (P <= 1 || q.stride(1) == 1) && (N <= 1 || q.stride(0) >= P);
  const Operand o = rows ? Operand{q, N > 1 ? q.stride(0) : up(P, 16)} : packed4(q);  // (a row-major [K / 2, N] weight)
  Tensor y = empty(with_last(x, N), x, x.scalar_type());
  const bool few = f16acc_linear_fp4_few(M, N, K, x2.stride(1));
  const size_t n = few ? 0 : f16acc_linear_fp4_workspace(M, N, K, bytes(o.q), o.ld);
  Tensor ws;
  if (n) ws = empty({(int64_t)n}, x, at::kByte);
  const On on(x);
  check_rc(f16acc_linear_fp4(x2.const_data_ptr(), type_of(x), x2.stride(0), x2.stride(1), bytes(o.q), o.ld, bytes(s),
                             s.stride(0), s.stride(1), data(bias), y.data_ptr(), M, N, K, bytes(ws), n, on.stream));
  return y;
}

// linear on a stored 4-bit weight, with the gradients of x and the bias: dx's product takes the weight's values
// quantised again, along its own contraction.
struct Stored4 : torch::autograd::Function<Stored4> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& w_scale,
                        const Maybe& bias) {
    ctx->save_for_backward({w, w_scale});
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["need"] = (int64_t)x.requires_grad() + 2 * (int64_t)(bias && bias->requires_grad());
    return stored_linear4(x, w, w_scale, bias);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_derivative_only();
    const auto saved = ctx->get_saved_variables();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const int64_t need = ctx->saved_data["need"].toInt(), N = saved[0].size(0), K = shape.back();
    const Tensor dy = rows_of(check_grad("fp4.linear", grads[0]));
    Tensor dx, db;
    if (need & 1) {
      const Tensor &q = saved[0], &s = saved[1];
      const Quantised4 wt(K, N, dy), r(dy.size(0), N, dy);
      const f16acc_fp4_matrix m = matrix4(dy, r, Quantised4());
      quant4(&m, nullptr, dy);
      {
        const On on(dy);
        check_rc(f16acc_fp4_transpose(bytes(q), q.stride(0), q.stride(1), bytes(s), s.stride(0), s.stride(1), N, K,
                                      wt.q(), 64 * wt.quads, wt.s(), 4, 4 * K, on.stream));
      }
      dx = empty(shape, dy, dy.scalar_type());
      product4(r.operand(), wt.operand(), N, dx.view({dy.size(0), K}));
    }
    if (need & 2) db = column_sums(dy);
    return {dx, {}, {}, db};
  }
};

Tensor linear4(const Tensor& x, const Tensor& w, const Maybe& w_scale, const Maybe& bias) {
  check_call("fp4.linear", {&x, &w, maybe(w_scale), maybe(bias)});
  check_float("fp4.linear", x);
  check_device("fp4.linear", x, w);
  if (w_scale) check_device("fp4.linear", x, *w_scale);
  if (bias) check_device("fp4.linear", x, *bias);
  REQUIRE(x.dim() >= 1 && w.dim() == 2, "fp4.linear needs x [..., K] and a 2-d weight, got ", x.sizes(), " and ",
          w.sizes());
  const int64_t N = w.size(0), K = x.size(-1);
  REQUIRE(!bias || (bias->sizes() == at::IntArrayRef({N}) && bias->scalar_type() == x.scalar_type()), "bias must be ",
          x.scalar_type(), " [", N, "], got ", bias->scalar_type(), " ", bias->sizes());
  if (!w_scale) {
    REQUIRE(is_type(w.scalar_type()), "fp4.linear needs w_scale for a ", w.scalar_type(), " weight");
    REQUIRE(w.size(1) == K, "fp4.linear needs [..., K] and [N, K], got ", x.sizes(), " and ", w.sizes());
  } else {
    REQUIRE(w.scalar_type() == kF4 && w_scale->scalar_type() == kE8 &&
                w.sizes() == at::IntArrayRef({N, pairs(K)}) && w_scale->sizes() == at::IntArrayRef({N, mx_blocks(K)}),
            "fp4.linear needs a float4_e2m1fn_x2 weight ", at::IntArrayRef({N, pairs(K)}), " with float8_e8m0fnu ",
            at::IntArrayRef({N, mx_blocks(K)}), " scales, got ", w.scalar_type(), " ", w.sizes(), " with ",
            w_scale->scalar_type(), " ", w_scale->sizes());
  }
  if (x.numel() == 0 || N == 0) {  // nothing to multiply: torch gives the empty (or zero) result and its gradients
    const Tensor wt = w_scale ? at::zeros({N, K}, x.options().requires_grad(false)) : w.to(x.scalar_type());
    const Tensor y = at::matmul(x, wt.t());
    return bias ? y + *bias : y;
  }
  const bool grad = c10::GradMode::is_enabled();
  Maybe b;
  if (bias) b = bias->contiguous();
  if (!w_scale) {
    if (grad && (x.requires_grad() || w.requires_grad() || (b && b->requires_grad()))) return Train4::apply(x, w, b);
    Quantised4 xt, wt;
    return train_forward4(x, w, b, false, false, &xt, &wt);
  }
  if (grad && (x.requires_grad() || (b && b->requires_grad()))) return Stored4::apply(x, w, *w_scale, b);
  return stored_linear4(x, w, *w_scale, b);
}

}  // namespace
