// The torch side of the microscaled 4-bit operators (f16acc_amd.fp4).
#pragma once

#include "torch_common.h"

namespace {

constexpr int64_t kMx = 32;
constexpr auto kF4 = at::ScalarType::Float4_e2m1fn_x2;  // two values
constexpr auto kE8 = at::ScalarType::Float8_e8m0fnu;
int64_t pairs(int64_t v) { return (v + 1) / 2; }
int64_t mx_blocks(int64_t v) { return (v + kMx - 1) / kMx; }

// The bytes of a 4-bit operand or of scales (torch has few functions for their types).
Tensor as_bytes(const Tensor& t) { return t.detach().view(at::kByte); }

// An operand of a product: rows of `ld` bytes, the scales' dword of (row, quad of blocks) at row * row + quad * quad
// bytes, or, where quad is 0, the byte of (row, block) at row * row + block * block.
struct Operand4 {
  Tensor q, s;
  int64_t ld, row, block, quad;
};

// x's row blocks, and those of x transposed, from one pass; the scales in the products' order.
std::pair<Operand4, Operand4> quant4(const Tensor& x, bool rows, bool cols) {
  const int64_t M = x.size(0), K = x.size(1), qm = blocks(M), qk = blocks(K);
  Operand4 r{}, c{};
  if (rows) r = {empty({M, 64 * qk}, x, at::kByte), empty({qk, M}, x, at::kInt), 64 * qk, 4, 1, 4 * M};
  if (cols) c = {empty({K, 64 * qm}, x, at::kByte), empty({qm, K}, x, at::kInt), 64 * qm, 4, 1, 4 * K};
  const On on(x);
  check_rc(f16acc_fp4_quant(x.const_data_ptr(), type_of(x), M, K, x.stride(0), x.stride(1), bytes(r.q), r.ld,
                            bytes(r.s), r.row, r.quad, bytes(c.q), c.ld, bytes(c.s), c.row, c.quad, on.stream));
  return {r, c};
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
  uint8_t *to = bytes(q), *scales = bytes(s), *none = nullptr;
  const On on(x);
  check_rc(f16acc_fp4_quant(x2.const_data_ptr(), type_of(x), M, K, x2.stride(0), x2.stride(1), transposed ? none : to,
                            ld, scales, lds, 4, transposed ? to : none, ld, scales, lds, 4, on.stream));
  const Tensor qn = q.narrow(1, 0, pairs(C)), sn = s.narrow(1, 0, mx_blocks(C));
  if (transposed) return {qn, sn};
  return {qn.view(with_last(x, pairs(C))), sn.view(with_last(x, mx_blocks(C)))};
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
  const Tensor out = empty(with_last(q, C), q, dtype), q2 = rows_of(as_bytes(q)), s2 = rows_of(as_bytes(s));
  const On on(q);
  check_rc(f16acc_fp4_values(bytes(q2), q2.stride(0), q2.stride(1), bytes(s2), s2.stride(0), s2.stride(1), q2.size(0),
                             C, out.data_ptr(), type_of(out), on.stream));
  return out;
}

// Bytes [rows, pairs] as the products read them: themselves, or a copy whose rows are 16-byte aligned and zero to
// the next multiple of 16 bytes.
Operand packed4(const Tensor& q) {
  const int64_t rows = q.size(0), n = q.size(1), ld = rows > 1 ? q.stride(0) : up(n, 16);
  if (n % 16 == 0 && (q.stride(1) == 1 || n <= 1) && ld >= n && ld % 16 == 0 && ld <= kMaxRow &&
      (uintptr_t)q.const_data_ptr() % 16 == 0)
    return {q, ld};
  const Tensor out = empty({rows, up(n, 16)}, q, at::kByte);
  const On on(q);
  check_rc(f16acc_pack8(bytes(q), bytes(out), rows, n, q.stride(0), q.stride(1), up(n, 16), on.stream));
  return {out, up(n, 16)};
}
Operand4 stored4(const Tensor& q, const Tensor& s) {
  const Operand o = packed4(q);
  return {o.q, s, o.ld, s.stride(0), s.stride(1), 0};
}

// out [M, N] from x [M, K] and w [N, K].
void product4(const Operand4& x, const Operand4& w, int64_t K, const Tensor& out, const Maybe& bias = {}, int tile = -1,
              int splits = 0) {
  const int64_t M = out.size(0), N = out.size(1);
  const size_t n = f16acc_mm_fp4_workspace(M, N, K, x.quad, w.quad, tile, splits);
  Tensor ws;
  if (n) ws = empty({(int64_t)n}, out, at::kByte);
  const On on(out);
  check_rc(f16acc_mm_fp4(bytes(x.q), x.ld, bytes(x.s), x.row, x.block, x.quad, bytes(w.q), w.ld, bytes(w.s), w.row,
                         w.block, w.quad, data(bias), out.data_ptr(), out.stride(0), out.stride(1), M, N, K,
                         type_of(out), tile, splits, bytes(ws), n, on.stream));
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
  product4(stored4(as_bytes(a), as_bytes(a_scale)), stored4(as_bytes(b).t(), as_bytes(b_scale).t()), K, out, b_, tile,
           splits);
  return out;
}

// y = x w^T + bias; dx = dy w, dw = dy^T x, each from operands quantised along its own contraction.
Tensor train_forward4(const Tensor& x, const Tensor& w, const Maybe& bias, bool need_x, bool need_w, Operand4* xt,
                      Operand4* wt) {
  const Tensor x2 = rows_of(x);
  const auto [xr, xc] = quant4(x2, true, need_w);
  const auto [wr, wc] = quant4(w, true, need_x);
  *xt = xc, *wt = wc;
  const Tensor y = empty(with_last(x, w.size(0)), x, x.scalar_type());
  product4(xr, wr, x2.size(1), y.view({x2.size(0), w.size(0)}), bias);
  return y;
}

// An operand kept for the backward pass: rows [rows][64 quads], scales [quads][rows].
Operand4 kept4(const Tensor& q, const Tensor& s) { return {q, s, q.size(1), 4, 1, 4 * q.size(0)}; }

struct Train4 : torch::autograd::Function<Train4> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& bias) {
    Operand4 xt{}, wt{};
    const Tensor y = train_forward4(x, w, bias, x.requires_grad(), w.requires_grad(), &xt, &wt);
    ctx->save_for_backward({xt.q, xt.s, wt.q, wt.s});
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["dtype"] = (int64_t)w.scalar_type();
    ctx->saved_data["need"] = (int64_t)x.requires_grad() + 2 * (int64_t)w.requires_grad() +
                              4 * (int64_t)(bias && bias->requires_grad());
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_derivative_only();
    const auto saved = ctx->get_saved_variables();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const int64_t need = ctx->saved_data["need"].toInt(), K = shape.back();
    const Tensor dy = rows_of(check_grad("fp4.linear", grads[0]));
    const int64_t M = dy.size(0), N = dy.size(1);
    Operand4 r{}, c{};
    if (need & 3) std::tie(r, c) = quant4(dy, need & 1, need & 2);
    Tensor dx, dw, db;
    if (need & 1) {
      dx = empty({M, K}, dy, dy.scalar_type());
      product4(r, kept4(saved[2], saved[3]), N, dx);
      dx = dx.view(shape);
    }
    if (need & 2) {
      dw = empty({N, K}, dy, (at::ScalarType)ctx->saved_data["dtype"].toInt());
      product4(c, kept4(saved[0], saved[1]), M, dw);
    }
    if (need & 4) db = column_sums(dy);
    return {dx, dw, db};
  }
};

Tensor stored_linear4(const Tensor& x, const Tensor& w, const Tensor& w_scale, const Maybe& bias) {
  const Tensor x2 = rows_of(x), q = as_bytes(w), s = as_bytes(w_scale);
  const int64_t M = x2.size(0), K = x2.size(1), N = w.size(0), P = pairs(K);
  // rows of any alignment go as they are (the library copies them where it has to)
  const bool rows = (P <= 1 || q.stride(1) == 1) && (N <= 1 || q.stride(0) >= P);
  const Operand o = rows ? Operand{q, N > 1 ? q.stride(0) : up(P, 16)} : packed4(q);
  Tensor y = empty(with_last(x, N), x, x.scalar_type());
  const size_t n = f16acc_linear_fp4_workspace(M, N, K, bytes(o.q), o.ld);
  const Tensor ws = empty({(int64_t)n}, x, at::kByte);
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
      const Tensor q = as_bytes(saved[0]), s = as_bytes(saved[1]);
      const int64_t qn = blocks(N);
      const Operand4 wt{empty({K, 64 * qn}, dy, at::kByte), empty({qn, K}, dy, at::kInt), 64 * qn, 4, 1, 4 * K};
      const Operand4 r = quant4(dy, true, false).first;
      dx = empty({dy.size(0), K}, dy, dy.scalar_type());
      {
        const On on(dy);
        check_rc(f16acc_fp4_transpose(bytes(q), q.stride(0), q.stride(1), bytes(s), s.stride(0), s.stride(1), N, K,
                                      bytes(wt.q), wt.ld, bytes(wt.s), wt.row, wt.quad, on.stream));
      }
      product4(r, wt, N, dx);
      dx = dx.view(shape);
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
    Operand4 xt{}, wt{};
    return train_forward4(x, w, b, false, false, &xt, &wt);
  }
  if (grad && (x.requires_grad() || (b && b->requires_grad()))) return Stored4::apply(x, w, *w_scale, b);
  return stored_linear4(x, w, *w_scale, b);
}

}  // namespace
