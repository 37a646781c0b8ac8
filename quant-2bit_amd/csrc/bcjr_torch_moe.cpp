// Torch operators of the mixture-of-experts products, routing and distillation:
// HIP-device and Meta kernels over the C ABI, and the autograd formulas in C++
// (a single token's call pays for no Python autograd layer).
#include "bcjr_torch.h"

#include <torch/csrc/autograd/custom_function.h>

#include <limits>
#include <tuple>

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

int dtype_id(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return BCJR_F32;
    case at::kBFloat16: return BCJR_BF16;
    case at::kHalf: return BCJR_F16;
    default: TORCH_CHECK(false, name, " must be float32, bfloat16 or float16; got ", t.scalar_type());
  }
}

// t with rows that a kernel can walk by a row stride: unit stride within a row,
// rows that do not overlap.
Tensor strided_rows(const Tensor& t) {
  return t.stride(1) == 1 && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) ? t : t.contiguous();
}
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

const int32_t* iptr(const OptTensor& t) { return t ? t->data_ptr<int32_t>() : nullptr; }

Tensor as_int(const Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64; got ",
              t.scalar_type());
  return t.to(at::kInt).contiguous();
}
OptTensor as_int(const OptTensor& t, const char* name) {
  if (!t) return std::nullopt;
  return as_int(*t, name);
}

void need_2d(const Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() == 2, name, " must be 2-D; got ", t.sizes());
}

// -------------------------------------------------------------------- routing

using RouteOut = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

void route_args(const Tensor& logits, const OptTensor& valid, int64_t k) {
  need_2d(logits, "logits");
  const int64_t T = logits.size(0), E = logits.size(1);
  TORCH_CHECK(k >= 1 && k <= E, "top_k=", k, " outside [1, E=", E, "]");
  if (valid)
    TORCH_CHECK(valid->dim() == 1 && valid->size(0) == T && valid->scalar_type() == at::kBool, "valid must be (", T,
                ",) bool; got ", valid->sizes(), " ", valid->scalar_type());
}

RouteOut route_outputs(const Tensor& logits, int64_t k) {
  const int64_t T = logits.size(0), E = logits.size(1);
  const auto i32 = logits.options().dtype(at::kInt);
  return {at::empty({T, k}, logits.options().dtype(at::kFloat)), at::empty({T, k}, i32), at::empty({E + 1}, i32),
          at::empty({T * k}, i32), at::empty({T, k}, i32)};
}

const uint8_t* mask_ptr(const OptTensor& valid) {
  return valid ? reinterpret_cast<const uint8_t*>(valid->data_ptr<bool>()) : nullptr;
}

RouteOut moe_route_hip(const Tensor& logits_in, const OptTensor& valid_in, int64_t k, bool renormalize) {
  route_args(logits_in, valid_in, k);
  same_device(logits_in, valid_in, "valid");
  const c10::OptionalDeviceGuard guard(at::device_of(logits_in));
  const int dtype = dtype_id(logits_in, "logits");
  const Tensor logits = strided_rows(logits_in);
  const OptTensor valid = valid_in ? OptTensor(valid_in->contiguous()) : std::nullopt;
  const int64_t T = logits.size(0), E = logits.size(1);
  RouteOut out = route_outputs(logits, k);
  auto& [weights, experts, offsets, rows, slots] = out;
  size_t bytes = 0;
  check(bcjr_moe_route_workspace(T, E, &bytes), "bcjr_moe_route_workspace");
  Tensor ws;
  if (bytes) ws = at::empty({(int64_t)bytes}, logits.options().dtype(at::kByte));
  check(bcjr_moe_route(logits.data_ptr(), dtype, row_stride(logits), mask_ptr(valid), T, E, (int)k, renormalize,
                       weights.data_ptr<float>(), experts.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(),
                       rows.data_ptr<int32_t>(), slots.data_ptr<int32_t>(), bytes ? ws.data_ptr() : nullptr, bytes,
                       stream_of(logits)),
        "bcjr_moe_route");
  return out;
}

RouteOut moe_route_meta(const Tensor& logits, const OptTensor& valid, int64_t k, bool renormalize) {
  route_args(logits, valid, k);
  return route_outputs(logits, k);
}

Tensor moe_route_backward_hip(const Tensor& logits_in, const OptTensor& valid_in, const Tensor& weights,
                              const Tensor& experts, const Tensor& g_in, bool renormalize) {
  const int64_t T = logits_in.size(0), E = logits_in.size(1), k = weights.size(1);
  TORCH_CHECK(g_in.sizes() == weights.sizes(), "g_weights must be ", weights.sizes(), "; got ", g_in.sizes());
  same_device(logits_in, g_in, "g_weights");
  const c10::OptionalDeviceGuard guard(at::device_of(logits_in));
  const Tensor logits = strided_rows(logits_in), g = g_in.to(at::kFloat).contiguous();
  const Tensor wc = weights.contiguous(), ec = experts.contiguous();
  const OptTensor valid = valid_in ? OptTensor(valid_in->contiguous()) : std::nullopt;
  Tensor out = at::empty({T, E}, logits.options());
  check(bcjr_moe_route_backward(logits.data_ptr(), dtype_id(logits, "logits"), row_stride(logits), mask_ptr(valid), T,
                                E, (int)k, renormalize, wc.data_ptr<float>(), ec.data_ptr<int32_t>(),
                                g.data_ptr<float>(), out.data_ptr(), stream_of(logits)),
        "bcjr_moe_route_backward");
  return out;
}

Tensor moe_route_backward_meta(const Tensor& logits, const OptTensor&, const Tensor&, const Tensor&, const Tensor&,
                               bool) {
  return at::empty(logits.sizes(), logits.options());
}

RouteOut call_route(const Tensor& logits, const OptTensor& valid, int64_t k, bool renormalize) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("bcjr::moe_route", "")
                       .typed<RouteOut(const Tensor&, const OptTensor&, int64_t, bool)>();
  at::AutoDispatchBelowADInplaceOrView guard;
  return op.call(logits, valid, k, renormalize);
}

struct RouteFunction : torch::autograd::Function<RouteFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& valid, int64_t k,
                               bool renormalize) {
    auto [w, experts, offsets, rows, slots] = call_route(logits, valid, k, renormalize);
    ctx->save_for_backward({logits, valid ? *valid : Tensor(), w, experts});
    ctx->saved_data["renormalize"] = renormalize;
    ctx->mark_non_differentiable({experts, offsets, rows, slots});
    return {w, experts, offsets, rows, slots};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("bcjr::moe_route_backward", "")
                         .typed<Tensor(const Tensor&, const OptTensor&, const Tensor&, const Tensor&, const Tensor&,
                                       bool)>();
    const auto s = ctx->get_saved_variables();
    if (!g[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const OptTensor valid = s[1].defined() ? OptTensor(s[1]) : std::nullopt;
    return {op.call(s[0], valid, s[2], s[3], g[0], ctx->saved_data["renormalize"].toBool()), Tensor(), Tensor(),
            Tensor()};
  }
};

bool wants_grad(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

RouteOut moe_route_autograd(const Tensor& logits, const OptTensor& valid, int64_t k, bool renormalize) {
  if (!wants_grad(logits)) return call_route(logits, valid, k, renormalize);
  auto o = RouteFunction::apply(logits, valid, k, renormalize);
  return {o[0], o[1], o[2], o[3], o[4]};
}

// ----------------------------------------------------------- grouped products

// Whether t's rows (of a 16-bit type) are 16-byte chunks: a row stride in eights and
// an aligned start.  (By the offset in the storage, which tracing knows too; where
// a storage itself is not aligned the slow kernel runs.)
bool chunked(const Tensor& t) {
  const int64_t d = t.dim();
  return t.stride(d - 1) == 1 && t.stride(d - 2) % 8 == 0 && t.storage_offset() % 8 == 0;
}
// Row stride of rows with zeros behind them.
int64_t chunk_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : (t.size(1) + 7) / 8 * 8; }

// Rows (the last dimension) of t in `dtype` at a stride in eights with zeros
// behind them: a view of t's sizes into a padded copy.
Tensor padded(const Tensor& t, at::ScalarType dtype) {
  const Tensor c = t.dim() == 2 ? strided_rows(t) : t.contiguous();
  const int64_t n = t.size(-1), rows = n ? t.numel() / n : 0, ld = (n + 7) / 8 * 8;
  auto sizes = t.sizes().vec();
  sizes.back() = ld;
  Tensor out = at::empty(sizes, t.options().dtype(dtype));
  check(bcjr_pad_rows(c.data_ptr(), dtype_id(c, "x"), t.dim() == 2 ? row_stride(c) : n, rows, n, dtype_id(out, "x"),
                      out.data_ptr(), ld, stream_of(t)),
        "bcjr_pad_rows");
  return out.narrow(-1, 0, n);
}
Tensor pad_rows_hip(const Tensor& t, const Tensor& like) {
  const c10::OptionalDeviceGuard guard(at::device_of(t));
  return padded(t, like.scalar_type());
}
Tensor pad_rows_meta(const Tensor& t, const Tensor& like) {
  auto sizes = t.sizes().vec();
  sizes.back() = (sizes.back() + 7) / 8 * 8;
  return at::empty(sizes, t.options().dtype(like.scalar_type())).narrow(-1, 0, t.size(-1));
}

// Shapes of a product: x (T or M, K), w (E, N, K) or (E, K, N), offsets (E + 1), rows (M).
struct Product {
  int64_t E, M, N, K;
};
Product product_args(const Tensor& x, const Tensor& w, const Tensor& offsets, const OptTensor& rows, bool w_is_nk) {
  need_2d(x, "x");
  TORCH_CHECK(w.dim() == 3, "w must be 3-D; got ", w.sizes());
  Product p = {w.size(0), rows ? rows->numel() : x.size(0), w.size(w_is_nk ? 1 : 2), w.size(w_is_nk ? 2 : 1)};
  TORCH_CHECK(x.size(1) == p.K, "x has rows of ", x.size(1), ", w of ", p.K);
  TORCH_CHECK(w.scalar_type() == x.scalar_type(), "w is ", w.scalar_type(), ", x ", x.scalar_type());
  TORCH_CHECK(offsets.dim() == 1 && offsets.size(0) == p.E + 1, "offsets must be (E+1=", p.E + 1, ",); got ",
              offsets.sizes());
  if (rows) TORCH_CHECK(rows->dim() == 1, "rows must be 1-D; got ", rows->sizes());
  return p;
}

// zero_padded: x and w are chunked, with zeros behind rows that are not whole chunks.
Tensor grouped_matmul_hip(const Tensor& x_in, const Tensor& w_in, const Tensor& offsets_in, const OptTensor& rows_in,
                          bool w_is_nk, bool zero_padded) {
  const Product p = product_args(x_in, w_in, offsets_in, rows_in, w_is_nk);
  same_device(x_in, w_in, "w");
  same_device(x_in, offsets_in, "offsets");
  same_device(x_in, rows_in, "rows");
  const c10::OptionalDeviceGuard guard(at::device_of(x_in));
  const Tensor x = strided_rows(x_in), offsets = as_int(offsets_in, "offsets");
  const bool rows_ok = w_in.stride(2) == 1 && w_in.stride(1) >= w_in.size(2) &&
                       w_in.stride(0) == w_in.size(1) * w_in.stride(1);
  const Tensor w = rows_ok ? w_in : w_in.contiguous();
  const OptTensor rows = as_int(rows_in, "rows");
  Tensor out = at::empty({p.M, p.N}, x.options());
  check(bcjr_grouped_matmul(x.data_ptr(), dtype_id(x, "x"), zero_padded ? chunk_stride(x) : row_stride(x), x.size(0),
                            iptr(rows), w.data_ptr(), w.stride(1), w_is_nk, offsets.data_ptr<int32_t>(), p.E, p.M, p.N,
                            p.K, zero_padded, out.data_ptr(), stream_of(x)),
        "bcjr_grouped_matmul");
  return out;
}

Tensor grouped_matmul_meta(const Tensor& x, const Tensor& w, const Tensor& offsets, const OptTensor& rows,
                           bool w_is_nk, bool zero_padded) {
  const Product p = product_args(x, w, offsets, rows, w_is_nk);
  return at::empty({p.M, p.N}, x.options());
}

// The product on float32 weights w (E, N, K), and the weights rounded to x's type
// (of the experts that have places; empty without keep).
std::tuple<Tensor, Tensor> grouped_f32w_hip(const Tensor& x_in, const Tensor& w_in, const Tensor& offsets_in,
                                            const OptTensor& rows_in, bool keep) {
  TORCH_CHECK(w_in.dim() == 3 && x_in.dim() == 2 && x_in.size(1) == w_in.size(2), "x must be (rows, K), w (E, N, K); got ",
              x_in.sizes(), ", ", w_in.sizes());
  TORCH_CHECK(w_in.scalar_type() == at::kFloat, "w must be float32; got ", w_in.scalar_type());
  TORCH_CHECK(offsets_in.dim() == 1 && offsets_in.size(0) == w_in.size(0) + 1, "offsets must be (E+1=", w_in.size(0) + 1,
              ",); got ", offsets_in.sizes());
  same_device(x_in, w_in, "w");
  same_device(x_in, offsets_in, "offsets");
  same_device(x_in, rows_in, "rows");
  const c10::OptionalDeviceGuard guard(at::device_of(x_in));
  const Tensor x = strided_rows(x_in), w = w_in.contiguous(), offsets = as_int(offsets_in, "offsets");
  const OptTensor rows = as_int(rows_in, "rows");
  const int64_t E = w.size(0), N = w.size(1), K = w.size(2), M = rows ? rows->numel() : x.size(0);
  Tensor out = at::empty({M, N}, x.options());
  Tensor copy = keep ? at::empty({E, N, K}, x.options()) : at::empty({0}, x.options());
  check(bcjr_grouped_matmul_f32w(x.data_ptr(), dtype_id(x, "x"), row_stride(x), x.size(0), iptr(rows),
                                 w.data_ptr<float>(), K, offsets.data_ptr<int32_t>(), E, M, N, K, out.data_ptr(),
                                 keep ? copy.data_ptr() : nullptr, stream_of(x)),
        "bcjr_grouped_matmul_f32w");
  return {out, copy};
}

std::tuple<Tensor, Tensor> grouped_f32w_meta(const Tensor& x, const Tensor& w, const Tensor& offsets,
                                             const OptTensor& rows, bool keep) {
  return {at::empty({rows ? rows->numel() : x.size(0), w.size(1)}, x.options()),
          keep ? at::empty(w.sizes(), x.options()) : at::empty({0}, x.options())};
}

void wgrad_args(const Tensor& gy, const Tensor& x, const Tensor& offsets, const OptTensor& rows) {
  need_2d(gy, "gy");
  need_2d(x, "x");
  TORCH_CHECK(gy.scalar_type() == x.scalar_type(), "gy is ", gy.scalar_type(), ", x ", x.scalar_type());
  TORCH_CHECK(offsets.dim() == 1 && offsets.size(0) >= 2, "offsets must be (E+1,); got ", offsets.sizes());
  TORCH_CHECK(gy.size(0) == (rows ? rows->numel() : x.size(0)), "gy has ", gy.size(0), " rows");
}

Tensor grouped_wgrad_hip(const Tensor& gy_in, const Tensor& x_in, const Tensor& offsets_in, const OptTensor& rows_in,
                         bool zero_padded, bool out_f32) {
  wgrad_args(gy_in, x_in, offsets_in, rows_in);
  same_device(x_in, gy_in, "gy");
  same_device(x_in, offsets_in, "offsets");
  same_device(x_in, rows_in, "rows");
  const c10::OptionalDeviceGuard guard(at::device_of(x_in));
  const Tensor gy = strided_rows(gy_in), x = strided_rows(x_in), offsets = as_int(offsets_in, "offsets");
  const OptTensor rows = as_int(rows_in, "rows");
  const int64_t E = offsets.size(0) - 1, M = gy.size(0), N = gy.size(1), K = x.size(1);
  Tensor out = at::empty({E, N, K}, out_f32 ? x.options().dtype(at::kFloat) : x.options());
  check(bcjr_grouped_wgrad(gy.data_ptr(), dtype_id(x, "x"), zero_padded ? chunk_stride(gy) : row_stride(gy), x.data_ptr(),
                           zero_padded ? chunk_stride(x) : row_stride(x), x.size(0), iptr(rows),
                           offsets.data_ptr<int32_t>(), E, M, N, K, zero_padded, out_f32, out.data_ptr(),
                           stream_of(x)),
        "bcjr_grouped_wgrad");
  return out;
}

Tensor grouped_wgrad_meta(const Tensor& gy, const Tensor& x, const Tensor& offsets, const OptTensor& rows,
                          bool zero_padded, bool out_f32) {
  wgrad_args(gy, x, offsets, rows);
  return at::empty({offsets.size(0) - 1, gy.size(1), x.size(1)}, out_f32 ? x.options().dtype(at::kFloat) : x.options());
}

Tensor call_grouped(const Tensor& x, const Tensor& w, const Tensor& offsets, const OptTensor& rows, bool w_is_nk,
                    bool zero_padded) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("bcjr::grouped_product", "")
                       .typed<Tensor(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, bool, bool)>();
  return op.call(x, w, offsets, rows, w_is_nk, zero_padded);
}

Tensor call_wgrad(const Tensor& gy, const Tensor& x, const Tensor& offsets, const OptTensor& rows, bool zero_padded,
                  bool out_f32) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("bcjr::grouped_wgrad", "")
                       .typed<Tensor(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, bool, bool)>();
  return op.call(gy, x, offsets, rows, zero_padded, out_f32);
}

Tensor call_pad(const Tensor& t, const Tensor& like) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("bcjr::pad_rows", "")
                       .typed<Tensor(const Tensor&, const Tensor&)>();
  return op.call(t, like);
}

std::tuple<Tensor, Tensor> call_f32w(const Tensor& x, const Tensor& w, const Tensor& offsets, const OptTensor& rows,
                                     bool keep) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("bcjr::grouped_product_f32w", "")
                       .typed<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const OptTensor&,
                                                         bool)>();
  return op.call(x, w, offsets, rows, keep);
}

// Whether the product reads float32 weights themselves: rows in 16-byte chunks, and
// gathered rows within a buffer's reach.
bool reads_f32(const Tensor& x, const Tensor& w) {
  return w.scalar_type() == at::kFloat && x.scalar_type() != at::kFloat && x.size(1) % 8 == 0 && chunked(x) &&
         w.is_contiguous() && w.storage_offset() % 4 == 0 && x.size(0) * x.stride(0) < (int64_t(1) << 31) - 16;
}

Tensor call_combine(const Tensor& y, const OptTensor& weights, const Tensor& slots);

// t in `like`'s type with rows of 16-byte chunks: t itself, a converted copy or a padded one.
Tensor in_chunks(const Tensor& t, const Tensor& like) {
  if (t.size(-1) % 8 == 0) {
    const Tensor c = t.to(like.scalar_type());
    if (chunked(c)) return c;
  }
  return call_pad(t, like);
}

struct GroupedFunction : torch::autograd::Function<GroupedFunction> {
  static Variable forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& offsets,
                          const OptTensor& rows, const OptTensor& slots) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->saved_data["w_f32"] = w.scalar_type() == at::kFloat;
    if (reads_f32(x, w)) {
      auto [y, wx] = call_f32w(x, w, offsets, rows, ctx->needs_input_grad(0));
      ctx->save_for_backward({x, wx, offsets, rows ? *rows : Tensor(), slots ? *slots : Tensor()});
      return y;
    }
    // copies of float32 weights and of rows that are not 16-byte chunks serve the backward too
    const Tensor wx = in_chunks(w, x), xx = in_chunks(x, x);
    ctx->save_for_backward({xx, wx, offsets, rows ? *rows : Tensor(), slots ? *slots : Tensor()});
    return call_grouped(xx, wx, offsets, rows, true, x.size(1) % 8 != 0);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &offsets = s[2];
    const OptTensor rows = s[3].defined() ? OptTensor(s[3]) : std::nullopt;
    Tensor gx, gw;
    if (g[0].defined()) {
      const Tensor gy = in_chunks(g[0].dim() == 2 ? strided_rows(g[0]) : g[0], x);
      const bool pad = x.size(1) % 8 != 0 || gy.size(1) % 8 != 0;
      if (ctx->needs_input_grad(0)) {
        gx = call_grouped(gy, w, offsets, std::nullopt, false, pad);
        // the places' gradients, rounded to the rows' type, summed in float32 over each row's places
        if (rows) gx = call_combine(gx, std::nullopt, s[4]);
      }
      if (ctx->needs_input_grad(1)) gw = call_wgrad(gy, x, offsets, rows, pad, ctx->saved_data["w_f32"].toBool());
    }
    return {gx, gw, Tensor(), Tensor(), Tensor()};
  }
};

// x may be gathered through rows; slots (T, k) are rows' inverse, for x's gradient.
void grouped_args(const Tensor& x, const Tensor& w, const OptTensor& rows, const OptTensor& slots) {
  TORCH_CHECK(w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat, "w must be ", x.scalar_type(),
              " like x, or float32; got ", w.scalar_type());
  if (rows && wants_grad(x)) {
    TORCH_CHECK(slots.has_value(), "the gradient of gathered rows needs slots");
    TORCH_CHECK(slots->dim() == 2 && slots->size(0) == x.size(0), "slots must be (", x.size(0), ", k); got ",
                slots->sizes());
  }
}

Tensor grouped_matmul(const Tensor& x, const Tensor& w, const Tensor& offsets, const OptTensor& rows,
                      const OptTensor& slots) {
  grouped_args(x, w, rows, slots);
  const bool half = x.scalar_type() != at::kFloat;
  if (half && (wants_grad(x) || wants_grad(w))) return GroupedFunction::apply(x, w, offsets, rows, slots);
  at::AutoDispatchBelowADInplaceOrView guard;
  if (reads_f32(x, w)) return std::get<0>(call_f32w(x, w, offsets, rows, false));
  const int64_t M = rows ? rows->numel() : x.size(0);
  // Rows that are not 16-byte chunks: a padded copy of all weights pays once the
  // experts have rows enough or the weights are small (or copied in any case);
  // else the slow kernel reads the weights of the experts in use alone.  Padded /
  // slow, microseconds, bfloat16: 64 experts of 1023 x 2047, 512 rows 175 / 145,
  // 2,048 rows 183 / 253; 8 experts of 1001 x 1003, 8 rows 20 / 53.
  if (half && (M >= 16 * w.size(0) || w.numel() < (1 << 25) || w.scalar_type() == at::kFloat))
    return call_grouped(in_chunks(x, x), in_chunks(w, x), offsets, rows, true, x.size(1) % 8 != 0);
  return call_grouped(x, w.to(x.scalar_type()), offsets, rows, true, false);
}

// -------------------------------------------------------------------- combine

void combine_args(const Tensor& y, const OptTensor& weights, const Tensor& slots) {
  need_2d(y, "y");
  need_2d(slots, "slots");
  TORCH_CHECK(slots.size(1) >= 1, "slots must name a place per token; got ", slots.sizes());
  if (weights)
    TORCH_CHECK(weights->sizes() == slots.sizes(), "weights must be ", slots.sizes(), "; got ", weights->sizes());
}

Tensor moe_combine_hip(const Tensor& y_in, const OptTensor& weights_in, const Tensor& slots_in) {
  combine_args(y_in, weights_in, slots_in);
  same_device(y_in, weights_in, "weights");
  same_device(y_in, slots_in, "slots");
  const c10::OptionalDeviceGuard guard(at::device_of(y_in));
  const Tensor y = strided_rows(y_in), slots = as_int(slots_in, "slots");
  Tensor w;
  if (weights_in) w = weights_in->to(at::kFloat).contiguous();
  const int64_t T = slots.size(0), k = slots.size(1), M = y.size(0), N = y.size(1);
  Tensor out = at::empty({T, N}, y.options());
  check(bcjr_moe_combine(y.data_ptr(), dtype_id(y, "y"), row_stride(y), weights_in ? w.data_ptr<float>() : nullptr,
                         slots.data_ptr<int32_t>(), T, (int)k, M, N, out.data_ptr(), stream_of(y)),
        "bcjr_moe_combine");
  return out;
}

Tensor moe_combine_meta(const Tensor& y, const OptTensor& weights, const Tensor& slots) {
  combine_args(y, weights, slots);
  return at::empty({slots.size(0), y.size(1)}, y.options());
}

std::tuple<Tensor, Tensor> moe_combine_backward_hip(const Tensor& y_in, const Tensor& weights_in,
                                                    const Tensor& rows_in, const Tensor& slots_in,
                                                    const Tensor& g_in) {
  combine_args(y_in, weights_in, slots_in);
  const c10::OptionalDeviceGuard guard(at::device_of(y_in));
  const Tensor y = strided_rows(y_in), slots = as_int(slots_in, "slots"), rows = as_int(rows_in, "rows");
  const Tensor w = weights_in.to(at::kFloat).contiguous(), g = strided_rows(g_in.to(y.scalar_type()));
  const int64_t T = slots.size(0), k = slots.size(1), M = y.size(0), N = y.size(1);
  TORCH_CHECK(rows.numel() == M, "rows must be (", M, ",); got ", rows.sizes());
  TORCH_CHECK(g.dim() == 2 && g.size(0) == T && g.size(1) == N, "g_out must be (", T, ", ", N, "); got ", g.sizes());
  Tensor gy = at::empty({M, N}, y.options()), gw = at::empty({T, k}, w.options());
  check(bcjr_moe_combine_backward(y.data_ptr(), dtype_id(y, "y"), row_stride(y), w.data_ptr<float>(),
                                  slots.data_ptr<int32_t>(), rows.data_ptr<int32_t>(), g.data_ptr(), row_stride(g), T,
                                  (int)k, M, N, gy.data_ptr(), gw.data_ptr<float>(), stream_of(y)),
        "bcjr_moe_combine_backward");
  return {gy, gw};
}

std::tuple<Tensor, Tensor> moe_combine_backward_meta(const Tensor& y, const Tensor& weights, const Tensor& rows,
                                                     const Tensor& slots, const Tensor& g) {
  return {at::empty(y.sizes(), y.options()), at::empty(slots.sizes(), y.options().dtype(at::kFloat))};
}

Tensor call_combine(const Tensor& y, const OptTensor& weights, const Tensor& slots) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("bcjr::combine", "")
                       .typed<Tensor(const Tensor&, const OptTensor&, const Tensor&)>();
  return op.call(y, weights, slots);
}

struct CombineFunction : torch::autograd::Function<CombineFunction> {
  static Variable forward(AutogradContext* ctx, const Tensor& y, const Tensor& weights, const Tensor& rows,
                          const Tensor& slots) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({y, weights, rows, slots});
    return call_combine(y, weights, slots);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("bcjr::combine_backward", "")
                         .typed<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                           const Tensor&)>();
    const auto s = ctx->get_saved_variables();
    if (!g[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    auto [gy, gw] = op.call(s[0], s[1], s[2], s[3], g[0]);
    return {gy, gw.to(s[1].scalar_type()), Tensor(), Tensor()};
  }
};

Tensor moe_combine(const Tensor& y, const Tensor& weights, const Tensor& rows, const Tensor& slots) {
  combine_args(y, weights, slots);
  TORCH_CHECK(rows.dim() == 1 && rows.size(0) == y.size(0) && y.size(0) == slots.numel(), "y has ", y.size(0),
              " rows, rows ", rows.sizes(), " places, slots ", slots.sizes(), ": all must be T*k");
  if (wants_grad(y) || wants_grad(weights)) return CombineFunction::apply(y, weights, rows, slots);
  at::AutoDispatchBelowADInplaceOrView guard;
  return call_combine(y, weights, slots);
}

// --------------------------------------------------------------- distillation

struct Distill {
  Tensor logits, values, indices, lse;
  int dtype;
  int64_t T, V, K;
};

void distill_args(const Tensor& logits, const Tensor& values, const Tensor& indices, const OptTensor& lse) {
  need_2d(logits, "logits");
  need_2d(values, "teacher values");
  const int64_t T = logits.size(0);
  TORCH_CHECK(values.size(0) == T, "teacher values must be (", T, ", K); got ", values.sizes());
  TORCH_CHECK(indices.sizes() == values.sizes(), "teacher indices must be ", values.sizes(), "; got ",
              indices.sizes());
  if (lse) TORCH_CHECK(lse->dim() == 1 && lse->size(0) == T, "teacher_lse must be (", T, ",); got ", lse->sizes());
}

Distill distill_inputs(const Tensor& logits, const Tensor& values, const Tensor& indices, const OptTensor& lse) {
  distill_args(logits, values, indices, lse);
  same_device(logits, values, "teacher values");
  same_device(logits, indices, "teacher indices");
  same_device(logits, lse, "teacher_lse");
  Distill d;
  d.dtype = dtype_id(logits, "logits");
  d.logits = strided_rows(logits);
  d.values = values.to(at::kFloat).contiguous();
  d.indices = as_int(indices, "teacher indices");
  if (lse) d.lse = lse->to(at::kFloat).contiguous();
  d.T = logits.size(0), d.V = logits.size(1), d.K = values.size(1);
  return d;
}

const float* lse_ptr(const Distill& d) { return d.lse.defined() ? d.lse.data_ptr<float>() : nullptr; }

// loss (T,) and, with keep, stats (T, 8) for the backward (else (0, 8)).
std::tuple<Tensor, Tensor> topk_distill_hip(const Tensor& logits, const Tensor& values, const Tensor& indices,
                                            const OptTensor& lse, double temperature, bool keep) {
  const c10::OptionalDeviceGuard guard(at::device_of(logits));
  const Distill d = distill_inputs(logits, values, indices, lse);
  const auto f32 = logits.options().dtype(at::kFloat);
  Tensor loss = at::empty({d.T}, f32), stats = at::empty({keep ? d.T : 0, 8}, f32);
  check(bcjr_topk_distill(d.logits.data_ptr(), d.dtype, row_stride(d.logits), d.values.data_ptr<float>(),
                          d.indices.data_ptr<int32_t>(), lse_ptr(d), (float)temperature, d.T, d.V, d.K,
                          loss.data_ptr<float>(), keep ? stats.data_ptr<float>() : nullptr, stream_of(logits)),
        "bcjr_topk_distill");
  return {loss, stats};
}

std::tuple<Tensor, Tensor> topk_distill_meta(const Tensor& logits, const Tensor& values, const Tensor& indices,
                                             const OptTensor& lse, double temperature, bool keep) {
  distill_args(logits, values, indices, lse);
  const auto f32 = logits.options().dtype(at::kFloat);
  return {at::empty({logits.size(0)}, f32), at::empty({keep ? logits.size(0) : 0, 8}, f32)};
}

Tensor topk_distill_backward_hip(const Tensor& logits, const Tensor& values, const Tensor& indices,
                                 double temperature, const Tensor& stats, const Tensor& g_loss) {
  const c10::OptionalDeviceGuard guard(at::device_of(logits));
  const Distill d = distill_inputs(logits, values, indices, std::nullopt);
  TORCH_CHECK(g_loss.dim() == 1 && g_loss.size(0) == d.T, "g_loss must be (", d.T, ",); got ", g_loss.sizes());
  const Tensor g = g_loss.to(at::kFloat).contiguous(), st = stats.contiguous();
  Tensor out = at::empty({d.T, d.V}, logits.options());
  check(bcjr_topk_distill_backward(d.logits.data_ptr(), d.dtype, row_stride(d.logits), d.values.data_ptr<float>(),
                                   d.indices.data_ptr<int32_t>(), (float)temperature, d.T, d.V, d.K,
                                   st.data_ptr<float>(), g.data_ptr<float>(), out.data_ptr(), stream_of(logits)),
        "bcjr_topk_distill_backward");
  return out;
}

Tensor topk_distill_backward_meta(const Tensor& logits, const Tensor&, const Tensor&, double, const Tensor&,
                                  const Tensor&) {
  return at::empty(logits.sizes(), logits.options());
}

std::tuple<Tensor, Tensor> topk_distill_both_hip(const Tensor& logits, const Tensor& values, const Tensor& indices,
                                                 const Tensor& g_loss, const OptTensor& lse, double temperature) {
  const c10::OptionalDeviceGuard guard(at::device_of(logits));
  const Distill d = distill_inputs(logits, values, indices, lse);
  same_device(logits, g_loss, "row_weights");
  TORCH_CHECK(g_loss.dim() == 1 && g_loss.size(0) == d.T, "row_weights must be (", d.T, ",); got ", g_loss.sizes());
  const Tensor g = g_loss.to(at::kFloat).contiguous();
  Tensor loss = at::empty({d.T}, g.options()), out = at::empty({d.T, d.V}, logits.options());
  check(bcjr_topk_distill_both(d.logits.data_ptr(), d.dtype, row_stride(d.logits), d.values.data_ptr<float>(),
                               d.indices.data_ptr<int32_t>(), lse_ptr(d), (float)temperature, d.T, d.V, d.K,
                               g.data_ptr<float>(), loss.data_ptr<float>(), out.data_ptr(), stream_of(logits)),
        "bcjr_topk_distill_both");
  return {loss, out};
}

std::tuple<Tensor, Tensor> topk_distill_both_meta(const Tensor& logits, const Tensor& values, const Tensor& indices,
                                                  const Tensor& g_loss, const OptTensor& lse, double temperature) {
  distill_args(logits, values, indices, lse);
  return {at::empty({logits.size(0)}, logits.options().dtype(at::kFloat)), at::empty(logits.sizes(), logits.options())};
}

std::tuple<Tensor, Tensor> call_distill(const Tensor& logits, const Tensor& values, const Tensor& indices,
                                        const OptTensor& lse, double temperature, bool keep) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("bcjr::topk_distill", "")
                       .typed<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const OptTensor&,
                                                         double, bool)>();
  at::AutoDispatchBelowADInplaceOrView guard;
  return op.call(logits, values, indices, lse, temperature, keep);
}

struct DistillFunction : torch::autograd::Function<DistillFunction> {
  static Variable forward(AutogradContext* ctx, const Tensor& logits, const Tensor& values, const Tensor& indices,
                          const OptTensor& lse, double temperature) {
    auto [loss, stats] = call_distill(logits, values, indices, lse, temperature, true);
    ctx->save_for_backward({logits, values, indices, stats});
    ctx->saved_data["temperature"] = temperature;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("bcjr::topk_distill_backward", "")
                         .typed<Tensor(const Tensor&, const Tensor&, const Tensor&, double, const Tensor&,
                                       const Tensor&)>();
    const auto s = ctx->get_saved_variables();
    Tensor d;
    if (g[0].defined()) d = op.call(s[0], s[1], s[2], ctx->saved_data["temperature"].toDouble(), s[3], g[0]);
    return {d, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor topk_distill_loss(const Tensor& logits, const Tensor& values, const Tensor& indices, const OptTensor& lse,
                         double temperature) {
  if (wants_grad(logits)) return DistillFunction::apply(logits, values, indices, lse, temperature);
  return std::get<0>(call_distill(logits, values, indices, lse, temperature, false));
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(bcjr, m) {
  m.def("moe_route(Tensor logits, Tensor? valid, int k, bool renormalize) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("moe_route_backward(Tensor logits, Tensor? valid, Tensor weights, Tensor experts, Tensor g_weights, "
        "bool renormalize) -> Tensor");
  m.def("grouped_product(Tensor x, Tensor w, Tensor offsets, Tensor? rows, bool w_is_nk, bool zero_padded=False) -> Tensor");
  m.def("grouped_wgrad(Tensor gy, Tensor x, Tensor offsets, Tensor? rows, bool zero_padded, bool out_f32) -> Tensor");
  m.def("pad_rows(Tensor x, Tensor like) -> Tensor");
  m.def("grouped_product_f32w(Tensor x, Tensor w, Tensor offsets, Tensor? rows, bool keep) -> (Tensor, Tensor)");
  m.def("combine(Tensor y, Tensor? weights, Tensor slots) -> Tensor");
  m.def("combine_backward(Tensor y, Tensor weights, Tensor rows, Tensor slots, Tensor g_out) -> (Tensor, Tensor)");
  m.def("topk_distill(Tensor logits, Tensor values, Tensor indices, Tensor? teacher_lse, float temperature, bool keep) "
        "-> (Tensor, Tensor)");
  m.def("topk_distill_backward(Tensor logits, Tensor values, Tensor indices, float temperature, Tensor stats, "
        "Tensor g_loss) -> Tensor");
  m.def("topk_distill_both(Tensor logits, Tensor values, Tensor indices, Tensor g_loss, Tensor? teacher_lse, "
        "float temperature) -> (Tensor, Tensor)");
  // differentiable forms, made of the operators above
  m.def("grouped_matmul(Tensor x, Tensor w, Tensor offsets, Tensor? rows, Tensor? slots) -> Tensor");
  m.def("moe_combine(Tensor y, Tensor weights, Tensor rows, Tensor slots) -> Tensor");
  m.def("topk_distill_loss(Tensor logits, Tensor values, Tensor indices, Tensor? teacher_lse, float temperature) -> Tensor");
}

TORCH_LIBRARY_IMPL(bcjr, CUDA, m) {
  m.impl("moe_route", &moe_route_hip);
  m.impl("moe_route_backward", &moe_route_backward_hip);
  m.impl("grouped_product", &grouped_matmul_hip);
  m.impl("grouped_wgrad", &grouped_wgrad_hip);
  m.impl("pad_rows", &pad_rows_hip);
  m.impl("grouped_product_f32w", &grouped_f32w_hip);
  m.impl("combine", &moe_combine_hip);
  m.impl("combine_backward", &moe_combine_backward_hip);
  m.impl("topk_distill", &topk_distill_hip);
  m.impl("topk_distill_backward", &topk_distill_backward_hip);
  m.impl("topk_distill_both", &topk_distill_both_hip);
}

TORCH_LIBRARY_IMPL(bcjr, Meta, m) {
  m.impl("moe_route", &moe_route_meta);
  m.impl("moe_route_backward", &moe_route_backward_meta);
  m.impl("grouped_product", &grouped_matmul_meta);
  m.impl("grouped_wgrad", &grouped_wgrad_meta);
  m.impl("pad_rows", &pad_rows_meta);
  m.impl("grouped_product_f32w", &grouped_f32w_meta);
  m.impl("combine", &moe_combine_meta);
  m.impl("combine_backward", &moe_combine_backward_meta);
  m.impl("topk_distill", &topk_distill_meta);
  m.impl("topk_distill_backward", &topk_distill_backward_meta);
  m.impl("topk_distill_both", &topk_distill_both_meta);
}

TORCH_LIBRARY_IMPL(bcjr, Autograd, m) { m.impl("moe_route", &moe_route_autograd); }

// Composite: their autograd formula is in them.
TORCH_LIBRARY_IMPL(bcjr, CompositeImplicitAutograd, m) {
  m.impl("grouped_matmul", &grouped_matmul);
  m.impl("moe_combine", &moe_combine);
  m.impl("topk_distill_loss", &topk_distill_loss);
}
