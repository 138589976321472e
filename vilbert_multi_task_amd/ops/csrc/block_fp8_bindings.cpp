// Registration of the block-scaled 8-bit operators and of the root-mean-square
// norm under torch.ops.vilbert_amd (kernels: block_fp8.hip, block_fp8_gemm.hip).

#include <ATen/ATen.h>
#include <ATen/core/DimVector.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_bf16.h>
#include <hip/hip_runtime.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

using bf16 = __hip_bfloat16;

template <typename T>
void launch_block_norm(int form, const T*, const T*, const T*, const T*, T*, T*,
                       unsigned char*, void*, bool, float*, long, int, float,
                       hipStream_t);
int rms_bwd_parts(long rows, int dim);
template <typename T>
void launch_rms_bwd(const T*, const T*, const T*, const float*, const T*, T*,
                    T*, float*, long, int, hipStream_t);
template <typename T>
void launch_quantize_block(const T*, unsigned char*, void*, bool, long, int,
                           hipStream_t);
template <typename T>
void launch_quantize_block_weight(const T*, unsigned char*, void*, bool, int, int,
                                  hipStream_t);
void launch_block_gemm(const unsigned char*, const void*, const unsigned char*,
                       const void*, bool, const void*, bool, void*, bool, void*,
                       long, long, int, int, int, bool, hipStream_t);

namespace {

constexpr long kBlock = 128;
constexpr long kMaxPitch = 1l << 24;  // a tile's rows have 32-bit offsets
constexpr long kMaxNorm = 65536;  // a row's values stay in registers
constexpr long kMaxIndex = (1l << 31) - 1024;  // rounded up to a tile, still an int

using OptTensor = c10::optional<at::Tensor>;

hipStream_t cur_stream() { return c10::hip::getCurrentHIPStream().stream(); }
long ceil_to(long a, long b) { return (a + b - 1) / b; }

// a bf16/f32 tensor of at least one column; how many rows it has
long rows_of(const char* op, const at::Tensor& x) {
  TORCH_CHECK(x.is_cuda(), op, ": a GPU tensor is needed");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat,
              op, ": dtype must be bf16/f32, got ", x.scalar_type());
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, op, ": the last dimension is empty");
  TORCH_CHECK(x.size(-1) <= kMaxIndex, op, ": the last dimension is too long");
  return x.numel() / x.size(-1);
}
// a parameter of the last dimension, or a tensor like x
void check_like(const char* op, const char* name, const at::Tensor& x,
                const at::Tensor& t, bool whole) {
  TORCH_CHECK(t.device() == x.device(), op, ": ", name, " is on ", t.device(),
              ", x on ", x.device());
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), op, ": ", name, " is ",
              t.scalar_type(), ", x ", x.scalar_type());
  if (whole) {
    TORCH_CHECK(t.sizes() == x.sizes(), op, ": ", name, " has the sizes ",
                t.sizes(), ", x ", x.sizes());
  } else {
    TORCH_CHECK(t.dim() == 1 && t.size(0) == x.size(-1), op, ": ", name,
                " has the sizes ", t.sizes(), ", x's rows ", x.size(-1), " values");
  }
}

// at::empty on like's device, without the dispatcher's part of it
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt));
}
at::Tensor fresh_like(const at::Tensor& t) { return fresh(t.sizes(), t.scalar_type(), t); }

// 8-bit rows of `k` values that begin at multiples of 16 bytes
at::Tensor empty_rows8(at::IntArrayRef sizes, const at::Tensor& like) {
  at::DimVector s(sizes.begin(), sizes.end());
  const long k = s.back();
  s.back() = ceil_to(k, 16) * 16;
  auto y = fresh(s, at::kFloat8_e4m3fn, like);
  return s.back() == k ? y : y.narrow(-1, 0, k);
}
at::Tensor empty_scales(at::IntArrayRef sizes, const at::Tensor& like, bool f32) {
  at::DimVector s(sizes.begin(), sizes.end());
  s.back() = ceil_to(s.back(), kBlock);
  return fresh(s, f32 ? at::kFloat : at::kBFloat16, like);
}
unsigned char* bytes(const at::Tensor& t) { return (unsigned char*)t.data_ptr(); }

OptTensor dense(const OptTensor& t) {
  return t.has_value() ? OptTensor(t->contiguous()) : t;
}

template <typename T>
const T* ptr(const OptTensor& t) {
  return t.has_value() && t->defined() ? (const T*)t->data_ptr() : nullptr;
}

template <typename T>
void norm_as(int form, const at::Tensor& x, const OptTensor& res,
             const at::Tensor& w, const OptTensor& b, const OptTensor& y,
             const OptTensor& sum, const OptTensor& y8,
             const OptTensor& scales, const OptTensor& rstd, double eps) {
  const long rows = x.numel() / x.size(-1);
  if (rows == 0) return;
  launch_block_norm<T>(
      form, (const T*)x.data_ptr(), ptr<T>(res), (const T*)w.data_ptr(),
      ptr<T>(b), (T*)ptr<T>(y), (T*)ptr<T>(sum),
      (unsigned char*)ptr<unsigned char>(y8), (void*)ptr<void>(scales),
      scales.has_value() && scales->scalar_type() == at::kFloat,
      (float*)ptr<float>(rstd), rows, (int)x.size(-1), (float)eps, cur_stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

void norm(int form, const at::Tensor& x, const OptTensor& res,
          const at::Tensor& w, const OptTensor& b, const OptTensor& y,
          const OptTensor& sum, const OptTensor& y8, const OptTensor& scales,
          const OptTensor& rstd, double eps) {
  if (x.scalar_type() == at::kFloat)
    norm_as<float>(form, x, res, w, b, y, sum, y8, scales, rstd, eps);
  else
    norm_as<bf16>(form, x, res, w, b, y, sum, y8, scales, rstd, eps);
}

void check_norm(const char* op, const at::Tensor& x, const OptTensor& res,
                const at::Tensor& w) {
  rows_of(op, x);
  TORCH_CHECK(x.size(-1) <= kMaxNorm, op, ": rows of at most ", kMaxNorm,
              " values, got ", x.size(-1));
  check_like(op, "weight", x, w, false);
  if (res.has_value()) check_like(op, "residual", x, *res, true);
}

// Operators by their names: autograd's part of one hands on through the dispatcher, so
// that what is between it and the kernels (fake tensors, modes, transforms) sees the
// call. Found once, typed, without boxing.
#define OPERATOR(name)                                                             \
  []() -> const auto& {                                                            \
    static const auto op = c10::Dispatcher::singleton()                            \
                               .findSchemaOrThrow("vilbert_amd::" #name, "")       \
                               .typed<decltype(name)>();                           \
    return op;                                                                     \
  }()

struct RmsForward {
  at::Tensor y, sum, rstd;  // sum with a residual alone, rstd where asked for
};
RmsForward rms_forward(const at::Tensor& x_in, const OptTensor& res,
                       const at::Tensor& w, double eps, bool stats) {
  check_norm("rms_norm", x_in, res, w);
  c10::DeviceGuard guard(x_in.device());
  const auto x = x_in.contiguous();
  RmsForward f;
  f.y = fresh_like(x);
  if (res.has_value()) f.sum = fresh_like(x);
  if (stats)
    f.rstd = fresh({x.numel() / x.size(-1)}, at::kFloat, x);
  norm(0, x, dense(res), w.contiguous(), {}, f.y, f.sum, {}, {}, f.rstd, eps);
  return f;
}

template <typename T>
void rms_bwd_as(const at::Tensor& gy, const OptTensor& gsum,
                const at::Tensor& t, const at::Tensor& rstd,
                const at::Tensor& w, at::Tensor& gx, at::Tensor& gw) {
  const int dim = (int)t.size(-1);
  const long rows = t.numel() / dim;
  auto part = fresh({rms_bwd_parts(rows, dim), (long)dim}, at::kFloat, t);
  launch_rms_bwd<T>((const T*)gy.data_ptr(), ptr<T>(gsum),
                    (const T*)t.data_ptr(), rstd.data_ptr<float>(),
                    (const T*)w.data_ptr(), (T*)gx.data_ptr(),
                    (T*)gw.data_ptr(), part.data_ptr<float>(), rows, dim,
                    cur_stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

// What training takes of the forward: y, the stream (empty without a residual, where
// it is x) and each row's 1/rms.
std::tuple<at::Tensor, at::Tensor, at::Tensor> rms_fwd_train(const at::Tensor& x,
                                                             const OptTensor& res,
                                                             const at::Tensor& w,
                                                             double eps) {
  auto f = rms_forward(x, res, w, eps, true);
  if (!f.sum.defined()) f.sum = fresh({0}, x.scalar_type(), x);
  return {f.y, f.sum, f.rstd};
}

std::tuple<at::Tensor, at::Tensor> rms_bwd(const at::Tensor& gy, const OptTensor& gsum,
                                           const at::Tensor& t, const at::Tensor& rstd,
                                           const at::Tensor& w) {
  const char* op = "rms_bwd";
  check_norm(op, t, gsum, w);
  check_like(op, "gy", t, gy, true);
  const long rows = t.numel() / t.size(-1);
  TORCH_CHECK(rstd.device() == t.device() && rstd.scalar_type() == at::kFloat &&
                  rstd.dim() == 1 && rstd.size(0) == rows && rstd.is_contiguous(),
              op, ": rstd must be ", rows, " values in f32 on ", t.device());
  c10::DeviceGuard guard(t.device());
  const auto tc = t.contiguous(), wc = w.contiguous(), gc = gy.contiguous();
  auto gx = fresh_like(tc);
  auto gw = rows ? fresh_like(wc) : at::zeros_like(wc);
  if (rows) {
    if (t.scalar_type() == at::kFloat)
      rms_bwd_as<float>(gc, dense(gsum), tc, rstd, wc, gx, gw);
    else
      rms_bwd_as<bf16>(gc, dense(gsum), tc, rstd, wc, gx, gw);
  }
  return {gx, gw};
}

// The stream t that the forward leaves (x itself without a residual) and a row's
// 1/rms are all that the backward needs besides the weight.
struct RmsNorm : torch::autograd::Function<RmsNorm> {
  using List = torch::autograd::variable_list;

  static List forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                      const at::Tensor& w, const OptTensor& res, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    const auto [y, sum, rstd] = OPERATOR(rms_fwd_train).call(x, res, w, eps);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({res.has_value() ? sum : x, rstd, w});
    ctx->saved_data["res"] = res.has_value();
    return res.has_value() ? List{y, sum} : List{y};
  }

  static List backward(torch::autograd::AutogradContext* ctx, List g) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "rms_norm: its gradient has no gradient (create_graph)");
    const auto saved = ctx->get_saved_variables();
    const bool res = ctx->saved_data["res"].toBool();
    const at::Tensor gsum = res ? g[1] : at::Tensor();
    at::Tensor gx, gw;
    if (g[0].defined()) {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(gx, gw) = OPERATOR(rms_bwd).call(
          g[0], gsum.defined() ? OptTensor(gsum) : OptTensor(), saved[0], saved[1],
          saved[2]);
    } else {  // the stream alone was used
      gx = gsum;
    }
    return {gx, gw, res ? gx : at::Tensor(), at::Tensor()};
  }
};

// No operator here has a forward-mode derivative: left unseen, a tangent would be
// dropped, and the derivative read as zero.
bool has_tangent(const at::Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }
template <typename T>
bool has_tangent(const T&) { return false; }
template <typename... A>
void refuse_tangents(const char* op, const A&... args) {
  TORCH_CHECK(!c10::AutogradState::get_tls_state().get_fw_grad_mode() ||
                  !(has_tangent(args) || ...),
              op, " has no forward-mode derivative");
}

bool wants_grad(const at::Tensor& x, const OptTensor& res, const at::Tensor& w) {
  refuse_tangents("rms_norm", x, res, w);
  return at::GradMode::is_enabled() &&
         (x.requires_grad() || w.requires_grad() ||
          (res.has_value() && res->requires_grad()));
}

at::Tensor rms_norm(const at::Tensor& x, const at::Tensor& w, double eps) {
  return rms_forward(x, {}, w, eps, false).y;
}
at::Tensor rms_norm_autograd(const at::Tensor& x, const at::Tensor& w, double eps) {
  if (wants_grad(x, {}, w)) return RmsNorm::apply(x, w, OptTensor(), eps)[0];
  at::AutoDispatchBelowADInplaceOrView below;
  return OPERATOR(rms_norm).call(x, w, eps);
}

std::tuple<at::Tensor, at::Tensor> rms_norm_residual(const at::Tensor& x,
                                                     const at::Tensor& res,
                                                     const at::Tensor& w,
                                                     double eps) {
  const auto f = rms_forward(x, res, w, eps, false);
  return {f.y, f.sum};
}
std::tuple<at::Tensor, at::Tensor> rms_norm_residual_autograd(
    const at::Tensor& x, const at::Tensor& res, const at::Tensor& w, double eps) {
  if (wants_grad(x, res, w)) {
    const auto y = RmsNorm::apply(x, w, OptTensor(res), eps);
    return {y[0], y[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return OPERATOR(rms_norm_residual).call(x, res, w, eps);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> rms_norm_fp8_block(
    const at::Tensor& x_in, const OptTensor& res, const at::Tensor& w,
    double eps, bool f32_scales) {
  check_norm("rms_norm_fp8_block", x_in, res, w);
  c10::DeviceGuard guard(x_in.device());
  const auto x = x_in.contiguous();
  auto y8 = empty_rows8(x.sizes(), x);
  auto scales = empty_scales(x.sizes(), x, f32_scales);
  auto sum = res.has_value() ? fresh_like(x) : fresh({0}, x.scalar_type(), x);
  norm(1, x, dense(res), w.contiguous(), {}, {}, res.has_value() ? OptTensor(sum) : OptTensor(),
       y8, scales, {}, eps);
  return {y8, scales, sum};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_fp8_block(
    const at::Tensor& x_in, const OptTensor& res, const at::Tensor& w,
    const at::Tensor& b, double eps, bool f32_scales) {
  const char* op = "layer_norm_fp8_block";
  check_norm(op, x_in, res, w);
  check_like(op, "bias", x_in, b, false);
  c10::DeviceGuard guard(x_in.device());
  const auto x = x_in.contiguous();
  auto y = fresh_like(x);
  auto y8 = empty_rows8(x.sizes(), x);
  auto scales = empty_scales(x.sizes(), x, f32_scales);
  norm(2, x, dense(res), w.contiguous(), b.contiguous(), y, {}, y8, scales, {},
       eps);
  return {y, y8, scales};
}

std::tuple<at::Tensor, at::Tensor> quantize_fp8_block(const at::Tensor& x_in,
                                                      bool f32_scales) {
  const long rows = rows_of("quantize_fp8_block", x_in);
  c10::DeviceGuard guard(x_in.device());
  const auto x = x_in.contiguous();
  auto y8 = empty_rows8(x.sizes(), x);
  auto scales = empty_scales(x.sizes(), x, f32_scales);
  if (rows) {
    if (x.scalar_type() == at::kFloat)
      launch_quantize_block<float>(x.data_ptr<float>(), bytes(y8), scales.data_ptr(),
                                   f32_scales, rows, (int)x.size(-1), cur_stream());
    else
      launch_quantize_block<bf16>((const bf16*)x.data_ptr(), bytes(y8),
                                  scales.data_ptr(), f32_scales, rows,
                                  (int)x.size(-1), cur_stream());
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return {y8, scales};
}

std::tuple<at::Tensor, at::Tensor> quantize_fp8_block_weight(
    const at::Tensor& w_in, bool f32_scales) {
  const char* op = "quantize_fp8_block_weight";
  const long rows = rows_of(op, w_in);
  TORCH_CHECK(w_in.dim() == 2, op, ": a weight has two dimensions, got ",
              w_in.dim());
  TORCH_CHECK(ceil_to(rows, kBlock) <= 65535, op, ": too many rows");
  c10::DeviceGuard guard(w_in.device());
  const auto w = w_in.contiguous();
  auto w8 = empty_rows8(w.sizes(), w);
  auto scales = fresh({ceil_to(rows, kBlock), ceil_to(w.size(1), kBlock)},
                      f32_scales ? at::kFloat : at::kBFloat16, w);
  if (rows) {
    if (w.scalar_type() == at::kFloat)
      launch_quantize_block_weight<float>(w.data_ptr<float>(), bytes(w8),
                                          scales.data_ptr(), f32_scales, (int)rows,
                                          (int)w.size(1), cur_stream());
    else
      launch_quantize_block_weight<bf16>((const bf16*)w.data_ptr(), bytes(w8),
                                         scales.data_ptr(), f32_scales, (int)rows,
                                         (int)w.size(1), cur_stream());
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return {w8, scales};
}

// The rows of an 8-bit tensor at one distance, a multiple of 16 bytes: as they
// are where they lie so (what the producers here return does), else copied.
struct Rows8 {
  at::Tensor t;
  long rows, pitch;
};
Rows8 rows8(const at::Tensor& t) {
  const long k = t.size(-1);
  const long rows = t.numel() / k;
  long pitch = -1;
  bool even = t.stride(-1) == 1 || k == 1;
  for (long i = t.dim() - 2, inner = 1; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (pitch < 0) pitch = t.stride(i);
    even = even && t.stride(i) == pitch * inner;
    inner *= t.size(i);
  }
  if (pitch < 0) pitch = ceil_to(k, 16) * 16;  // one row
  if (even && pitch % 16 == 0 && pitch < kMaxPitch && (size_t)t.data_ptr() % 16 == 0)
    return {t, rows, pitch};
  auto to = empty_rows8({rows, k}, t);
  to.view(at::kByte).copy_(t.view(at::kByte).reshape({rows, k}));
  return {to, rows, ceil_to(k, 16) * 16};
}

struct Product {
  Rows8 x, w;
  at::Tensor xs, ws, bias;
  at::DimVector sizes;
  long n, k;
};
Product product(const char* op, const at::Tensor& x8, const at::Tensor& xs,
                const at::Tensor& w8, const at::Tensor& ws,
                const OptTensor& bias) {
  TORCH_CHECK(x8.is_cuda(), op, ": a GPU tensor is needed");
  for (auto* t : {&xs, &w8, &ws})
    TORCH_CHECK(t->device() == x8.device(), op, ": arguments on ", t->device(),
                " and ", x8.device());
  TORCH_CHECK(x8.scalar_type() == at::kFloat8_e4m3fn &&
                  w8.scalar_type() == at::kFloat8_e4m3fn,
              op, ": x8 and w8 must be float8_e4m3fn, got ", x8.scalar_type(),
              " and ", w8.scalar_type());
  TORCH_CHECK(xs.scalar_type() == ws.scalar_type() &&
                  (xs.scalar_type() == at::kBFloat16 || xs.scalar_type() == at::kFloat),
              op, ": scales must be both bf16 or both f32, got ", xs.scalar_type(),
              " and ", ws.scalar_type());
  TORCH_CHECK(x8.dim() >= 1 && w8.dim() == 2 && x8.size(-1) == w8.size(1), op,
              ": x8 [..., K] and w8 [N, K] are needed, got ", x8.sizes(), " and ",
              w8.sizes());
  const long k = w8.size(1), n = w8.size(0), kb = ceil_to(k, kBlock);
  TORCH_CHECK(k >= 1 && n >= 1, op, ": w8 is empty");
  const long rows = x8.numel() / k;
  TORCH_CHECK(rows <= kMaxIndex && n <= kMaxIndex && k <= kMaxPitch - 16 &&
                  ceil_to(n, kBlock) * ceil_to(rows, 16) < (1l << 31),
              op, ": too large");
  at::DimVector want(x8.sizes().begin(), x8.sizes().end());
  want.back() = kb;
  TORCH_CHECK(xs.sizes() == at::IntArrayRef(want), op, ": x_scales has the sizes ",
              xs.sizes(), ", x8 ", x8.sizes(), " needs ", at::IntArrayRef(want));
  TORCH_CHECK(ws.dim() == 2 && ws.size(0) == ceil_to(n, kBlock) &&
                  ws.size(1) == kb,
              op, ": w_scales has the sizes ", ws.sizes(), ", w8 ", w8.sizes(),
              " needs ", ceil_to(n, kBlock), " x ", kb);
  at::Tensor b;
  if (bias.has_value() && bias->defined()) {
    TORCH_CHECK(bias->device() == x8.device() && bias->dim() == 1 &&
                    bias->size(0) == n &&
                    (bias->scalar_type() == at::kBFloat16 ||
                     bias->scalar_type() == at::kFloat),
                op, ": bias must be ", n, " values in bf16/f32 on ", x8.device());
    b = bias->contiguous();
  }
  at::DimVector sizes(x8.sizes().begin(), x8.sizes().end());
  sizes.back() = n;
  return {rows8(x8), rows8(w8), xs.contiguous(), ws.contiguous(), b, sizes, n, k};
}

bool f32_scales(const Product& p) { return p.xs.scalar_type() == at::kFloat; }
void launch(const Product& p, const at::Tensor& y, void* ys, bool gelu) {
  if (p.x.rows == 0) return;
  launch_block_gemm(
      bytes(p.x.t), p.xs.data_ptr(), bytes(p.w.t), p.ws.data_ptr(), f32_scales(p),
      p.bias.defined() ? p.bias.data_ptr() : nullptr,
      p.bias.defined() && p.bias.scalar_type() == at::kFloat, y.data_ptr(),
      y.scalar_type() == at::kFloat, ys, p.x.pitch, p.w.pitch, (int)p.x.rows,
      (int)p.n, (int)p.k, gelu, cur_stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

at::Tensor fp8_block_linear(const at::Tensor& x8, const at::Tensor& xs,
                            const at::Tensor& w8, const at::Tensor& ws,
                            const OptTensor& bias, bool gelu, bool f32_out) {
  const char* op = "fp8_block_linear";
  TORCH_CHECK(x8.is_cuda(), op, ": a GPU tensor is needed");
  c10::DeviceGuard guard(x8.device());
  const Product p = product(op, x8, xs, w8, ws, bias);
  auto y = fresh(p.sizes, f32_out ? at::kFloat : at::kBFloat16, x8);
  launch(p, y, nullptr, gelu);
  return y;
}

std::tuple<at::Tensor, at::Tensor> fp8_block_linear_fp8(
    const at::Tensor& x8, const at::Tensor& xs, const at::Tensor& w8,
    const at::Tensor& ws, const OptTensor& bias, bool gelu) {
  const char* op = "fp8_block_linear_fp8";
  TORCH_CHECK(x8.is_cuda(), op, ": a GPU tensor is needed");
  c10::DeviceGuard guard(x8.device());
  const Product p = product(op, x8, xs, w8, ws, bias);
  auto y8 = empty_rows8(p.sizes, x8);
  auto scales = empty_scales(p.sizes, x8, f32_scales(p));
  launch(p, y8, scales.data_ptr(), gelu);
  return {y8, scales};
}

// The operators without a gradient: what needs one is refused here, for all callers,
// and the rest is handed on. (The dispatcher's own fallback would box the arguments.)
bool needs_grad(const at::Tensor& t) { return t.requires_grad(); }
bool needs_grad(const OptTensor& t) { return t.has_value() && t->requires_grad(); }
template <typename T>
bool needs_grad(const T&) { return false; }

template <typename F, const char* const* name>
struct Serving;
template <typename R, typename... A, const char* const* name>
struct Serving<R(A...), name> {
  static R call(A... args) {
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow(*name, "")
                               .typed<R(A...)>();
    TORCH_CHECK(!at::GradMode::is_enabled() || !(needs_grad(args) || ...),
                *name + sizeof("vilbert_amd::") - 1,
                " has no gradient: call it under torch.no_grad()");
    refuse_tangents(*name + sizeof("vilbert_amd::") - 1, args...);
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(args...);
  }
};

}  // namespace

TORCH_LIBRARY_FRAGMENT(vilbert_amd, m) {
  m.def("rms_norm(Tensor x, Tensor w, float eps) -> Tensor");
  m.def("rms_norm_residual(Tensor x, Tensor res, Tensor w, float eps) -> (Tensor, Tensor)");
  m.def("rms_fwd_train(Tensor x, Tensor? res, Tensor w, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("rms_bwd(Tensor gy, Tensor? gsum, Tensor t, Tensor rstd, Tensor w) -> (Tensor, Tensor)");
  m.def("rms_norm_fp8_block(Tensor x, Tensor? res, Tensor w, float eps, bool f32_scales=False) -> (Tensor, Tensor, Tensor)");
  m.def("layer_norm_fp8_block(Tensor x, Tensor? res, Tensor w, Tensor b, float eps, bool f32_scales=False) -> (Tensor, Tensor, Tensor)");
  m.def("quantize_fp8_block(Tensor x, bool f32_scales=False) -> (Tensor, Tensor)");
  m.def("quantize_fp8_block_weight(Tensor w, bool f32_scales=False) -> (Tensor, Tensor)");
  m.def("fp8_block_linear(Tensor x8, Tensor x_scales, Tensor w8, Tensor w_scales, Tensor? bias, bool gelu, bool f32_out=False) -> Tensor");
  m.def("fp8_block_linear_fp8(Tensor x8, Tensor x_scales, Tensor w8, Tensor w_scales, Tensor? bias, bool gelu) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(vilbert_amd, CUDA, m) {
  m.impl("rms_norm", rms_norm);
  m.impl("rms_norm_residual", rms_norm_residual);
  m.impl("rms_fwd_train", rms_fwd_train);
  m.impl("rms_bwd", rms_bwd);
  m.impl("rms_norm_fp8_block", rms_norm_fp8_block);
  m.impl("layer_norm_fp8_block", layer_norm_fp8_block);
  m.impl("quantize_fp8_block", quantize_fp8_block);
  m.impl("quantize_fp8_block_weight", quantize_fp8_block_weight);
  m.impl("fp8_block_linear", fp8_block_linear);
  m.impl("fp8_block_linear_fp8", fp8_block_linear_fp8);
}

TORCH_LIBRARY_IMPL(vilbert_amd, AutogradCUDA, m) {
  m.impl("rms_norm", rms_norm_autograd);
  m.impl("rms_norm_residual", rms_norm_residual_autograd);
#define SERVING(op)                                             \
  static constexpr const char* op##_name = "vilbert_amd::" #op; \
  m.impl(#op, Serving<decltype(op), &op##_name>::call)
  SERVING(rms_fwd_train);
  SERVING(rms_bwd);
  SERVING(rms_norm_fp8_block);
  SERVING(layer_norm_fp8_block);
  SERVING(quantize_fp8_block);
  SERVING(quantize_fp8_block_weight);
  SERVING(fp8_block_linear);
  SERVING(fp8_block_linear_fp8);
#undef SERVING
}
