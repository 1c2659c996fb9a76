// Torch bindings of the feed-forward kernels: the linear and the gated layer
// with their gradients, and activations in 8 bits.  Every function checks
// device, type and shape, works on the device of its input and on that
// device's current stream, and takes its workspace from torch's allocator.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <optional>
#include <tuple>
#include <vector>

#include "linear.h"

namespace {

using MaybeTensor = std::optional<at::Tensor>;

hipStream_t stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index())
      .stream();
}

int type_of(const at::Tensor& t, const char* op) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf,
              op, ": bfloat16 or float16 on the GPU, got ", t.scalar_type());
  return t.scalar_type() == at::kBFloat16 ? 0 : 1;
}

void check_2d(const at::Tensor& t, const at::Tensor& like, const char* op,
              const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), op, ": ", name,
              " is on ", t.device(), ", not ", like.device());
  TORCH_CHECK(t.dim() == 2, op, ": ", name, " has ", t.dim(),
              " dimensions, not 2");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), op, ": ", name, " is ",
              t.scalar_type(), ", not ", like.scalar_type());
}

long up_to(long n, long to) { return (n + to - 1) / to * to; }

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

// An operand as the tiled product takes it: the tensor itself where its rows
// are whole 16 bytes, else a copy with zeros behind each row.
struct Rows {
  at::Tensor keep;
  const void* p;
  long ld;
  at::Tensor from;  // what `keep` is to be a copy of
};

// `n` of its columns: a copy that is one already has more.  What is to be
// copied goes to `todo`.
Rows whole_rows(const at::Tensor& t, long n, ff::Repack& todo,
                const char* op) {
  const long m = t.size(0);
  if (t.size(1) != n) return {t, t.data_ptr(), t.stride(0)};
  TORCH_CHECK(up_to(n, 8) < ff::kMaxPitch, op, ": a row of ", n,
              " is too long");
  at::Tensor u = n > 1 && t.stride(1) != 1 ? t.contiguous() : t;
  const long ld = m > 1 ? u.stride(0) : up_to(n, 8);
  // ld < n: rows that overlap, as an expanded tensor's
  if (aligned(u.data_ptr()) && n % 8 == 0 && ld % 8 == 0 && ld >= n &&
      ld < ff::kMaxPitch)
    return {u, u.data_ptr(), ld};
  const long ldo = up_to(n, 8);
  auto out = at::empty({m, ldo}, t.options());
  todo = {u.data_ptr(), m > 1 ? u.stride(0) : n, m, n, out.data_ptr(), ldo};
  return {out, out.data_ptr(), ldo, u};
}

// rows of any alignment, their values side by side
at::Tensor inner_contiguous(const at::Tensor& t) {
  return t.size(1) > 1 && t.stride(1) != 1 ? t.contiguous() : t;
}

// A launch that was refused (more blocks than a grid can have, say) has written
// nothing.
void check_launch(const char* op) {
  const hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, op, ": ", hipGetErrorString(e));
}

// t has `n` columns, or is whole_rows' copy of such
bool fits(const at::Tensor& t, long m, long n) {
  return t.size(0) == m &&
         (t.size(1) == n || (t.size(1) == up_to(n, 8) && t.is_contiguous()));
}

}  // namespace

// keep: 0 nothing, 1 the pre-activations in their type (the gated layer's in
// 24 bits: a byte tensor of both planes), 2 in 8 bits.  Returns y, pre or
// codes, scales.  x_used and w_used, if given: what the products took, for the
// backward pass.
static std::tuple<at::Tensor, MaybeTensor, MaybeTensor> linear_forward(
    at::Tensor x, at::Tensor w, MaybeTensor bias, MaybeTensor res, long act,
    bool gated, long keep, at::Tensor* x_used, at::Tensor* w_used) {
  const char* op = gated ? "gated_linear" : "linear_act";
  TORCH_CHECK(x.is_cuda(), op, ": x must be on the GPU");
  ff::Forward f{};
  f.type = type_of(x, op);
  check_2d(x, x, op, "x");
  check_2d(w, x, op, "weight");
  TORCH_CHECK(act >= 0 && act <= 3 && keep >= 0 && keep <= 2, op,
              ": unknown activation or checkpoint");
  TORCH_CHECK(!gated || act != 0, op, ": a gate needs an activation");
  const long m = x.size(0), k = x.size(1);
  const long n = gated ? w.size(0) / 2 : w.size(0);
  TORCH_CHECK(w.size(1) == k, op, ": x has ", k, " features, weight ",
              w.size(1));
  TORCH_CHECK(n > 0 && k > 0 && (!gated || w.size(0) % 2 == 0), op,
              ": weight of ", w.size(0), " x ", w.size(1));
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
  auto st = stream_of(x);
  auto y = at::empty({m, n}, x.options());
  f.act = (int)act;
  f.gated = gated;
  f.m = m, f.n = n, f.k = k;
  f.y = y.data_ptr();
  at::Tensor b, r;
  if (bias.has_value()) {
    TORCH_CHECK(bias->device() == x.device() &&
                    bias->scalar_type() == x.scalar_type() &&
                    bias->dim() == 1 && bias->size(0) == w.size(0),
                op, ": bias must be (", w.size(0), ",) of ", x.scalar_type(),
                " on ", x.device());
    b = bias->contiguous();
    f.bias = b.data_ptr();
  }
  if (res.has_value()) {
    TORCH_CHECK(!gated, op, ": no residual");
    check_2d(*res, x, op, "residual");
    TORCH_CHECK(res->size(0) == m && res->size(1) == n, op, ": residual of ",
                res->size(0), " x ", res->size(1), ", not ", m, " x ", n);
    r = inner_contiguous(*res);
    f.res = r.data_ptr();
    f.ldr = m > 1 ? r.stride(0) : n;
  }
  MaybeTensor pre, scales;
  if (keep != 0 && act != 0) {
    f.ldp = up_to(n, keep == 1 ? 8 : 32) * (gated ? 2 : 1);
    if (keep == 1 && gated) {
      pre = at::empty({m, 3 * f.ldp}, x.options().dtype(at::kByte));
      f.pre = pre->data_ptr();
      f.low = pre->data_ptr<unsigned char>() + 2 * m * f.ldp;
    } else if (keep == 1) {
      pre = at::empty({m, f.ldp}, x.options());
      f.pre = pre->data_ptr();
    } else {
      pre = at::empty({m, f.ldp}, x.options().dtype(at::kByte));
      scales = at::empty({m, f.ldp / 32}, x.options().dtype(at::kByte));
      f.codes = pre->data_ptr<unsigned char>();
      f.scales = scales->data_ptr<unsigned char>();
    }
  }
  if (m == 0) return {y, pre, scales};
  TORCH_CHECK(m < (1L << 30), op, ": ", m, " rows are too many");
  TORCH_CHECK(keep == 0 || up_to(w.size(0), 8) < ff::kMaxPitch, op, ": ",
              w.size(0), " features are too many for a backward pass");
  ff::Repack copies[2] = {};
  const Rows xr = whole_rows(x, k, copies[0], op);
  const Rows wr = whole_rows(w, k, copies[1], op);
  ff::launch_repack(copies[0], copies[1], st);
  if (x_used != nullptr) *x_used = xr.keep;
  if (w_used != nullptr) *w_used = wr.keep;
  f.x = xr.p, f.ldx = xr.ld;
  f.w = wr.p, f.ldw = wr.ld;
  at::Tensor part;
  ff::choose_forward(f);
  if (!f.by_rows && f.choice.splits > 1) {
    part = at::empty({f.choice.splits, m, w.size(0)},
                     x.options().dtype(at::kFloat));
    f.part = part.data_ptr<float>();
  }
  ff::launch_linear_forward(f, st);
  check_launch(op);
  return {y, pre, scales};
}

// The gradients of x, weight and bias, each where asked for.  x: its values,
// or with `x_scales` their codes; pre: as linear_forward kept them.
static std::tuple<MaybeTensor, MaybeTensor, MaybeTensor> linear_backward(
    at::Tensor dy, MaybeTensor x, MaybeTensor x_scales, MaybeTensor w,
    MaybeTensor pre, MaybeTensor scales, long act, bool gated, long k,
    bool need_x, bool need_w, bool need_b) {
  const char* op = gated ? "gated_linear" : "linear_act";
  TORCH_CHECK(dy.is_cuda(), op, ": the gradient must be on the GPU");
  check_2d(dy, dy, op, "the gradient");
  const int type = type_of(dy, op);
  const long m = dy.size(0), n = dy.size(1);
  const long outs = gated ? 2 * n : n;
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(dy.device());
  auto st = stream_of(dy);
  auto opt = dy.options();
  auto f32 = opt.dtype(at::kFloat);
  MaybeTensor dx, dw, db;
  if (need_x) dx = at::empty({m, k}, opt);
  if (m == 0) {
    if (need_w) dw = at::zeros({outs, k}, opt);
    if (need_b) db = at::zeros({outs}, opt);
    return {dx, dw, db};
  }

  // ---- the pre-activations' gradient, and its column sums
  at::Tensor d = inner_contiguous(dy);
  const bool products = need_x || need_w;
  ff::Slope s{};
  s.type = type, s.act = (int)act, s.gated = gated;
  s.m = m, s.n = n;
  s.dy = d.data_ptr();
  s.ldy = m > 1 ? d.stride(0) : up_to(n, 8);
  s.vec_dy = n % 8 == 0 && aligned(s.dy) && s.ldy % 8 == 0;
  at::Tensor g, sums;
  const void* gp = s.dy;
  long ldg = s.ldy;
  if (act != 0 || !s.vec_dy || ldg < n || ldg >= ff::kMaxPitch) {
    ldg = up_to(outs, 8);
    TORCH_CHECK(ldg < ff::kMaxPitch, op, ": ", outs, " features are too many");
    if (products) {
      g = at::empty({m, ldg}, opt);
      gp = s.out = g.data_ptr();
      s.ldo = ldg;
    }
  }
  if (act != 0) {
    const bool eight = scales.has_value();
    s.ldp = up_to(n, eight ? 32 : 8) * (gated ? 2 : 1);
    TORCH_CHECK(pre.has_value() && pre->is_contiguous() &&
                    pre->device() == dy.device() && pre->size(0) == m &&
                    pre->size(1) == s.ldp * (gated && !eight ? 3 : 1),
                op, ": no pre-activations of this gradient's shape");
    if (eight) {
      s.codes = pre->data_ptr<unsigned char>();
      s.scales = scales->data_ptr<unsigned char>();
    } else if (gated) {
      s.pre = pre->data_ptr<unsigned char>();
      s.low = pre->data_ptr<unsigned char>() + 2 * m * s.ldp;
    } else {
      TORCH_CHECK(pre->scalar_type() == dy.scalar_type(), op, ": gradient of ",
                  dy.scalar_type(), " for values of ", pre->scalar_type());
      s.pre = pre->data_ptr();
    }
  }
  s.chunks = ff::slope_chunks(m, n);
  if (need_b) {
    db = at::empty({outs}, opt);
    sums = at::empty({s.chunks, outs}, f32);
    s.sums = sums.data_ptr<float>();
  }
  Rows wr, xr;
  ff::Repack copies[2] = {};
  if (need_w) {
    TORCH_CHECK(x.has_value(), op, ": no input");
    if (x_scales.has_value()) {
      const long ldx = up_to(k, 8), ldc = up_to(k, 32);
      TORCH_CHECK(x->is_contiguous() && x->size(0) == m && x->size(1) == ldc &&
                      x->device() == dy.device(),
                  op, ": no input of this gradient's shape");
      xr.keep = at::empty({m, ldx}, opt);
      ff::Pack& p = s.input;
      p.type = type, p.vec = true;
      p.m = m, p.n = k;
      p.x = xr.keep.data_ptr(), p.ldx = ldx;
      p.codes = x->data_ptr<unsigned char>();
      p.scales = x_scales->data_ptr<unsigned char>();
      p.ldc = ldc;
      xr.p = p.x, xr.ld = ldx;
    } else {
      check_2d(*x, dy, op, "x");
      TORCH_CHECK(fits(*x, m, k), op, ": no input of this gradient's shape");
      xr = whole_rows(*x, k, copies[0], op);
    }
  }
  if (need_x) {
    TORCH_CHECK(w.has_value(), op, ": no weight");
    check_2d(*w, dy, op, "weight");
    TORCH_CHECK(fits(*w, outs, k), op,
                ": no weight of this gradient's shape");
    wr = whole_rows(*w, k, copies[1], op);
  }
  ff::launch_repack(copies[0], copies[1], st);
  ff::launch_slope(s, st);

  // ---- the products, and the bias gradient's last sums
  ff::Backward q{};
  q.type = type;
  if (need_b) {
    q.sums = s.sums;
    q.chunks = s.chunks;
    q.width = outs;
    q.dbias = db->data_ptr();
  }
  if (need_x) {
    q.dx.m = m, q.dx.n = k, q.dx.k = outs;
    q.dx.a = gp, q.dx.lda = ldg;
    q.dx.b = wr.p, q.dx.ldb = wr.ld;
    q.dx.out = dx->data_ptr();
  }
  if (need_w) {
    dw = at::empty({outs, k}, opt);
    q.dw.m = outs, q.dw.n = k, q.dw.k = m;
    q.dw.a = gp, q.dw.lda = ldg;
    q.dw.b = xr.p, q.dw.ldb = xr.ld;
    q.dw.out = dw->data_ptr();
  }
  const long ms[2] = {q.dx.m, q.dw.m}, ns[2] = {q.dx.n, q.dw.n},
             ks[2] = {q.dx.k, q.dw.k};
  q.choice = ff::choose_pair(ms, ns, ks);
  at::Tensor parts[2];
  for (int i = 0; i < 2; i++) {
    ff::Matmul& p = i == 0 ? q.dx : q.dw;
    p.splits = q.choice.splits[i];
    if (p.splits > 1) {
      parts[i] = at::empty({p.splits, p.m, p.n}, f32);
      p.part = parts[i].data_ptr<float>();
    }
  }
  ff::launch_backward(q, st);
  check_launch(op);
  return {dx, dw, db};
}

static int pack_type(const at::Tensor& t, const char* op) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat ||
                       t.scalar_type() == at::kBFloat16 ||
                       t.scalar_type() == at::kHalf,
                   op, ": ", t.scalar_type(),
                   " is not bfloat16, float16 or float32");
  return t.scalar_type() == at::kFloat ? 2 : type_of(t, op);
}

// x (..., n) -> codes (rows, n to a multiple of 32), scales (rows, that / 32)
std::tuple<at::Tensor, at::Tensor> act8_pack(at::Tensor x) {
  const char* op = "pack_activation";
  TORCH_CHECK(x.is_cuda(), op, ": x must be on the GPU");
  TORCH_CHECK_VALUE(x.dim() > 0, op, ": a scalar has no last axis");
  ff::Pack p{};
  p.type = pack_type(x, op);
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
  p.m = 1, p.n = x.size(-1);
  for (int i = 0; i + 1 < x.dim(); i++) p.m *= x.size(i);
  auto v = inner_contiguous(x.dim() == 2 ? x : x.reshape({p.m, p.n}));
  p.ldc = up_to(p.n, 32);
  auto bytes = x.options().dtype(at::kByte).requires_grad(false);
  auto codes = at::empty({p.m, p.ldc}, bytes);
  auto scales = at::empty({p.m, p.ldc / 32}, bytes);
  if (codes.numel() == 0) return {codes, scales};
  p.x = v.data_ptr();
  p.ldx = p.m > 1 ? v.stride(0) : p.n;
  p.vec = aligned(p.x) && p.n % 8 == 0 && p.ldx % 8 == 0;
  p.codes = codes.data_ptr<unsigned char>();
  p.scales = scales.data_ptr<unsigned char>();
  ff::launch_pack(p, stream_of(x));
  check_launch(op);
  return {codes, scales};
}

at::Tensor act8_unpack(at::Tensor codes, at::Tensor scales,
                       std::vector<int64_t> shape, at::ScalarType dtype) {
  const char* op = "unpack_activation";
  TORCH_CHECK_VALUE(codes.is_cuda() && codes.device() == scales.device() &&
                        codes.scalar_type() == at::kByte &&
                        scales.scalar_type() == at::kByte &&
                        codes.dim() == 2 && scales.dim() == 2 &&
                        codes.is_contiguous() && scales.is_contiguous() &&
                        !shape.empty(),
                    op, ": codes and scales as pack_activation gives them");
  ff::Pack p{};
  p.m = 1, p.n = shape.back(), p.ldc = up_to(p.n, 32);
  for (size_t i = 0; i + 1 < shape.size(); i++) p.m *= shape[i];
  TORCH_CHECK_VALUE(codes.size(0) == p.m && codes.size(1) == p.ldc &&
                        scales.size(0) == p.m && scales.size(1) == p.ldc / 32,
                    op, ": codes and scales as pack_activation gives them");
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(codes.device());
  auto x = at::empty(shape, codes.options().dtype(dtype));
  p.type = pack_type(x, op);
  if (x.numel() == 0) return x;
  p.x = x.data_ptr();
  p.ldx = p.n;
  p.vec = p.n % 8 == 0;
  p.codes = codes.data_ptr<unsigned char>();
  p.scales = scales.data_ptr<unsigned char>();
  ff::launch_unpack(p, stream_of(codes));
  check_launch(op);
  return x;
}

// ---- the layers, with autograd ----------------------------------------------

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

MaybeTensor maybe(const at::Tensor& t) {
  return t.defined() ? MaybeTensor(t) : std::nullopt;
}

// In C++, so that a step of a small layer is not one of Python's.
struct LayerFunction : torch::autograd::Function<LayerFunction> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor x, at::Tensor w,
                            MaybeTensor b, MaybeTensor r, int64_t act,
                            bool gated, bool eight) {
    const bool need_x = x.requires_grad(), need_w = w.requires_grad();
    const bool need = need_x || need_w || (b && b->requires_grad());
    // where rows had to be copied, the copies serve the backward pass too
    at::Tensor kept = x, kept_scales, kept_w = w;
    auto [y, pre, scales] =
        linear_forward(x, w, b, r, act, gated, need ? (eight ? 2 : 1) : 0,
                       eight ? nullptr : &kept, &kept_w);
    if (!need_w)
      kept = at::Tensor();
    else if (eight)
      std::tie(kept, kept_scales) = act8_pack(x);
    else if (kept.size(1) == x.size(1))
      kept = x;
    if (!need_x)
      kept_w = at::Tensor();
    else if (kept_w.size(1) == w.size(1))
      kept_w = w;
    ctx->save_for_backward({kept, kept_scales, kept_w,
                            pre.value_or(at::Tensor()),
                            scales.value_or(at::Tensor())});
    ctx->saved_data["act"] = act;
    ctx->saved_data["gated"] = gated;
    ctx->saved_data["k"] = x.size(1);
    ctx->saved_data["bias"] = b.has_value();
    ctx->saved_data["residual"] = r.has_value();
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto& dy = grads[0];
    const bool need_x = ctx->needs_input_grad(0);
    const bool need_w = ctx->needs_input_grad(1);
    // counted among the tensors that there are
    const bool b = ctx->saved_data["bias"].toBool();
    const bool r = ctx->saved_data["residual"].toBool();
    const bool need_b = b && ctx->needs_input_grad(2);
    const bool need_r = r && ctx->needs_input_grad(b ? 3 : 2);
    variable_list out(7);
    if (!dy.defined()) return out;
    if (need_x || need_w || need_b) {
      at::NoGradGuard no_grad;
      auto [dx, dw, db] = linear_backward(
          dy, maybe(saved[0]), maybe(saved[1]), maybe(saved[2]),
          maybe(saved[3]), maybe(saved[4]), ctx->saved_data["act"].toInt(),
          ctx->saved_data["gated"].toBool(), ctx->saved_data["k"].toInt(),
          need_x, need_w, need_b);
      out[0] = dx.value_or(at::Tensor());
      out[1] = dw.value_or(at::Tensor());
      out[2] = db.value_or(at::Tensor());
    }
    if (need_r) out[3] = dy;
    if (at::GradMode::is_enabled()) {
      // these gradients are constants to autograd; a second derivative
      // through them would be wrong, so it raises
      for (int i = 0; i < 3; i++)
        if (out[i].defined()) {
          auto fail = std::make_shared<torch::autograd::DelayedError>(
              "linear_act and gated_linear are differentiable once", 1);
          auto v = out[i].detach();
          v.set_requires_grad(true);
          out[i] = (*fail)({v})[0];
        }
    }
    return out;
  }
};

}  // namespace

// The layer of rocps/ops/linear.py (or gated.py) for x of any leading axes.
at::Tensor linear_layer(at::Tensor x, at::Tensor w, MaybeTensor bias,
                        MaybeTensor res, long act, bool gated, bool eight) {
  const char* op = gated ? "gated_linear" : "linear_act";
  TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1),
                    op, ": x ", x.sizes(), " and weight ", w.sizes(),
                    " do not fit");
  TORCH_CHECK_VALUE(w.numel() > 0, op, ": weight ", w.sizes(), " is empty");
  TORCH_CHECK_VALUE(!gated || w.size(0) % 2 == 0, op, ": weight ", w.sizes(),
                    " has no two halves");
  TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16 ||
                       x.scalar_type() == at::kHalf,
                   op, ": ", x.scalar_type(),
                   " on the GPU; bfloat16 or float16 there");
  auto same = [&](const at::Tensor& t, const char* name) {
    TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type() &&
                         t.device() == x.device(),
                     op, ": ", name, " is ", t.scalar_type(), " on ",
                     t.device(), ", x is ", x.scalar_type(), " on ",
                     x.device());
  };
  same(w, "weight");
  if (bias.has_value()) {
    same(*bias, "bias");
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == w.size(0), op,
                      ": bias ", bias->sizes(), ", not (", w.size(0), ",)");
  }
  const long n = gated ? w.size(0) / 2 : w.size(0);
  auto shape = x.sizes().vec();
  shape.back() = n;
  if (res.has_value()) {
    same(*res, "residual");
    TORCH_CHECK_VALUE(res->sizes() == at::IntArrayRef(shape), op,
                      ": residual ", res->sizes(), ", not ",
                      at::IntArrayRef(shape));
  }
  // without this they would be lost where no input requires a gradient
  for (const at::Tensor* t : {&x, &w, bias ? &*bias : nullptr,
                              res ? &*res : nullptr})
    TORCH_CHECK_NOT_IMPLEMENTED(
        t == nullptr || !t->_fw_grad(0).defined(), op,
        ": no forward-mode derivatives");
  const bool flat = x.dim() == 2;
  long m = 1;
  for (int i = 0; i + 1 < x.dim(); i++) m *= x.size(i);
  if (!flat) {
    x = x.reshape({m, x.size(-1)});
    if (res.has_value()) res = res->reshape({m, n});
  }
  auto grad = [](const MaybeTensor& t) {
    return t.has_value() && t->requires_grad();
  };
  at::Tensor y;
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() ||
                                     grad(bias) || grad(res)))
    y = LayerFunction::apply(x, w, bias, res, (int64_t)act, gated, eight);
  else
    y = std::get<0>(
        linear_forward(x, w, bias, res, act, gated, 0, nullptr, nullptr));
  return flat ? y : y.view(shape);
}

void bind_linear(pybind11::module& m) {
  m.def("linear_layer", &linear_layer);
  m.def("act8_pack", &act8_pack);
  m.def("act8_unpack", &act8_unpack);
}
