// torch_dense.cpp -- the dense operators of the C ABI (embedding, rms_norm, gated_ffn, fp8) in the torch.ops.dgsparse_spmm registry, with their
// autograd nodes.  Same division of labour as torch_binding.cpp: arguments are checked here, outputs and workspaces come from ATen on the
// current stream of the inputs' device, everything below is torch-free.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <climits>
#include <initializer_list>
#include <tuple>

#include "dgsparse_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using Guard = c10::hip::HIPGuardMasqueradingAsCUDA;

void check_rc(int rc, const char *what) { TORCH_CHECK(rc == 0, "dgsparse: ", what, " failed: ", dgs_strerror(rc), " (", rc, ")"); }
dgsStream_t cur_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }
Tensor workspace(size_t bytes, const Tensor &like) { return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)); }

int dtype_of(const Tensor &t, const char *name) {
  switch (t.scalar_type()) {
    case at::kFloat: return DGS_F32;
    case at::kHalf: return DGS_F16;
    case at::kBFloat16: return DGS_BF16;
    default: TORCH_CHECK(false, "dgsparse: ", name, " must be float32, float16 or bfloat16, not ", t.scalar_type());
  }
}
void on_gpu(const Tensor &t, const char *name) {
  TORCH_CHECK(t.is_cuda(), "dgsparse: ", name, " must live on a GPU (this build has only the HIP back end; no CPU fallback)");
}
void like(const Tensor &t, const Tensor &other, const char *name, const char *oname) {
  TORCH_CHECK(t.device() == other.device(), "dgsparse: ", name, " and ", oname, " live on different devices (", t.device(), " vs ", other.device(), ")");
  TORCH_CHECK(t.scalar_type() == other.scalar_type(), "dgsparse: ", name, " must have the type of ", oname, " (", other.scalar_type(), "), not ",
              t.scalar_type());
}
// t as rows of its last dimension with a distance between rows: a 2-D view with unit stride in a row as it is, anything else made contiguous
Tensor rows_of(const Tensor &t, int64_t &ld) {
  const int64_t D = t.size(-1);
  if (t.dim() == 2 && (t.stride(1) == 1 || D == 1) && t.stride(0) >= 0) {
    ld = t.stride(0);
    return t;
  }
  ld = D;
  return t.contiguous().view({t.numel() / D, D});
}
// These nodes are differentiable once: with create_graph the second gradient would silently miss their part.
void once(const char *what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "dgsparse: ", what, " is differentiable once (its backward pass has no gradient of its own: no create_graph)");
}
// Nor have they a forward-mode derivative: where no gradient is recorded, a tangent would be dropped without a word, which stands for 0.
void no_tangent(const char *what, std::initializer_list<const Tensor *> inputs) {
  for (const Tensor *t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), "dgsparse: ", what, " has no forward-mode derivative");
}

// ---- embedding -------------------------------------------------------------------------------------------------------------
Tensor ids_of(const Tensor &ids, const Tensor &table) {
  on_gpu(ids, "ids");
  on_gpu(table, "table");
  TORCH_CHECK(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong, "dgsparse: ids must be int32 or int64, not ", ids.scalar_type());
  TORCH_CHECK(ids.device() == table.device(), "dgsparse: ids and table live on different devices (", ids.device(), " vs ", table.device(), ")");
  return ids.contiguous();
}
Tensor embedding_fwd(const Tensor &ids_, const Tensor &table_, double scale) {
  const Tensor ids = ids_of(ids_, table_);
  TORCH_CHECK(table_.dim() == 2 && table_.size(1) > 0, "dgsparse: table must be [tokens, features] with at least one feature");
  const int dtype = dtype_of(table_, "table");
  const Guard guard(table_.device());
  int64_t ld = 0;
  const Tensor table = rows_of(table_, ld);
  const int64_t n = ids.numel(), V = table.size(0), D = table.size(1);
  auto shape = ids.sizes().vec();
  shape.push_back(D);
  Tensor out = at::empty(shape, table.options());
  check_rc(dgs_embedding(dtype, (int)ids.element_size(), n, V, D, n ? ids.data_ptr() : nullptr, V ? table.data_ptr() : nullptr, ld, (float)scale,
                         n ? out.data_ptr() : nullptr, cur_stream()),
           "embedding");
  return out;
}
struct Embedding : public torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext *ctx, Tensor table, Tensor ids, double scale, int64_t padding_idx) {
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["pad"] = padding_idx;
    ctx->saved_data["V"] = table.size(0);
    return embedding_fwd(ids, table, scale);
  }
  static tensor_list backward(AutogradContext *ctx, tensor_list grads) {
    once("embedding");
    const Tensor &dout_ = grads[0];
    const Tensor ids = ctx->get_saved_variables()[0].contiguous();
    const Guard guard(dout_.device());
    const int64_t V = ctx->saved_data["V"].toInt(), n = ids.numel(), D = dout_.size(-1);
    int64_t ld = D;
    const Tensor dout = n ? rows_of(dout_, ld) : dout_;
    Tensor dtable = at::empty({V, D}, dout.options());
    const size_t wsb = dgs_embedding_bwd_workspace_bytes(n, V, D);
    Tensor ws = workspace(wsb, dout);
    check_rc(dgs_embedding_bwd(dtype_of(dout, "the output's gradient"), (int)ids.element_size(), n, V, D, n ? ids.data_ptr() : nullptr,
                               ctx->saved_data["pad"].toInt(), n ? dout.data_ptr() : nullptr, ld, (float)ctx->saved_data["scale"].toDouble(),
                               V ? dtable.data_ptr() : nullptr, ws.data_ptr(), wsb, cur_stream()),
             "embedding backward");
    return {dtable, Tensor(), Tensor(), Tensor()};
  }
};
Tensor embedding_op(Tensor ids, Tensor table, double scale, int64_t padding_idx) {
  TORCH_CHECK(padding_idx < table.size(0), "dgsparse: padding_idx ", padding_idx, " is not a row of the table");
  no_tangent("embedding", {&table});
  if (!(at::GradMode::is_enabled() && table.requires_grad())) return embedding_fwd(ids, table, scale);
  return Embedding::apply(table, ids, scale, padding_idx);
}

// ---- RMS norm --------------------------------------------------------------------------------------------------------------
struct NormOut { Tensor y, s, scales; };
NormOut norm_fwd(const Tensor &x_, const Tensor &res_, const Tensor &w_, double eps, bool fp8) {
  on_gpu(x_, "x");
  on_gpu(w_, "weight");
  const int dtype = dtype_of(x_, "x");
  TORCH_CHECK(x_.dim() >= 1 && x_.size(-1) > 0, "dgsparse: x must have at least one feature");
  TORCH_CHECK(w_.dim() == 1 && w_.size(0) == x_.size(-1), "dgsparse: weight must be [", x_.size(-1), "]");
  like(w_, x_, "weight", "x");
  if (res_.defined()) {
    on_gpu(res_, "residual");
    like(res_, x_, "residual", "x");
    TORCH_CHECK(res_.sizes() == x_.sizes(), "dgsparse: residual must have the shape of x");
  }
  TORCH_CHECK(eps >= 0.0, "dgsparse: eps must not be negative");
  const Guard guard(x_.device());
  const int64_t D = x_.size(-1), rows = x_.numel() / D;
  NormOut o;
  o.y = at::empty(x_.sizes(), x_.options().dtype(fp8 ? at::kFloat8_e4m3fn : x_.scalar_type()));
  if (res_.defined()) o.s = at::empty(x_.sizes(), x_.options());
  if (fp8) {
    auto shape = x_.sizes().vec();
    shape.back() = (D + 127) / 128;
    o.scales = at::empty(shape, x_.options().dtype(at::kFloat));
  }
  if (rows == 0) return o;
  int64_t ldx = D, ldr = D;
  const Tensor x = rows_of(x_, ldx), res = res_.defined() ? rows_of(res_, ldr) : Tensor(), w = w_.contiguous();
  check_rc(dgs_rms_norm(dtype, rows, D, x.data_ptr(), ldx, res.defined() ? res.data_ptr() : nullptr, ldr, w.data_ptr(), (float)eps,
                        fp8 ? nullptr : o.y.data_ptr(), o.s.defined() ? o.s.data_ptr() : nullptr,
                        fp8 ? static_cast<uint8_t *>(o.y.data_ptr()) : nullptr, fp8 ? o.scales.data_ptr<float>() : nullptr, cur_stream()),
           "rms_norm");
  return o;
}
// (dx, dweight) from the normed rows s; dy or ds may be undefined (an output that nothing was computed from)
std::tuple<Tensor, Tensor> norm_bwd(const Tensor &s_, const Tensor &w_, double eps, const Tensor &dy_, const Tensor &ds_, bool need_w) {
  once("rms_norm");
  const Guard guard(s_.device());
  const int64_t D = s_.size(-1), rows = s_.numel() / D;
  if (!dy_.defined() || rows == 0) {
    Tensor dx = ds_.defined() ? ds_ : at::zeros_like(s_);
    return {dx, need_w ? at::zeros_like(w_) : Tensor()};
  }
  const Tensor s = s_.contiguous(), w = w_.contiguous(), dy = dy_.contiguous(), ds = ds_.defined() ? ds_.contiguous() : Tensor();
  const int dtype = dtype_of(s, "x");
  Tensor dx = at::empty(s.sizes(), s.options()), dw = need_w ? at::empty(w.sizes(), w.options()) : Tensor();
  const size_t wsb = need_w ? dgs_rms_norm_bwd_workspace_bytes(dtype, rows, D) : 0;
  Tensor ws = wsb ? workspace(wsb, s) : Tensor();
  check_rc(dgs_rms_norm_bwd(dtype, rows, D, s.data_ptr(), w.data_ptr(), (float)eps, dy.data_ptr(), ds.defined() ? ds.data_ptr() : nullptr,
                            dx.data_ptr(), need_w ? dw.data_ptr() : nullptr, wsb ? ws.data_ptr() : nullptr, wsb, cur_stream()),
           "rms_norm backward");
  return {dx, dw};
}
struct RmsNorm : public torch::autograd::Function<RmsNorm> {
  static Tensor forward(AutogradContext *ctx, Tensor x, Tensor weight, double eps) {
    ctx->save_for_backward({x, weight});
    ctx->saved_data["eps"] = eps;
    return norm_fwd(x, Tensor(), weight, eps, false).y;
  }
  static tensor_list backward(AutogradContext *ctx, tensor_list grads) {
    const auto saved = ctx->get_saved_variables();
    auto [dx, dw] = norm_bwd(saved[0], saved[1], ctx->saved_data["eps"].toDouble(), grads[0], Tensor(), ctx->needs_input_grad(1));
    return {dx, dw, Tensor()};
  }
};
struct AddRmsNorm : public torch::autograd::Function<AddRmsNorm> {
  static tensor_list forward(AutogradContext *ctx, Tensor x, Tensor residual, Tensor weight, double eps) {
    ctx->set_materialize_grads(false);
    NormOut o = norm_fwd(x, residual, weight, eps, false);
    ctx->save_for_backward({o.s, weight});
    ctx->saved_data["eps"] = eps;
    return {o.y, o.s};
  }
  static tensor_list backward(AutogradContext *ctx, tensor_list grads) {
    const auto saved = ctx->get_saved_variables();
    auto [dx, dw] = norm_bwd(saved[0], saved[1], ctx->saved_data["eps"].toDouble(), grads[0], grads[1], ctx->needs_input_grad(2));
    return {dx, dx, dw, Tensor()};
  }
};
Tensor rms_norm_op(Tensor x, Tensor weight, double eps) {
  no_tangent("rms_norm", {&x, &weight});
  if (!(at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad()))) return norm_fwd(x, Tensor(), weight, eps, false).y;
  return RmsNorm::apply(x, weight, eps);
}
std::tuple<Tensor, Tensor> add_rms_norm_op(Tensor x, Tensor residual, Tensor weight, double eps) {
  no_tangent("add_rms_norm", {&x, &residual, &weight});
  if (!(at::GradMode::is_enabled() && (x.requires_grad() || residual.requires_grad() || weight.requires_grad()))) {
    NormOut o = norm_fwd(x, residual, weight, eps, false);
    return {o.y, o.s};
  }
  auto r = AddRmsNorm::apply(x, residual, weight, eps);
  return {r[0], r[1]};
}
std::tuple<Tensor, Tensor, Tensor> add_rms_norm_fp8_op(Tensor x, Tensor residual, Tensor weight, double eps) {
  NormOut o = norm_fwd(x, residual, weight, eps, true);
  return {o.y, o.scales, o.s};
}

// ---- gated feed-forward ----------------------------------------------------------------------------------------------------
// rows whose base and distance suit 16-byte accesses, and whose distance the entries take (256 rows within 32 bits of bytes): t as it is, or a
// contiguous copy (of [batch, length, features][:, -1], say: few rows, far apart)
Tensor rows16_of(const Tensor &t, int64_t &ld) {
  Tensor r = rows_of(t, ld);
  const int64_t size = (int64_t)r.element_size(), v = 16 / size;
  const bool far = ld > std::max<int64_t>(INT32_MAX / 256 / size - 64, r.size(-1));
  if (far || (r.size(-1) % v == 0 && (ld % v || reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 || ld < r.size(-1)))) {
    r = r.clone(at::MemoryFormat::Contiguous);
    ld = r.size(-1);
  }
  return r;
}
Tensor aligned_contiguous(const Tensor &t) {
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}
void ffn_check(const Tensor &x, const Tensor &wg, const Tensor &wu, int64_t activation) {
  on_gpu(x, "x");
  on_gpu(wg, "w_gate");
  on_gpu(wu, "w_up");
  dtype_of(x, "x");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, "dgsparse: x must have at least one feature");
  TORCH_CHECK(wg.dim() == 2 && wg.size(1) == x.size(-1) && wg.size(0) > 0, "dgsparse: w_gate must be [hidden, ", x.size(-1), "] with hidden > 0");
  TORCH_CHECK(wu.sizes() == wg.sizes(), "dgsparse: w_up must have the shape of w_gate");
  like(wg, x, "w_gate", "x");
  like(wu, x, "w_up", "x");
  TORCH_CHECK(activation >= DGS_ACT_SILU && activation <= DGS_ACT_RELU, "dgsparse: unknown activation ", activation);
}
struct FfnIn { Tensor x, wg, wu; int64_t rows, D, F, ldx, ldw; int dtype; };
FfnIn ffn_in(const Tensor &x_, const Tensor &wg_, const Tensor &wu_) {
  FfnIn i;
  i.dtype = dtype_of(x_, "x");
  i.D = x_.size(-1);
  i.F = wg_.size(0);
  i.rows = x_.numel() / i.D;
  int64_t ldu = 0;
  i.x = rows16_of(x_, i.ldx);
  i.wg = rows16_of(wg_, i.ldw);
  i.wu = rows16_of(wu_, ldu);
  if (ldu != i.ldw) {  // (one distance for both)
    i.wg = wg_.clone(at::MemoryFormat::Contiguous);
    i.wu = wu_.clone(at::MemoryFormat::Contiguous);
    i.ldw = i.D;
  }
  return i;
}
// Whether the forward pass keeps the two products in 32 bits for the backward pass, where the caller leaves it open (keep < 0).  Kept they cost
// 16 bytes of memory traffic for each value of h, made again 4 D flops.  rows x D x F, forward and backward, kept and made again, us, 32 bits:
// 169343 x 128 x 512 1198 and 1176, 16384 x 160 x 1024 350 and 367, 30000 x 300 x 600 578 and 663, 4096 x 768 x 2048 580 and 712; bf16:
// 32768 x 256 x 1024 369 and 303, 16384 x 512 x 2048 481 and 465, 16384 x 768 x 2816 754 and 753, 8192 x 1024 x 2816 473 and 507, 4096 x 2048 x 5504 672 and 757.
// Beyond 1 GiB of them they are made again, so that a deep model's activations stay its own.
bool ffn_keeps(const Tensor &x, const Tensor &wg, int64_t keep) {
  if (keep >= 0) return keep != 0;
  const int64_t D = x.size(-1), count = x.numel() / D * wg.size(0);
  return D >= (x.element_size() == 4 ? 160 : 1024) && count <= (int64_t(1) << 27);
}
Tensor ffn_fwd(const Tensor &x, const Tensor &wg, const Tensor &wu, int64_t activation, Tensor *pre = nullptr) {
  const Guard guard(x.device());
  auto shape = x.sizes().vec();
  shape.back() = wg.size(0);
  Tensor h = at::empty(shape, x.options());
  if (h.numel() == 0) return h;
  const FfnIn i = ffn_in(x, wg, wu);
  if (pre) *pre = at::empty({2, i.rows, i.F}, x.options().dtype(at::kFloat));
  const size_t wsb = dgs_gated_ffn_workspace_bytes(i.dtype, i.rows, i.D, i.F, 0);
  Tensor ws = wsb ? workspace(wsb, x) : Tensor();
  check_rc(dgs_gated_ffn(i.dtype, (int)activation, i.rows, i.D, i.F, i.x.data_ptr(), i.ldx, i.wg.data_ptr(), i.wu.data_ptr(), i.ldw, h.data_ptr(),
                         pre ? pre->data_ptr<float>() : nullptr, wsb ? ws.data_ptr() : nullptr, wsb, cur_stream()),
           "gated_ffn");
  return h;
}
struct GatedFfn : public torch::autograd::Function<GatedFfn> {
  static Tensor forward(AutogradContext *ctx, Tensor x, Tensor wg, Tensor wu, int64_t activation, int64_t keep) {
    Tensor pre;
    Tensor h = ffn_fwd(x, wg, wu, activation, ffn_keeps(x, wg, keep) && x.numel() ? &pre : nullptr);
    ctx->save_for_backward({x, wg, wu, pre});
    ctx->saved_data["act"] = activation;
    return h;
  }
  static tensor_list backward(AutogradContext *ctx, tensor_list grads) {
    once("gated_ffn");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &wg = saved[1], &wu = saved[2];
    const Guard guard(x.device());
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    Tensor dx = need_x ? at::empty(x.sizes(), x.options()) : Tensor();
    Tensor dwg = need_w ? at::empty(wg.sizes(), wg.options()) : Tensor(), dwu = need_w ? at::empty(wu.sizes(), wu.options()) : Tensor();
    if (x.numel() == 0) {
      if (need_w) {
        dwg.zero_();
        dwu.zero_();
      }
      return {dx, dwg, dwu, Tensor(), Tensor()};
    }
    const FfnIn i = ffn_in(x, wg, wu);
    const Tensor dh = aligned_contiguous(grads[0]);
    const size_t wsb = dgs_gated_ffn_workspace_bytes(i.dtype, i.rows, i.D, i.F, 1);
    Tensor ws = workspace(wsb, x);
    check_rc(dgs_gated_ffn_bwd(i.dtype, (int)ctx->saved_data["act"].toInt(), i.rows, i.D, i.F, i.x.data_ptr(), i.ldx, i.wg.data_ptr(), i.wu.data_ptr(), i.ldw,
                               saved[3].defined() ? saved[3].data_ptr<float>() : nullptr, dh.data_ptr(), need_x ? dx.data_ptr() : nullptr, need_w ? dwg.data_ptr() : nullptr, need_w ? dwu.data_ptr() : nullptr,
                               ws.data_ptr(), wsb, cur_stream()),
             "gated_ffn backward");
    return {dx, dwg, dwu, Tensor(), Tensor()};
  }
};
Tensor gated_ffn_op(Tensor x, Tensor wg, Tensor wu, int64_t activation, int64_t keep) {
  ffn_check(x, wg, wu, activation);
  no_tangent("gated_ffn", {&x, &wg, &wu});
  if (!(at::GradMode::is_enabled() && (x.requires_grad() || wg.requires_grad() || wu.requires_grad()))) return ffn_fwd(x, wg, wu, activation);
  return GatedFfn::apply(x, wg, wu, activation, keep);
}

// ---- 8 bits ----------------------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> quantize_fp8_op(Tensor x_, int64_t block_rows) {
  on_gpu(x_, "x");
  const int dtype = dtype_of(x_, "x");
  TORCH_CHECK(x_.dim() >= 1 && x_.size(-1) > 0, "dgsparse: x must have at least one feature");
  TORCH_CHECK(block_rows == 1 || (block_rows == 128 && x_.dim() == 2), "dgsparse: block_rows is 1, or 128 for a 2-D tensor");
  const Guard guard(x_.device());
  const int64_t cols = x_.size(-1), rows = x_.numel() / cols;
  auto shape = x_.sizes().vec();
  shape.back() = (cols + 127) / 128;
  if (block_rows == 128) shape[0] = (rows + 127) / 128;
  Tensor q = at::empty(x_.sizes(), x_.options().dtype(at::kFloat8_e4m3fn)), scales = at::empty(shape, x_.options().dtype(at::kFloat));
  if (rows == 0) return {q, scales};
  int64_t ld = cols;
  const Tensor x = rows_of(x_, ld);
  check_rc(dgs_quantize_fp8(dtype, rows, cols, x.data_ptr(), ld, (int)block_rows, static_cast<uint8_t *>(q.data_ptr()), scales.data_ptr<float>(), cur_stream()),
           "quantize_fp8");
  return {q, scales};
}
Tensor matmul_fp8_op(Tensor a_, Tensor a_scale, Tensor b_, Tensor b_scale, at::ScalarType out_dtype) {
  on_gpu(a_, "a");
  on_gpu(a_scale, "a_scale");
  on_gpu(b_, "b");
  on_gpu(b_scale, "b_scale");
  TORCH_CHECK(a_.scalar_type() == at::kFloat8_e4m3fn && b_.scalar_type() == at::kFloat8_e4m3fn, "dgsparse: a and b must be float8_e4m3fn, not ",
              a_.scalar_type(), " and ", b_.scalar_type());
  TORCH_CHECK(a_scale.scalar_type() == at::kFloat && b_scale.scalar_type() == at::kFloat, "dgsparse: the scales must be float32");
  TORCH_CHECK(a_.dim() >= 1 && b_.dim() == 2 && a_.size(-1) == b_.size(1) && b_.size(1) > 0, "dgsparse: a must be [..., K] and b [N, K]");
  TORCH_CHECK(a_.device() == b_.device() && a_scale.device() == a_.device() && b_scale.device() == a_.device(), "dgsparse: a, b and their scales live on different devices");
  const int64_t K = a_.size(-1), M = a_.numel() / K, N = b_.size(0), blocks = (K + 127) / 128;
  auto shape = a_.sizes().vec();
  shape.back() = blocks;
  TORCH_CHECK(a_scale.sizes() == at::IntArrayRef(shape), "dgsparse: a_scale must be ", at::IntArrayRef(shape), ", one for each row and 128 of K");
  TORCH_CHECK(b_scale.dim() == 2 && b_scale.size(0) == (N + 127) / 128 && b_scale.size(1) == blocks, "dgsparse: b_scale must be [", (N + 127) / 128, ", ", blocks,
              "], one for each 128 x 128 of b");
  const Guard guard(a_.device());
  shape.back() = N;
  Tensor out = at::empty(shape, a_.options().dtype(out_dtype));
  const int dtype = dtype_of(out, "the result");
  if (out.numel() == 0) return out;
  int64_t lda = K, ldb = K;
  const Tensor a = rows16_of(a_, lda), b = rows16_of(b_, ldb), as = a_scale.contiguous(), bs = b_scale.contiguous();
  const size_t wsb = dgs_matmul_fp8_workspace_bytes(M, N, K);
  Tensor ws = wsb ? workspace(wsb, a) : Tensor();
  check_rc(dgs_matmul_fp8(dtype, M, N, K, static_cast<const uint8_t *>(a.data_ptr()), lda, as.data_ptr<float>(), static_cast<const uint8_t *>(b.data_ptr()), ldb,
                          bs.data_ptr<float>(), out.data_ptr(), wsb ? ws.data_ptr() : nullptr, wsb, cur_stream()),
           "matmul_fp8");
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(dgsparse_spmm, m) {
  m.def("embedding", &embedding_op);
  m.def("rms_norm", &rms_norm_op);
  m.def("add_rms_norm", &add_rms_norm_op);
  m.def("add_rms_norm_fp8", &add_rms_norm_fp8_op);
  m.def("gated_ffn", &gated_ffn_op);
  m.def("quantize_fp8", &quantize_fp8_op);
  m.def("matmul_fp8", &matmul_fp8_op);
}
