// C++ autograd nodes of the sparse window attention and of the encoder around
// it (linear layers, projection group, LayerNorms).
//
// Sparse attention: the same operation and contract as SparseAttentionFunction in attention.py
// (the reference op is CoreAttention.sparse_attention_bias,
// NeutronGT/models/graphormer_dist_node_level.py:67-98): (q, k, v) ->
// (out, node_scores), node scores without gradient, optional detached extra
// key rows (k_ext, v_ext).  Forward and backward call the library's C ABI
// (ngt_sparse_fwd_ext / ngt_sparse_bwd_strided) through function pointers that the
// Python side hands over once from the loaded libngt_attn.so, so a layer's
// forward and backward run no Python frame, take no GIL on the autograd
// engine's device thread and convert no ctypes arguments.  Host code only:
// every kernel is in libngt_attn.so.
//
// The window is passed as two tensors: `csr` (CPU bytes of one
// ngt_window_csr) and `csr_mem` (the device allocation its pointers point
// into).  Both are kept by the node until the backward has run.
//
// q, k, v may also come as [1, n, H, d], the layout the encoders hold: the
// output is then [1, n_q, H * d] and the gradients have the inputs' shape, so
// that no view node stands between the projections, the core and the output
// projection.
//
// Linear, Projection3, LayerNorm and AddLayerNorm are _WgradLinearFn,
// _ProjectionGroupFn (of three layers), _LayerNormFn and _AddLayerNormFn of
// linear.py and layernorm.py: the same casts, library GEMMs and kernels in the
// same order, bit for bit.  Those Python nodes and the view nodes cost 10-60 us
// of host time each: forward and backward of the 3-layer GPH_Slim model (254
// launches, 1.4 ms of kernels) took 4.0 ms and take 2.9, a GPH_Large block
// over 10,007 queries 1.37 -> 0.97 ms, and the core alone over a small window
// 113 -> 91 us (74 -> 60 us on a faster host).
//
// PackedAttention and LinearEpilogue are PackedAttentionFunction (packed.py) and
// LinearEpilogueFunction (linear.py); GatedLinear and NormRotary GatedLinearFunction
// (linear.py) and NormRotaryFunction (rotary.py).  Their entries return nothing where an
// argument is not one that they take (a forward-mode dual tensor among them, whose
// tangent a call without gradients would drop): Python then checks it and says why.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <string>
#include <unordered_set>

#include "ngt_attn.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;

decltype(&ngt_sparse_fwd_ext) g_fwd = nullptr;
decltype(&ngt_sparse_bwd_strided) g_bwd = nullptr;
decltype(&ngt_last_error) g_err = nullptr;
decltype(&ngt_colsum_workspace_bytes) g_colsum_ws = nullptr;
decltype(&ngt_colsum_bf16) g_colsum = nullptr;
decltype(&ngt_chunk_sum_f32) g_chunk_sum = nullptr;
decltype(&ngt_wgrad_workspace_bytes) g_wgrad_ws = nullptr;
decltype(&ngt_wgrad_pays) g_wgrad_pays = nullptr;
decltype(&ngt_wgrad_bf16) g_wgrad = nullptr;
decltype(&ngt_layernorm_fwd) g_ln_fwd = nullptr;
decltype(&ngt_layernorm_bwd_workspace_bytes) g_ln_bwd_ws = nullptr;
decltype(&ngt_layernorm_bwd) g_ln_bwd = nullptr;
decltype(&ngt_add_layernorm_fwd) g_add_ln_fwd = nullptr;
decltype(&ngt_add_layernorm_bwd) g_add_ln_bwd = nullptr;
decltype(&ngt_packed_workspace_bytes) g_packed_ws = nullptr;
decltype(&ngt_packed_fwd) g_packed_fwd = nullptr;
decltype(&ngt_packed_bwd) g_packed_bwd = nullptr;
decltype(&ngt_linear_fwd) g_linear_fwd = nullptr;
decltype(&ngt_linear_bwd_workspace_bytes) g_linear_bwd_ws = nullptr;
decltype(&ngt_linear_bwd) g_linear_bwd = nullptr;
decltype(&ngt_gated_keep_bytes) g_gated_keep = nullptr;
decltype(&ngt_gated_fwd_workspace_bytes) g_gated_fwd_ws = nullptr;
decltype(&ngt_gated_fwd) g_gated_fwd = nullptr;
decltype(&ngt_gated_bwd_workspace_bytes) g_gated_bwd_ws = nullptr;
decltype(&ngt_gated_bwd) g_gated_bwd = nullptr;
decltype(&ngt_norm_rotary_fwd) g_rotary_fwd = nullptr;
decltype(&ngt_norm_rotary_bwd_workspace_bytes) g_rotary_bwd_ws = nullptr;
decltype(&ngt_norm_rotary_bwd) g_rotary_bwd = nullptr;
decltype(&ngt_clip_workspace_bytes) g_clip_ws = nullptr;
decltype(&ngt_clip_gradients) g_clip = nullptr;

void check(int rc) {
  if (rc != NGT_OK) {
    const char* msg = g_err ? g_err() : nullptr;
    TORCH_CHECK(!(msg && *msg), msg);
    TORCH_CHECK(false, "libngt_attn error ", rc);
  }
}

int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kFloat) return NGT_F32;
  if (t.scalar_type() == at::kBFloat16) return NGT_BF16;
  TORCH_CHECK(false, "unsupported dtype ", t.scalar_type(), " (float32 or bfloat16)");
  return -1;
}

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

const ngt_window_csr* csr_of(const Tensor& bytes) {
  return reinterpret_cast<const ngt_window_csr*>(bytes.data_ptr());
}

// 16-byte aligned contiguous rows, as the library requires
Tensor rows16(const Tensor& t) {
  if (!t.is_contiguous()) return t.contiguous();
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return t.clone();
  return t;
}

// The library reads rows [n, H, d] of one dtype from 16-byte aligned,
// contiguous GPU memory on q's device; anything else is an error here rather
// than wrong reads in the kernels.
void check_rows(const char* name, const Tensor& t, const Tensor& q) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(t.device() == q.device(), name, " is on ", t.device(), ", q on ", q.device());
  TORCH_CHECK(t.scalar_type() == q.scalar_type(), name, " has dtype ", t.scalar_type(),
              ", q has ", q.scalar_type());
  TORCH_CHECK((t.dim() == 3 || (t.dim() == 4 && t.size(0) == 1)) && t.size(-2) == q.size(-2) &&
                  t.size(-1) == q.size(-1),
              name, " must be [n, ", q.size(-2), ", ", q.size(-1), "], got ", t.sizes());
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name,
              " must be 16-byte aligned");
}

Tensor workspace(int64_t bytes, const Tensor& like) {
  return at::empty({std::max<int64_t>(bytes, 1)}, like.options().dtype(at::kByte));
}

constexpr int kInputs = 15;  // forward arguments after ctx

struct SparseAttention : public torch::autograd::Function<SparseAttention> {
  static tensor_list forward(AutogradContext* ctx, Tensor q, Tensor k, Tensor v,
                             std::optional<Tensor> k_ext_opt, std::optional<Tensor> v_ext_opt,
                             Tensor csr, Tensor csr_mem, int64_t dst_end,
                             double scale, double lo, double hi, double eps, int64_t fwd_bytes,
                             int64_t bwd_bytes, bool interleave_grads) {
    TORCH_CHECK(g_fwd && g_bwd, "ngt_autograd.init() was not called");
    // an absent argument is an empty optional: autograd inputs may not be
    // undefined tensors
    const Tensor k_ext = k_ext_opt.value_or(Tensor()), v_ext = v_ext_opt.value_or(Tensor());
    const bool ext = k_ext.defined();
    TORCH_CHECK(ext == v_ext.defined(), "k_ext and v_ext must be given together");
    check_rows("q", q, q);
    check_rows("k", k, q);
    check_rows("v", v, q);
    TORCH_CHECK(k.sizes() == v.sizes(), "k and v differ in shape: ", k.sizes(), " vs ", v.sizes());
    if (ext) {
      check_rows("k_ext", k_ext, q);
      check_rows("v_ext", v_ext, q);
      TORCH_CHECK(k_ext.sizes() == v_ext.sizes(), "k_ext and v_ext differ in shape");
    }
    TORCH_CHECK(q.dim() == k.dim(), "q and k differ in dimensions");
    const int64_t n_q = q.size(-3), n_k = k.size(-3), H = q.size(-2), d = q.size(-1);
    Tensor out = q.dim() == 4 ? at::empty({1, n_q, H * d}, q.options()) : at::empty_like(q);
    const auto f32 = q.options().dtype(at::kFloat);
    Tensor rinv = at::empty({n_q, H}, f32);
    Tensor ns = at::empty({dst_end}, f32);
    Tensor ws = workspace(fwd_bytes, q);
    check(g_fwd(dtype_code(q), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                ext ? k_ext.data_ptr() : nullptr, ext ? v_ext.data_ptr() : nullptr,
                static_cast<int32_t>(n_k), csr_of(csr), static_cast<int32_t>(H),
                static_cast<int32_t>(d), static_cast<float>(scale), static_cast<float>(lo),
                static_cast<float>(hi), static_cast<float>(eps), out.data_ptr(),
                rinv.data_ptr<float>(), dst_end ? ns.data_ptr<float>() : nullptr,
                static_cast<int32_t>(dst_end), ws.data_ptr(), static_cast<size_t>(fwd_bytes),
                stream_of(q)));
    ctx->save_for_backward({q, k, v, out, rinv});
    ctx->saved_data["k_ext"] = k_ext;  // detached key rows (no gradient)
    ctx->saved_data["v_ext"] = v_ext;
    ctx->saved_data["csr"] = csr;
    ctx->saved_data["csr_mem"] = csr_mem;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["lo"] = lo;
    ctx->saved_data["hi"] = hi;
    ctx->saved_data["bwd_bytes"] = bwd_bytes;
    ctx->saved_data["interleave"] = interleave_grads && n_q == n_k;
    ctx->mark_non_differentiable({ns});
    // the node scores have no gradient: no zero tensor is made for them
    ctx->set_materialize_grads(false);
    return {out, ns};
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    tensor_list res(kInputs);
    if (!grads[0].defined()) return res;  // the output was not used by the loss
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &rinv = saved[4];
    const Tensor k_ext = ctx->saved_data["k_ext"].toTensor();
    const Tensor v_ext = ctx->saved_data["v_ext"].toTensor();
    const Tensor csr = ctx->saved_data["csr"].toTensor();
    const int64_t bwd_bytes = ctx->saved_data["bwd_bytes"].toInt();
    const Tensor g = rows16(grads[0].to(q.scalar_type()));
    const int64_t n_q = q.size(-3), n_k = k.size(-3), H = q.size(-2), d = q.size(-1);
    Tensor gq, gk, gv;
    int64_t ldg = 0;
    if (ctx->saved_data["interleave"].toBool()) {
      // one [N, 3, H, d] buffer: row i holds dQ, dK, dV of row i side by side
      const Tensor buf = at::empty({n_q, 3, H, d}, q.options());
      ldg = 3 * H * d;
      const auto rows = q.dim() == 4 ? std::vector<int64_t>{n_q * ldg, ldg, d, 1}
                                     : std::vector<int64_t>{ldg, d, 1};
      gq = buf.as_strided(q.sizes(), rows, 0);
      gk = buf.as_strided(q.sizes(), rows, H * d);
      gv = buf.as_strided(q.sizes(), rows, 2 * H * d);
    } else {
      gq = at::empty_like(q);
      gk = at::empty_like(k);
      gv = at::empty_like(v);
    }
    Tensor ws = workspace(bwd_bytes, q);
    const bool ext = k_ext.defined();
    check(g_bwd(dtype_code(q), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                ext ? k_ext.data_ptr() : nullptr, ext ? v_ext.data_ptr() : nullptr,
                static_cast<int32_t>(n_k), out.data_ptr(), g.data_ptr(),
                rinv.data_ptr<float>(), csr_of(csr), static_cast<int32_t>(H),
                static_cast<int32_t>(d),
                static_cast<float>(ctx->saved_data["scale"].toDouble()),
                static_cast<float>(ctx->saved_data["lo"].toDouble()),
                static_cast<float>(ctx->saved_data["hi"].toDouble()), gq.data_ptr(),
                gk.data_ptr(), gv.data_ptr(), ldg, ws.data_ptr(), static_cast<size_t>(bwd_bytes),
                stream_of(q)));
    res[0] = gq;
    res[1] = gk;
    res[2] = gv;
    return res;
  }
};

std::tuple<Tensor, Tensor> sparse_attention(Tensor q, Tensor k, Tensor v,
                                            std::optional<Tensor> k_ext,
                                            std::optional<Tensor> v_ext, Tensor csr,
                                            Tensor csr_mem, int64_t dst_end, double scale,
                                            double lo, double hi, double eps, int64_t fwd_bytes,
                                            int64_t bwd_bytes, bool interleave_grads) {
  TORCH_CHECK(csr.device().is_cpu() && csr.scalar_type() == at::kByte &&
                  csr.numel() == static_cast<int64_t>(sizeof(ngt_window_csr)),
              "csr must hold the bytes of one ngt_window_csr (", sizeof(ngt_window_csr), ")");
  auto r = SparseAttention::apply(q, k, v, k_ext, v_ext, csr, csr_mem, dst_end, scale, lo, hi, eps,
                                  fwd_bytes, bwd_bytes, interleave_grads);
  return {r[0], r[1]};
}

// ------------------------------------------------------- the encoder's layers
// torch's casts of the operands stay off inside these nodes: their GEMMs take
// the operands as they are
struct NoAutocast {
  c10::impl::ExcludeDispatchKeyGuard guard{c10::autocast_dispatch_keyset};
};

constexpr int64_t kChunk = 2048;  // as _CHUNK and _MAX_SPLITS of linear.py
constexpr int64_t kMaxSplits = 16;

// fp32 column sums of a contiguous bf16 [K, n] matrix
Tensor colsum(const Tensor& dy) {
  const int64_t K = dy.size(0);
  const auto n = static_cast<int32_t>(dy.size(1));
  Tensor out = at::empty({n}, dy.options().dtype(at::kFloat));
  size_t bytes = 0;
  check(g_colsum_ws(K, n, &bytes));
  Tensor ws = workspace(static_cast<int64_t>(bytes), dy);
  check(g_colsum(dy.data_ptr(), K, n, out.data_ptr<float>(), ws.data_ptr(), bytes, stream_of(dy)));
  return out;
}

// dY^T X in fp32 by library GEMMs split over rows (_library_weight_grad of
// linear.py)
Tensor library_weight_grad(const Tensor& x, const Tensor& dy) {
  const int64_t K = x.size(0), n_in = x.size(1), n_out = dy.size(1);
  const int64_t most = n_out * n_in < 1500000 ? kMaxSplits : kMaxSplits / 2;
  const int64_t splits = std::max<int64_t>(1, std::min(most, K / kChunk));
  const int64_t c = K / splits, main = splits * c;
  if (splits == 1) return at::mm(dy.t(), x, at::kFloat);
  Tensor parts = at::bmm(dy.narrow(0, 0, main).view({splits, c, n_out}).transpose(1, 2),
                         x.narrow(0, 0, main).view({splits, c, n_in}), at::kFloat)
                     .contiguous();
  Tensor dw = at::empty({n_out, n_in}, parts.options());
  check(g_chunk_sum(parts.data_ptr<float>(), static_cast<int32_t>(splits), n_out * n_in,
                    dw.data_ptr<float>(), stream_of(x)));
  if (main < K) dw.add_(at::mm(dy.narrow(0, main, K - main).t(), x.narrow(0, main, K - main),
                               at::kFloat));
  return dw;
}

// dw = dY^T X and, where wanted, db = column sums of dY, in fp32 from
// contiguous bf16 rows (_grads of linear.py).  x may be undefined where dw is not
// wanted.
void linear_grads(const Tensor& x, const Tensor& dy, Tensor* dw, Tensor* db) {
  if (!dw) {
    if (db) *db = colsum(dy);
    return;
  }
  const int64_t K = x.size(0), n_in = x.size(1), n_out = dy.size(1);
  // (a vmapped backward's tensors have no storage: torch's GEMMs take them)
  if (at::GradMode::is_enabled() || !x.has_storage() || !dy.has_storage() ||
      !g_wgrad_pays(K, n_out, n_in)) {
    *dw = library_weight_grad(x, dy);
    if (db) *db = colsum(dy);
    return;
  }
  const auto opt = x.options().dtype(at::kFloat);
  *dw = at::empty({n_out, n_in}, opt);
  if (db) *db = at::empty({n_out}, opt);
  size_t bytes = 0;
  check(g_wgrad_ws(K, static_cast<int32_t>(n_out), static_cast<int32_t>(n_in), &bytes));
  Tensor ws = workspace(static_cast<int64_t>(bytes), x);
  check(g_wgrad(x.data_ptr(), dy.data_ptr(), K, static_cast<int32_t>(n_out),
                static_cast<int32_t>(n_in), dw->data_ptr<float>(),
                db ? db->data_ptr<float>() : nullptr, ws.data_ptr(), bytes, stream_of(x)));
}

Tensor bf16(const Tensor& t) { return t.to(at::kBFloat16); }

std::optional<Tensor> bf16(const std::optional<Tensor>& t) {
  return t.has_value() ? std::optional<Tensor>(bf16(*t)) : std::nullopt;
}

// y = x W^T + b in bf16; fp32 dW and db
struct Linear : public torch::autograd::Function<Linear> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor weight,
                        std::optional<Tensor> bias) {
    NoAutocast off;
    const Tensor x16 = bf16(x), w16 = bf16(weight);
    Tensor y = at::linear(x16, w16, bf16(bias));
    ctx->save_for_backward({x16, w16});
    ctx->saved_data["bias"] = bias.has_value();
    return y;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    NoAutocast off;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x16 = saved[0], &w16 = saved[1];
    const int64_t n_out = w16.size(0), n_in = w16.size(1);
    tensor_list res(3);
    const Tensor g2 = bf16(grads[0]).reshape({-1, n_out}).contiguous();
    if (ctx->needs_input_grad(0)) res[0] = at::mm(g2, w16).view(x16.sizes());
    const bool want_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
    const bool want_w = ctx->needs_input_grad(1);
    linear_grads(want_w ? x16.reshape({-1, n_in}).contiguous() : Tensor(), g2,
                 want_w ? &res[1] : nullptr, want_b ? &res[2] : nullptr);
    return res;
  }
};

Tensor linear(Tensor x, Tensor weight, std::optional<Tensor> bias) {
  return Linear::apply(x, weight, bias);
}

// the [M, 3 * n_out] matrix whose column blocks are the gradients g, when they
// are views of one buffer laid out that way (linear.py's _joint_rows, the one
// place that knows the layout); else undefined
Tensor joint_rows(const tensor_list& g, int64_t n_out) {
  pybind11::gil_scoped_acquire gil;
  pybind11::tuple views(g.size());
  for (size_t i = 0; i < g.size(); ++i)
    views[i] = g[i].defined() ? pybind11::cast(g[i]) : pybind11::none();
  const pybind11::object r =
      pybind11::module_::import("neutrongt_amd.linear").attr("_joint_rows")(views, n_out);
  return r.is_none() ? Tensor() : r.cast<Tensor>();
}

// Three projections of one input (Q, K, V) as one node.  heads > 0: the
// outputs as [..., heads, n_out / heads].
struct Projection3 : public torch::autograd::Function<Projection3> {
  static tensor_list forward(AutogradContext* ctx, Tensor x, Tensor w0, std::optional<Tensor> b0,
                             Tensor w1, std::optional<Tensor> b1, Tensor w2,
                             std::optional<Tensor> b2, int64_t heads) {
    NoAutocast off;
    const Tensor x16 = bf16(x);
    const Tensor w[3] = {bf16(w0), bf16(w1), bf16(w2)};
    const std::optional<Tensor> b[3] = {b0, b1, b2};
    tensor_list ys;
    int64_t has_bias = 0;
    for (int i = 0; i < 3; ++i) {
      Tensor y = at::linear(x16, w[i], bf16(b[i]));
      if (heads > 0) {
        auto shape = y.sizes().vec();
        shape.back() /= heads;
        shape.insert(shape.end() - 1, heads);
        y = y.view(shape);
      }
      ys.push_back(y);
      has_bias |= int64_t(b[i].has_value()) << i;
    }
    ctx->save_for_backward({x16, w[0], w[1], w[2]});
    ctx->saved_data["bias"] = has_bias;
    ctx->set_materialize_grads(false);  // an unused output: no GEMMs, no weight gradient
    return ys;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    NoAutocast off;
    const auto saved = ctx->get_saved_variables();
    const Tensor& x16 = saved[0];
    const tensor_list w(saved.begin() + 1, saved.end());
    const int64_t has_bias = ctx->saved_data["bias"].toInt();
    const int64_t n_in = x16.size(-1), n_out = w[0].size(0);
    // the node's edges are numbered over the tensors that were given
    bool want_w[3], want_b[3];
    size_t edge = 1;
    for (int i = 0; i < 3; ++i) {
      want_w[i] = ctx->needs_input_grad(edge++);
      want_b[i] = (has_bias >> i & 1) && ctx->needs_input_grad(edge++);
    }
    tensor_list res(8);
    Tensor joint;
    if (w[1].size(0) == n_out && w[2].size(0) == n_out && want_w[0] && want_w[1] && want_w[2] &&
        ((want_b[0] && want_b[1] && want_b[2]) || has_bias == 0))
      joint = joint_rows(grads, n_out);
    if (joint.defined()) {
      if (ctx->needs_input_grad(0)) res[0] = at::mm(joint, at::cat(w, 0)).view(x16.sizes());
      Tensor dw, db;
      linear_grads(x16.reshape({-1, n_in}).contiguous(), joint, &dw, has_bias ? &db : nullptr);
      for (int i = 0; i < 3; ++i) {
        res[1 + 2 * i] = dw.narrow(0, i * n_out, n_out);
        if (has_bias) res[2 + 2 * i] = db.narrow(0, i * n_out, n_out);
      }
      return res;
    }
    Tensor x2, gx;
    for (int i = 0; i < 3; ++i) {
      if (!grads[i].defined()) continue;
      const Tensor g2 = bf16(grads[i]).reshape({-1, w[i].size(0)}).contiguous();
      if (ctx->needs_input_grad(0)) {
        if (gx.defined())
          gx.addmm_(g2, w[i]);
        else
          gx = at::mm(g2, w[i]);
      }
      if (want_w[i] && !x2.defined()) x2 = x16.reshape({-1, n_in}).contiguous();
      linear_grads(x2, g2, want_w[i] ? &res[1 + 2 * i] : nullptr,
                   want_b[i] ? &res[2 + 2 * i] : nullptr);
    }
    if (gx.defined()) res[0] = gx.view(x16.sizes());
    return res;
  }
};

tensor_list project3(Tensor x, Tensor w0, std::optional<Tensor> b0, Tensor w1,
                     std::optional<Tensor> b1, Tensor w2, std::optional<Tensor> b2,
                     int64_t heads) {
  return Projection3::apply(x, w0, b0, w1, b1, w2, b2, heads);
}

// [n, n_cols] contiguous rows whose base meets the LayerNorm kernels'
// alignment: 16 bytes for fp32, 8 for bf16
Tensor ln_rows(const Tensor& t, int64_t n_cols) {
  const Tensor r = t.reshape({-1, n_cols});
  const uintptr_t align = r.scalar_type() == at::kFloat ? 16 : 8;
  if (!r.is_contiguous() || reinterpret_cast<uintptr_t>(r.data_ptr()) % align)
    return r.clone(at::MemoryFormat::Contiguous);
  return r;
}

Tensor ln_grad(const Tensor& g) {
  return g.scalar_type() == at::kFloat || g.scalar_type() == at::kBFloat16 ? g : g.to(at::kFloat);
}

Tensor f32(const Tensor& t) { return t.to(at::kFloat).contiguous(); }

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor weight, Tensor bias, double eps,
                        bool out_bf16) {
    NoAutocast off;
    const int64_t n_cols = weight.numel();
    const Tensor x2 = ln_rows(x, n_cols), w = f32(weight), b = f32(bias);
    const int64_t n = x2.size(0);
    const auto opt = x.options().dtype(at::kFloat);
    Tensor y = at::empty(x.sizes(), out_bf16 ? x.options().dtype(at::kBFloat16) : opt,
                         at::MemoryFormat::Contiguous);
    Tensor mean = at::empty({n}, opt), rstd = at::empty({n}, opt);
    check(g_ln_fwd(dtype_code(x2), x2.data_ptr(), n, static_cast<int32_t>(n_cols),
                   w.data_ptr<float>(), b.data_ptr<float>(), static_cast<float>(eps),
                   dtype_code(y), y.data_ptr(), mean.data_ptr<float>(), rstd.data_ptr<float>(),
                   stream_of(x)));
    ctx->save_for_backward({x2, w, mean, rstd});
    ctx->saved_data["shape"] = x.sizes().vec();
    return y;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    NoAutocast off;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x2 = saved[0], &w = saved[1], &mean = saved[2], &rstd = saved[3];
    const int64_t n = x2.size(0), n_cols = x2.size(1);
    const Tensor g2 = ln_rows(ln_grad(grads[0]), n_cols);
    Tensor dx = at::empty_like(x2);
    Tensor dw = at::empty({n_cols}, w.options()), db = at::empty({n_cols}, w.options());
    size_t bytes = 0;
    check(g_ln_bwd_ws(n, static_cast<int32_t>(n_cols), &bytes));
    Tensor ws = workspace(static_cast<int64_t>(bytes), x2);
    check(g_ln_bwd(dtype_code(x2), x2.data_ptr(), dtype_code(g2), g2.data_ptr(), n,
                   static_cast<int32_t>(n_cols), w.data_ptr<float>(), mean.data_ptr<float>(),
                   rstd.data_ptr<float>(), dx.data_ptr(), dw.data_ptr<float>(),
                   db.data_ptr<float>(), ws.data_ptr(), bytes, stream_of(x2)));
    return {dx.view(ctx->saved_data["shape"].toIntVector()), dw, db, Tensor(), Tensor()};
  }
};

Tensor layernorm(Tensor x, Tensor weight, Tensor bias, double eps, bool out_bf16) {
  return LayerNorm::apply(x, weight, bias, eps, out_bf16);
}

// (s, LayerNorm(s)) with s = x + dropout(y)
struct AddLayerNorm : public torch::autograd::Function<AddLayerNorm> {
  static tensor_list forward(AutogradContext* ctx, Tensor x, Tensor y, Tensor weight, Tensor bias,
                             double eps, double p, std::optional<Tensor> seed_opt, bool out_bf16) {
    NoAutocast off;
    const int64_t n_cols = weight.numel();
    const Tensor x2 = ln_rows(x, n_cols), y2 = ln_rows(y, n_cols), w = f32(weight), b = f32(bias);
    TORCH_CHECK(y2.scalar_type() == x2.scalar_type() && y2.sizes() == x2.sizes(),
                "x and y differ in dtype or shape");
    const Tensor seed = seed_opt.value_or(Tensor());
    const int64_t n = x2.size(0);
    const auto opt = x.options().dtype(at::kFloat);
    Tensor s = at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous);
    Tensor out = at::empty(x.sizes(), out_bf16 ? x.options().dtype(at::kBFloat16) : opt,
                           at::MemoryFormat::Contiguous);
    Tensor mean = at::empty({n}, opt), rstd = at::empty({n}, opt);
    check(g_add_ln_fwd(dtype_code(x2), x2.data_ptr(), y2.data_ptr(), n,
                       static_cast<int32_t>(n_cols), static_cast<float>(p), 0, seed_ptr(seed),
                       w.data_ptr<float>(), b.data_ptr<float>(), static_cast<float>(eps),
                       s.data_ptr(), dtype_code(out), out.data_ptr(), mean.data_ptr<float>(),
                       rstd.data_ptr<float>(), stream_of(x)));
    ctx->save_for_backward({s, w, mean, rstd, seed});
    ctx->saved_data["p"] = p;
    ctx->set_materialize_grads(false);  // an unused sum: no zero tensor for its gradient
    return {s, out};
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    NoAutocast off;
    const auto saved = ctx->get_saved_variables();
    const Tensor &s = saved[0], &w = saved[1], &mean = saved[2], &rstd = saved[3];
    const int64_t n = mean.numel(), n_cols = w.numel();
    tensor_list res(8);
    if (!grads[0].defined() && !grads[1].defined()) return res;
    const Tensor g_out =
        grads[1].defined() ? ln_rows(ln_grad(grads[1]), n_cols) : at::zeros({n, n_cols}, w.options());
    const Tensor g_s =
        grads[0].defined() ? ln_rows(grads[0].to(s.scalar_type()), n_cols) : Tensor();
    Tensor dx = at::empty_like(s), dy = at::empty_like(s);
    Tensor dw = at::empty({n_cols}, w.options()), db = at::empty({n_cols}, w.options());
    size_t bytes = 0;
    check(g_ln_bwd_ws(n, static_cast<int32_t>(n_cols), &bytes));
    Tensor ws = workspace(static_cast<int64_t>(bytes), s);
    check(g_add_ln_bwd(dtype_code(s), s.data_ptr(), dtype_code(g_out), g_out.data_ptr(),
                       g_s.defined() ? g_s.data_ptr() : nullptr, n, static_cast<int32_t>(n_cols),
                       static_cast<float>(ctx->saved_data["p"].toDouble()), 0, seed_ptr(saved[4]),
                       w.data_ptr<float>(), mean.data_ptr<float>(), rstd.data_ptr<float>(),
                       dx.data_ptr(), dy.data_ptr(), dw.data_ptr<float>(), db.data_ptr<float>(),
                       ws.data_ptr(), bytes, stream_of(s)));
    res[0] = dx;
    res[1] = dy;
    res[2] = dw;
    res[3] = db;
    return res;
  }

 private:
  static const uint64_t* seed_ptr(const Tensor& seed) {
    return seed.defined() ? static_cast<const uint64_t*>(seed.data_ptr()) : nullptr;
  }
};

std::tuple<Tensor, Tensor> add_layernorm(Tensor x, Tensor y, Tensor weight, Tensor bias, double eps,
                                         double p, std::optional<Tensor> seed, bool out_bf16) {
  auto r = AddLayerNorm::apply(x, y, weight, bias, eps, p, seed, out_bf16);
  return {r[0], r[1]};
}

// ------------------------------------------------------------ packed windows
// A forward-mode tangent, which requires_grad does not show.
bool has_tangent(const Tensor& t) { return t._fw_grad(0).defined(); }
bool has_tangent(const std::optional<Tensor>& t) { return t.has_value() && has_tangent(*t); }

// Gradients of a backward that cannot itself be differentiated: under
// create_graph they carry a node that says so.
tensor_list once(const char* name, tensor_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  tensor_list given;
  for (auto& g : grads)
    if (g.defined()) {
      Tensor t = g.detach();
      t.set_requires_grad(true);
      given.push_back(t);
    }
  if (given.empty()) return grads;
  const auto n = static_cast<int64_t>(given.size());
  auto node = std::make_shared<torch::autograd::DelayedError>(
      std::string(name) + " is differentiable once", n);
  given = (*node)(std::move(given));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = given[i++];
  return grads;
}

// rows [n, heads, d] that the kernels read where they are
Tensor packed_rows(const Tensor& t) {
  const int64_t es = t.element_size();
  if (t.size(0) == 0 ||
      (t.stride(2) == 1 && t.stride(1) == t.size(2) && t.stride(0) >= t.size(1) * t.size(2) &&
       t.stride(0) * es % 16 == 0 && t.stride(0) * es < (1 << 23) &&
       reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0))
    return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

const ngt_packed_windows* windows_of(const Tensor& bytes) {
  return reinterpret_cast<const ngt_packed_windows*>(bytes.data_ptr());
}

// the dtype of a call: the rows', and whether the table is fp32
int packed_type(const Tensor& q, const Tensor& table) {
  return dtype_code(q) |
         (table.defined() && table.scalar_type() == at::kFloat ? NGT_TABLE_F32 : 0);
}

struct PackedForward {
  Tensor out, out32, lse;
};

PackedForward packed_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table,
                             const Tensor& win, const Tensor& by_query, double scale,
                             bool want_grad) {
  const int64_t n_q = q.size(0), H = q.size(1), d = q.size(2);
  const auto f32 = q.options().dtype(at::kFloat);
  PackedForward r;
  r.out = at::empty({n_q, H, d}, q.options());
  if (want_grad) {
    r.out32 = q.scalar_type() == at::kFloat ? r.out : at::empty({n_q, H, d}, f32);
    r.lse = at::empty({table.defined() ? 2 * H : H, n_q}, f32);
  }
  const int dt = packed_type(q, table);
  const auto h = static_cast<int32_t>(H), hkv = static_cast<int32_t>(k.size(1));
  size_t bytes = 0;
  check(g_packed_ws(dt, windows_of(win), h, hkv, static_cast<int32_t>(d), 0, &bytes, nullptr));
  const Tensor ws = bytes ? workspace(static_cast<int64_t>(bytes), q) : Tensor();
  check(g_packed_fwd(dt, q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), k.stride(0),
                     v.stride(0), windows_of(win), h, hkv, static_cast<int32_t>(d),
                     static_cast<float>(scale), table.defined() ? table.data_ptr() : nullptr,
                     table.defined() ? static_cast<int32_t>(table.size(0)) : 0,
                     table.defined() ? by_query.data_ptr<uint8_t>() : nullptr, r.out.data_ptr(),
                     want_grad && !r.out32.is_same(r.out) ? r.out32.data_ptr<float>() : nullptr,
                     want_grad ? r.lse.data_ptr<float>() : nullptr,
                     bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q)));
  return r;
}

struct PackedAttention : public torch::autograd::Function<PackedAttention> {
  static Tensor forward(AutogradContext* ctx, Tensor q, Tensor k, Tensor v,
                        std::optional<Tensor> table_opt, Tensor win, Tensor win_mem,
                        std::optional<Tensor> by_query, std::optional<Tensor> by_key,
                        double scale) {
    q = packed_rows(q), k = packed_rows(k), v = packed_rows(v);
    const Tensor table = table_opt.has_value() ? table_opt->contiguous() : Tensor();
    const Tensor bq = by_query.value_or(Tensor()), bk = by_key.value_or(Tensor());
    const auto r = packed_forward(q, k, v, table, win, bq, scale, true);
    ctx->save_for_backward({q, k, v, table, r.out32, r.lse});
    ctx->saved_data["win"] = win;
    ctx->saved_data["win_mem"] = win_mem;
    ctx->saved_data["by_query"] = bq;
    ctx->saved_data["by_key"] = bk;
    ctx->saved_data["scale"] = scale;
    return r.out;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &table = saved[3], &out32 = saved[4],
                 &lse = saved[5];
    const at::DeviceGuard guard(q.device());
    const Tensor win = ctx->saved_data["win"].toTensor();
    const bool bias = table.defined();
    const Tensor bq = ctx->saved_data["by_query"].toTensor();
    const Tensor bk = ctx->saved_data["by_key"].toTensor();
    const int64_t H = q.size(1), d = q.size(2);
    const Tensor g = rows16(grads[0].to(q.scalar_type()));
    tensor_list res(9);
    res[0] = at::empty(q.sizes(), q.options());
    res[1] = at::empty(k.sizes(), k.options());
    res[2] = at::empty(v.sizes(), v.options());
    const bool want_table = bias && ctx->needs_input_grad(3);
    if (want_table) res[3] = at::empty_like(table);
    const int dt = packed_type(q, table);
    const auto h = static_cast<int32_t>(H), hkv = static_cast<int32_t>(k.size(1)),
               nb = bias ? static_cast<int32_t>(table.size(0)) : 0;
    size_t bytes = 0;
    check(g_packed_ws(dt, windows_of(win), h, hkv, static_cast<int32_t>(d), want_table ? nb : 0,
                      nullptr, &bytes));
    const Tensor ws = workspace(static_cast<int64_t>(bytes), q);
    check(g_packed_bwd(dt, q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), k.stride(0),
                       v.stride(0), out32.data_ptr<float>(), g.data_ptr(), lse.data_ptr<float>(),
                       windows_of(win), h, hkv, static_cast<int32_t>(d),
                       static_cast<float>(ctx->saved_data["scale"].toDouble()),
                       bias ? table.data_ptr() : nullptr, nb,
                       bias ? bq.data_ptr<uint8_t>() : nullptr,
                       bias ? bk.data_ptr<uint8_t>() : nullptr, res[0].data_ptr(),
                       res[1].data_ptr(), res[2].data_ptr(),
                       want_table ? res[3].data_ptr() : nullptr, ws.data_ptr(), bytes,
                       stream_of(q)));
    return once("packed_attention", res);
  }
};

// The checks of packed.py's packed_attention, without their messages: nothing
// where one of them fails.
std::optional<Tensor> packed_attention(const Tensor& q, const Tensor& k, const Tensor& v,
                                       const std::optional<Tensor>& table, const Tensor& win,
                                       const Tensor& win_mem,
                                       const std::optional<Tensor>& by_query,
                                       const std::optional<Tensor>& by_key, double scale) {
  const ngt_packed_windows* w = windows_of(win);
  if (q.dim() != 3 || k.dim() != 3 || v.dim() != 3) return std::nullopt;
  const int64_t H = q.size(1), hkv = k.size(1), d = q.size(2);
  const auto type = q.scalar_type();
  if (q.size(0) != w->n_q || k.size(0) != w->n_k || k.sizes() != v.sizes() || k.size(2) != d ||
      H < 1 || hkv < 1 || H % hkv || d < 8 || d > 128 || d % 8 ||
      (type != at::kFloat && type != at::kBFloat16) || k.scalar_type() != type ||
      v.scalar_type() != type || q.device() != win_mem.device() ||
      k.device() != win_mem.device() || v.device() != win_mem.device() || !(scale >= 0x1p-100) ||
      !(scale <= 0x1p100) || !q.has_storage() || !k.has_storage() || !v.has_storage())
    return std::nullopt;
  if (table.has_value() != by_query.has_value()) return std::nullopt;
  if (has_tangent(q) || has_tangent(k) || has_tangent(v) || has_tangent(table))
    return std::nullopt;
  if (table.has_value() &&
      (table->dim() != 2 || table->size(1) != H || table->size(0) < 1 || table->size(0) > 255 ||
       (table->scalar_type() != type && table->scalar_type() != at::kFloat) ||
       table->device() != q.device()))
    return std::nullopt;
  const at::DeviceGuard guard(q.device());
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() ||
                                     (table.has_value() && table->requires_grad())))
    return PackedAttention::apply(q, k, v, table, win, win_mem, by_query, by_key, scale);
  return packed_forward(packed_rows(q), packed_rows(k), packed_rows(v),
                        table.has_value() ? table->contiguous() : Tensor(), win,
                        by_query.value_or(Tensor()), scale, false)
      .out;
}

// ------------------------------------------------------ linear with epilogue
struct EpilogueForward {
  Tensor x2, w16, y, z;
};

EpilogueForward epilogue_forward(const Tensor& x, const Tensor& weight,
                                 const std::optional<Tensor>& bias,
                                 const std::optional<Tensor>& residual, int64_t act,
                                 bool want_grad) {
  NoAutocast off;
  const int64_t n_out = weight.size(0), n_in = weight.size(1);
  EpilogueForward r;
  r.x2 = bf16(x).reshape({-1, n_in});
  const int64_t m = r.x2.size(0);
  if ((n_in > 1 && r.x2.stride(1) != 1) || (m > 1 && r.x2.stride(0) < n_in))
    r.x2 = r.x2.clone(at::MemoryFormat::Contiguous);
  r.w16 = bf16(weight).contiguous();
  const Tensor b = bias.has_value() ? bf16(*bias).contiguous() : Tensor();
  const Tensor res =
      residual.has_value() ? bf16(*residual).reshape({-1, n_out}).contiguous() : Tensor();
  auto shape = x.sizes().vec();
  shape.back() = n_out;
  r.y = at::empty(shape, r.x2.options());
  if (want_grad && act) r.z = at::empty({m, n_out}, r.x2.options());
  check(g_linear_fwd(r.x2.data_ptr(), m > 1 ? r.x2.stride(0) : n_in, r.w16.data_ptr(),
                     b.defined() ? b.data_ptr() : nullptr,
                     res.defined() ? res.data_ptr() : nullptr, m, static_cast<int32_t>(n_out),
                     static_cast<int32_t>(n_in), static_cast<int32_t>(act), r.y.data_ptr(),
                     r.z.defined() ? r.z.data_ptr() : nullptr, stream_of(x)));
  return r;
}

struct LinearEpilogue : public torch::autograd::Function<LinearEpilogue> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor weight, std::optional<Tensor> bias,
                        std::optional<Tensor> residual, int64_t act) {
    const auto r = epilogue_forward(x, weight, bias, residual, act, true);
    ctx->save_for_backward({r.x2, r.w16, r.z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["x_type"] = x.scalar_type();
    ctx->saved_data["w_type"] = weight.scalar_type();
    ctx->saved_data["b_type"] =
        static_cast<int64_t>(bias.has_value() ? static_cast<int>(bias->scalar_type()) : -1);
    ctx->saved_data["r_type"] =
        static_cast<int64_t>(residual.has_value() ? static_cast<int>(residual->scalar_type()) : -1);
    ctx->saved_data["shape"] = x.sizes().vec();
    return r.y;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    NoAutocast off;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x2 = saved[0], &w16 = saved[1], &z = saved[2];
    const at::DeviceGuard guard(x2.device());
    const int64_t m = x2.size(0), n_in = x2.size(1), n_out = w16.size(0);
    const int64_t act = ctx->saved_data["act"].toInt();
    const int64_t b_type = ctx->saved_data["b_type"].toInt();
    const int64_t r_type = ctx->saved_data["r_type"].toInt();
    // the node's edges are numbered over the tensors that were given
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
    const bool want_b = b_type >= 0 && ctx->needs_input_grad(2);
    const bool want_r = r_type >= 0 && ctx->needs_input_grad(b_type >= 0 ? 3 : 2);
    const Tensor g = rows16(bf16(grads[0]));
    tensor_list res(5);
    Tensor dx, dz = g.view({m, n_out});
    if (want_x || want_w || want_b) {
      const Tensor gz = dz;
      if (act) dz = at::empty({m, n_out}, g.options());
      if (want_x) dx = at::empty({m, n_in}, g.options());
      size_t bytes = 0;
      check(g_linear_bwd_ws(m, static_cast<int32_t>(n_out), static_cast<int32_t>(n_in), &bytes));
      const Tensor ws = want_x ? workspace(static_cast<int64_t>(bytes), g) : Tensor();
      check(g_linear_bwd(gz.data_ptr(), z.defined() ? z.data_ptr() : nullptr, w16.data_ptr(), m,
                         static_cast<int32_t>(n_out), static_cast<int32_t>(n_in),
                         static_cast<int32_t>(act), dz.data_ptr(),
                         want_x ? dx.data_ptr() : nullptr, want_x ? ws.data_ptr() : nullptr, bytes,
                         stream_of(x2)));
    }
    if (want_x)
      res[0] = dx.view(ctx->saved_data["shape"].toIntVector())
                   .to(ctx->saved_data["x_type"].toScalarType());
    if (want_w) {
      const Tensor xc = x2.contiguous();
      const auto opt = x2.options().dtype(at::kFloat);
      Tensor dw = at::empty({n_out, n_in}, opt), db = want_b ? at::empty({n_out}, opt) : Tensor();
      size_t bytes = 0;
      check(g_wgrad_ws(m, static_cast<int32_t>(n_out), static_cast<int32_t>(n_in), &bytes));
      const Tensor ws = workspace(static_cast<int64_t>(bytes), x2);
      check(g_wgrad(xc.data_ptr(), dz.data_ptr(), m, static_cast<int32_t>(n_out),
                    static_cast<int32_t>(n_in), dw.data_ptr<float>(),
                    want_b ? db.data_ptr<float>() : nullptr, ws.data_ptr(), bytes, stream_of(x2)));
      res[1] = dw.to(ctx->saved_data["w_type"].toScalarType());
      if (want_b) res[2] = db;
    } else if (want_b) {
      res[2] = colsum(dz);
    }
    if (want_b) res[2] = res[2].to(static_cast<at::ScalarType>(b_type));
    if (want_r) res[3] = grads[0].to(static_cast<at::ScalarType>(r_type));
    return once("linear_epilogue", res);
  }
};

bool linear_type(const Tensor& t, const Tensor& x) {
  return (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat) &&
         t.device() == x.device() && t.has_storage();
}

// The checks of linear.py's linear_epilogue, without their messages: nothing
// where one of them fails.
std::optional<Tensor> linear_epilogue(const Tensor& x, const Tensor& weight,
                                      const std::optional<Tensor>& bias,
                                      const std::optional<Tensor>& residual, int64_t act) {
  if (!x.is_cuda() || !linear_type(x, x) || !linear_type(weight, x) || weight.dim() != 2 ||
      x.dim() < 1 || x.size(-1) != weight.size(1) || weight.numel() == 0)
    return std::nullopt;
  if (bias.has_value() &&
      (!linear_type(*bias, x) || bias->dim() != 1 || bias->size(0) != weight.size(0)))
    return std::nullopt;
  if (residual.has_value() &&
      (!linear_type(*residual, x) || residual->dim() != x.dim() ||
       residual->size(-1) != weight.size(0) ||
       residual->sizes().slice(0, x.dim() - 1) != x.sizes().slice(0, x.dim() - 1)))
    return std::nullopt;
  if (has_tangent(x) || has_tangent(weight) || has_tangent(bias) || has_tangent(residual))
    return std::nullopt;
  const at::DeviceGuard guard(x.device());
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || weight.requires_grad() || (bias.has_value() && bias->requires_grad()) ||
       (residual.has_value() && residual->requires_grad())))
    return LinearEpilogue::apply(x, weight, bias, residual, act);
  return epilogue_forward(x, weight, bias, residual, act, false).y;
}

// --------------------------------------------------------------- gated linear
struct GatedForward {
  Tensor x2, wg, wu, y, keep;
};

GatedForward gated_forward(const Tensor& x, const Tensor& w_gate, const Tensor& w_up,
                           const std::optional<Tensor>& b_gate, const std::optional<Tensor>& b_up,
                           int64_t act, bool want_grad) {
  NoAutocast off;
  const int64_t n_out = w_gate.size(0), n_in = w_gate.size(1);
  GatedForward r;
  r.x2 = bf16(x).reshape({-1, n_in});
  const int64_t m = r.x2.size(0);
  if ((n_in > 1 && r.x2.stride(1) != 1) || (m > 1 && r.x2.stride(0) < n_in))
    r.x2 = r.x2.clone(at::MemoryFormat::Contiguous);
  r.wg = bf16(w_gate).contiguous(), r.wu = bf16(w_up).contiguous();
  const Tensor bg = b_gate.has_value() ? bf16(*b_gate).contiguous() : Tensor();
  const Tensor bu = b_up.has_value() ? bf16(*b_up).contiguous() : Tensor();
  auto shape = x.sizes().vec();
  shape.back() = n_out;
  r.y = at::empty(shape, r.x2.options());
  if (want_grad) {
    size_t bytes = 0;
    check(g_gated_keep(m, static_cast<int32_t>(n_out), &bytes));
    r.keep = workspace(static_cast<int64_t>(bytes), r.x2);
  }
  const auto n = static_cast<int32_t>(n_out), k = static_cast<int32_t>(n_in);
  size_t bytes = 0;
  check(g_gated_fwd_ws(m, n, k, &bytes));
  const Tensor ws = bytes ? workspace(static_cast<int64_t>(bytes), r.x2) : Tensor();
  check(g_gated_fwd(r.x2.data_ptr(), m > 1 ? r.x2.stride(0) : n_in, r.wg.data_ptr(),
                    r.wu.data_ptr(), bg.defined() ? bg.data_ptr() : nullptr,
                    bu.defined() ? bu.data_ptr() : nullptr, m, n, k,
                    static_cast<int32_t>(act), r.y.data_ptr(),
                    want_grad ? r.keep.data_ptr() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes,
                    stream_of(x)));
  return r;
}

int64_t type_of(const std::optional<Tensor>& t) {
  return t.has_value() ? static_cast<int64_t>(t->scalar_type()) : -1;
}

struct GatedLinear : public torch::autograd::Function<GatedLinear> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor w_gate, Tensor w_up,
                        std::optional<Tensor> b_gate, std::optional<Tensor> b_up, int64_t act) {
    const auto r = gated_forward(x, w_gate, w_up, b_gate, b_up, act, true);
    ctx->save_for_backward({r.x2, r.wg, r.wu, r.keep});
    ctx->saved_data["types"] = std::vector<int64_t>{
        type_of(x), type_of(w_gate), type_of(w_up), type_of(b_gate), type_of(b_up)};
    ctx->saved_data["shape"] = x.sizes().vec();
    return r.y;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    NoAutocast off;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x2 = saved[0], &keep = saved[3];
    const at::DeviceGuard guard(x2.device());
    const Tensor wg = rows16(saved[1]), wu = rows16(saved[2]);
    const int64_t m = x2.size(0), n_in = x2.size(1), n_out = wg.size(0);
    const auto types = ctx->saved_data["types"].toIntVector();
    // the node's edges are numbered over the tensors that were given
    bool want[5];
    for (int i = 0, edge = 0; i < 5; ++i)
      want[i] = types[i] >= 0 && ctx->needs_input_grad(static_cast<size_t>(edge++));
    const auto n = static_cast<int32_t>(n_out), k = static_cast<int32_t>(n_in);
    const Tensor g = rows16(bf16(grads[0])), xc = rows16(x2);
    auto type = [&](int i) { return static_cast<at::ScalarType>(types[i]); };
    tensor_list res(6);
    ngt_gated_grads out{};
    if (want[0]) res[0] = at::empty({m, n_in}, g.options());
    for (int i = 1; i < 5; ++i)
      if (want[i])
        res[i] = i < 3 ? at::empty({n_out, n_in}, g.options().dtype(type(i)))
                       : at::empty({n_out}, g.options().dtype(type(i)));
    auto at_of = [&](int i) { return want[i] ? res[i].data_ptr() : nullptr; };
    auto code = [&](int i) { return want[i] ? dtype_code(res[i]) : NGT_F32; };
    out.dx = at_of(0), out.dw_gate = at_of(1), out.dw_up = at_of(2);
    out.db_gate = at_of(3), out.db_up = at_of(4);
    out.dw_gate_dtype = code(1), out.dw_up_dtype = code(2);
    out.db_gate_dtype = code(3), out.db_up_dtype = code(4);
    size_t bytes = 0;
    check(g_gated_bwd_ws(m, n, k, &bytes));
    const Tensor ws = workspace(static_cast<int64_t>(bytes), g);
    check(g_gated_bwd(g.data_ptr(), keep.data_ptr(), xc.data_ptr(), wg.data_ptr(), wu.data_ptr(), m,
                      n, k, &out, ws.data_ptr(), bytes, stream_of(x2)));
    if (want[0]) res[0] = res[0].view(ctx->saved_data["shape"].toIntVector()).to(type(0));
    return once("gated_linear", res);
  }
};

// The checks of linear.py's gated_linear, without their messages: nothing where one
// of them fails.
std::optional<Tensor> gated_linear(const Tensor& x, const Tensor& w_gate, const Tensor& w_up,
                                   const std::optional<Tensor>& b_gate,
                                   const std::optional<Tensor>& b_up, int64_t act) {
  if (!x.is_cuda() || !linear_type(x, x) || !linear_type(w_gate, x) || !linear_type(w_up, x) ||
      w_gate.dim() != 2 || w_up.sizes() != w_gate.sizes() || x.dim() < 1 ||
      x.size(-1) != w_gate.size(1) || w_gate.numel() == 0)
    return std::nullopt;
  bool grad = x.requires_grad() || w_gate.requires_grad() || w_up.requires_grad();
  for (const auto* b : {&b_gate, &b_up}) {
    if (!b->has_value()) continue;
    if (!linear_type(**b, x) || (*b)->dim() != 1 || (*b)->size(0) != w_gate.size(0))
      return std::nullopt;
    grad = grad || (*b)->requires_grad();
  }
  if (has_tangent(x) || has_tangent(w_gate) || has_tangent(w_up) || has_tangent(b_gate) ||
      has_tangent(b_up))
    return std::nullopt;
  const at::DeviceGuard guard(x.device());
  if (at::GradMode::is_enabled() && grad)
    return GatedLinear::apply(x, w_gate, w_up, b_gate, b_up, act);
  return gated_forward(x, w_gate, w_up, b_gate, b_up, act, false).y;
}

// -------------------------------------------------------- norm and rotation
// heads [..., H, d] as rows [n, H, d] that the kernels read where they are
Tensor head_rows(const Tensor& t) {
  const Tensor r = t.dim() == 3 ? t : t.reshape({-1, t.size(-2), t.size(-1)});
  if (r.numel() && r.stride(2) != 1) return r.contiguous();
  return r;
}

ngt_head_rows head_struct(const Tensor& x, const Tensor& gain) {
  ngt_head_rows r{};
  r.x = x.data_ptr();
  r.x_row = x.stride(0), r.x_head = x.stride(1);
  r.n_heads = static_cast<int32_t>(x.size(1));
  if (gain.defined()) r.gain = gain.data_ptr(), r.gain_dtype = dtype_code(gain);
  return r;
}

struct Turns {
  Tensor positions, turns;
  bool interleaved;
  double magnitude;
  ngt_rotation rotation() const {
    ngt_rotation r{};
    if (!turns.defined()) return r;
    r.positions = positions.data_ptr();
    r.turns = turns.data_ptr<double>();
    r.position_bytes = static_cast<int32_t>(positions.element_size());
    r.dim = static_cast<int32_t>(2 * turns.numel());
    r.interleaved = interleaved;
    r.magnitude = static_cast<float>(magnitude);
    return r;
  }
};

tensor_list rotary_forward(const Tensor& q, const Tensor& k, const Tensor& q_gain,
                           const Tensor& k_gain, const Turns& t, double eps) {
  auto hq = head_struct(q, q_gain), hk = k.defined() ? head_struct(k, k_gain) : ngt_head_rows{};
  tensor_list y{at::empty(q.sizes(), q.options()), k.defined() ? at::empty(k.sizes(), k.options()) : Tensor()};
  hq.y = y[0].data_ptr();
  if (k.defined()) hk.y = y[1].data_ptr();
  const auto rot = t.rotation();
  check(g_rotary_fwd(dtype_code(q), &hq, k.defined() ? &hk : nullptr, q.size(0),
                     static_cast<int32_t>(q.size(2)), &rot, static_cast<float>(eps),
                     stream_of(q)));
  return y;
}

struct NormRotary : public torch::autograd::Function<NormRotary> {
  // q [.., H, d], k [.., H_kv, d]; the results have their shapes
  static tensor_list forward(AutogradContext* ctx, Tensor q, std::optional<Tensor> k,
                             std::optional<Tensor> q_gain, std::optional<Tensor> k_gain,
                             std::optional<Tensor> positions_opt, std::optional<Tensor> turns_opt,
                             bool interleaved, double magnitude, double eps) {
    const Tensor positions = positions_opt.value_or(Tensor()), turns = turns_opt.value_or(Tensor());
    const Tensor q3 = head_rows(q), k3 = k.has_value() ? head_rows(*k) : Tensor();
    const Tensor gq = q_gain.has_value() ? q_gain->contiguous() : Tensor();
    const Tensor gk = k_gain.has_value() ? k_gain->contiguous() : Tensor();
    const auto y = rotary_forward(q3, k3, gq, gk, {positions, turns, interleaved, magnitude}, eps);
    // (without a gain the backward does not need the input)
    ctx->save_for_backward({gq.defined() ? q3 : Tensor(), gk.defined() ? k3 : Tensor(), gq, gk,
                            positions, turns});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["q_shape"] = q.sizes().vec();
    tensor_list out{y[0].view(q.sizes())};
    if (k.has_value()) {
      ctx->saved_data["k_shape"] = k->sizes().vec();
      out.push_back(y[1].view(k->sizes()));
    }
    return out;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q_gain = saved[2], &k_gain = saved[3];
    const at::DeviceGuard guard(grads[0].device());
    const bool has_k = ctx->saved_data.count("k_shape") > 0;
    // the node's edges are numbered over the tensors that were given
    size_t edge = 0;
    tensor_list res(9);
    auto heads = [&](int i, const char* shape) {
      const auto s = ctx->saved_data[shape].toIntVector();
      if (ctx->needs_input_grad(edge++)) res[i] = at::empty(s, grads[i].options());
    };
    heads(0, "q_shape");
    if (has_k) heads(1, "k_shape");
    for (int i = 2; i < 4; ++i)
      if (saved[i].defined() && ctx->needs_input_grad(edge++))
        res[i] = at::empty(saved[i].sizes(), saved[i].options());
    const Tensor gq = head_rows(grads[0]), gk = has_k ? head_rows(grads[1]) : Tensor();
    auto fill = [](const Tensor& dy, const Tensor& x, const Tensor& gain, const Tensor& dx,
                   const Tensor& dgain) {
      auto h = gain.defined() ? head_struct(x, gain) : ngt_head_rows{};
      h.n_heads = static_cast<int32_t>(dy.size(1));
      h.dy = dy.data_ptr(), h.dy_row = dy.stride(0), h.dy_head = dy.stride(1);
      if (dx.defined()) h.y = dx.data_ptr();
      if (dgain.defined()) h.dgain = dgain.data_ptr();
      return h;
    };
    const auto hq = fill(gq, saved[0], q_gain, res[0], res[2]);
    const auto hk = has_k ? fill(gk, saved[1], k_gain, res[1], res[3]) : ngt_head_rows{};
    const int64_t n = gq.size(0);
    const auto d = static_cast<int32_t>(gq.size(2));
    size_t bytes = 0;
    if (res[2].defined() || res[3].defined()) check(g_rotary_bwd_ws(n, d, &bytes));
    const Tensor ws = bytes ? workspace(static_cast<int64_t>(bytes), gq) : Tensor();
    const auto rot = Turns{saved[4], saved[5], ctx->saved_data["interleaved"].toBool(),
                           ctx->saved_data["magnitude"].toDouble()}
                         .rotation();
    check(g_rotary_bwd(dtype_code(gq), &hq, has_k ? &hk : nullptr, n, d, &rot,
                       static_cast<float>(ctx->saved_data["eps"].toDouble()),
                       bytes ? ws.data_ptr() : nullptr, bytes, stream_of(gq)));
    return once("norm_rotary", res);
  }
};

// The checks of rotary.py's norm_rotary, without their messages: nothing where one of
// them fails.
std::optional<tensor_list> norm_rotary(const Tensor& q, const std::optional<Tensor>& k,
                                       const std::optional<Tensor>& q_gain,
                                       const std::optional<Tensor>& k_gain,
                                       const std::optional<Tensor>& positions,
                                       const std::optional<Tensor>& turns, bool interleaved,
                                       double magnitude, double eps) {
  if (!q.is_cuda() || q.dim() < 2 || !q.has_storage()) return std::nullopt;
  const int64_t d = q.size(-1), lead = q.dim() - 2;
  const auto type = q.scalar_type();
  if ((type != at::kFloat && type != at::kBFloat16) || d < 2 || d > 256 || d % 2 ||
      q.size(-2) < 1 || !(eps >= 0) || !(eps < INFINITY) || turns.has_value() != positions.has_value())
    return std::nullopt;
  bool grad = q.requires_grad();
  if (k.has_value()) {
    if (k->dim() != q.dim() || k->size(-1) != d || k->size(-2) < 1 || k->scalar_type() != type ||
        k->device() != q.device() || !k->has_storage() ||
        k->sizes().slice(0, lead) != q.sizes().slice(0, lead))
      return std::nullopt;
    grad = grad || k->requires_grad();
  } else if (k_gain.has_value()) {
    return std::nullopt;
  }
  for (const auto* g : {&q_gain, &k_gain}) {
    if (!g->has_value()) continue;
    const auto gt = (*g)->scalar_type();
    if ((*g)->dim() != 1 || (*g)->size(0) != d || (*g)->device() != q.device() ||
        (gt != type && gt != at::kFloat) || !(*g)->has_storage())
      return std::nullopt;
    grad = grad || (*g)->requires_grad();
  }
  std::optional<Tensor> pos;
  if (turns.has_value()) {
    const auto pt = positions->scalar_type();
    if (turns->device() != q.device() || 2 * turns->numel() > d ||
        positions->device() != q.device() || (pt != at::kInt && pt != at::kLong) ||
        positions->sizes() != q.sizes().slice(0, lead) || !positions->has_storage())
      return std::nullopt;
    pos = positions->reshape({-1}).contiguous();
  }
  if (has_tangent(q) || has_tangent(k) || has_tangent(q_gain) || has_tangent(k_gain))
    return std::nullopt;
  const at::DeviceGuard guard(q.device());
  if (at::GradMode::is_enabled() && grad)
    return NormRotary::apply(q, k, q_gain, k_gain, pos, turns, interleaved, magnitude, eps);
  auto y = rotary_forward(head_rows(q), k.has_value() ? head_rows(*k) : Tensor(),
                          q_gain.has_value() ? q_gain->contiguous() : Tensor(),
                          k_gain.has_value() ? k_gain->contiguous() : Tensor(),
                          {pos.value_or(Tensor()), turns.value_or(Tensor()), interleaved, magnitude},
                          eps);
  y[0] = y[0].view(q.sizes());
  if (k.has_value()) y[1] = y[1].view(k->sizes());
  else y.pop_back();
  return y;
}

// ------------------------------------------------------------------ clipping
bool clip_type(const Tensor& t, const Tensor& like) {
  return t.layout() == at::kStrided && t.device() == like.device() && t.has_storage() &&
         (t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16) &&
         (t.numel() == 0 || t.is_non_overlapping_and_dense());
}

// gradients.py's call: the norm, or nothing where one of its checks fails.
std::optional<Tensor> clip_gradients(const std::vector<Tensor>& parameters,
                                     const std::optional<std::vector<Tensor>>& out,
                                     double max_norm) {
  std::vector<Tensor> grads;
  grads.reserve(parameters.size());
  std::unordered_set<const void*> seen;
  for (const Tensor& p : parameters)
    if (p.grad().defined() && seen.insert(p.unsafeGetTensorImpl()).second) grads.push_back(p.grad());
  if (grads.empty() || !grads[0].is_cuda() || (out.has_value() && out->size() != grads.size()))
    return std::nullopt;
  const size_t n = grads.size();
  std::vector<ngt_gradient> table(n);
  struct Run {
    uintptr_t from, to;
    size_t tensor;
    bool result;
  };
  std::vector<Run> runs;
  runs.reserve(out.has_value() ? 2 * n : n);
  auto add = [&](const Tensor& t, size_t i, bool result) {
    const auto at = reinterpret_cast<uintptr_t>(t.data_ptr());
    if (t.numel()) runs.push_back({at, at + t.numel() * t.element_size(), i, result});
  };
  for (size_t i = 0; i < n; ++i) {
    const Tensor& g = grads[i];
    if (!clip_type(g, grads[0])) return std::nullopt;
    table[i] = {g.data_ptr(), nullptr, g.numel(), dtype_code(g), 0};
    add(g, i, false);
    if (!out.has_value()) continue;
    const Tensor& o = (*out)[i];
    if (!clip_type(o, grads[0]) || o.sizes() != g.sizes()) return std::nullopt;
    for (int64_t a = 0; g.numel() && a < g.dim(); ++a)
      if (g.size(a) != 1 && g.stride(a) != o.stride(a)) return std::nullopt;
    table[i].out = o.data_ptr(), table[i].out_dtype = dtype_code(o);
    add(o, i, true);
  }
  if (max_norm >= 0) {
    // a result may lie in its own gradient's memory, nothing else may overlap
    std::sort(runs.begin(), runs.end(), [](const Run& a, const Run& b) {
      return a.from != b.from ? a.from < b.from : a.tensor != b.tensor ? a.tensor < b.tensor
                                                                       : a.result < b.result;
    });
    for (size_t i = 1, last = 0; i < runs.size(); ++i) {
      const Run &a = runs[last], &b = runs[i];
      if (b.from < a.to && !(a.tensor == b.tensor && a.from == b.from && a.to == b.to))
        return std::nullopt;
      if (b.to > a.to) last = i;
    }
  }
  const at::DeviceGuard guard(grads[0].device());
  size_t bytes = 0;
  check(g_clip_ws(table.data(), static_cast<int32_t>(n), &bytes));
  const Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
  const Tensor ws = workspace(static_cast<int64_t>(bytes), norm);
  check(g_clip(table.data(), static_cast<int32_t>(n), max_norm, norm.data_ptr<float>(),
               ws.data_ptr(), bytes, stream_of(norm)));
  if (max_norm >= 0)
    for (const Tensor& t : out.has_value() ? *out : grads)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return norm;
}

template <typename F>
void entry(F*& fn, const std::map<std::string, int64_t>& addr, const char* name) {
  const auto it = addr.find(name);
  TORCH_CHECK(it != addr.end() && it->second, "ngt_autograd.init: no address of ", name);
  fn = reinterpret_cast<F*>(it->second);
}

void init(const std::map<std::string, int64_t>& addr) {
  entry(g_fwd, addr, "ngt_sparse_fwd_ext");
  entry(g_bwd, addr, "ngt_sparse_bwd_strided");
  entry(g_err, addr, "ngt_last_error");
  entry(g_colsum_ws, addr, "ngt_colsum_workspace_bytes");
  entry(g_colsum, addr, "ngt_colsum_bf16");
  entry(g_chunk_sum, addr, "ngt_chunk_sum_f32");
  entry(g_wgrad_ws, addr, "ngt_wgrad_workspace_bytes");
  entry(g_wgrad_pays, addr, "ngt_wgrad_pays");
  entry(g_wgrad, addr, "ngt_wgrad_bf16");
  entry(g_ln_fwd, addr, "ngt_layernorm_fwd");
  entry(g_ln_bwd_ws, addr, "ngt_layernorm_bwd_workspace_bytes");
  entry(g_ln_bwd, addr, "ngt_layernorm_bwd");
  entry(g_add_ln_fwd, addr, "ngt_add_layernorm_fwd");
  entry(g_add_ln_bwd, addr, "ngt_add_layernorm_bwd");
  entry(g_packed_ws, addr, "ngt_packed_workspace_bytes");
  entry(g_packed_fwd, addr, "ngt_packed_fwd");
  entry(g_packed_bwd, addr, "ngt_packed_bwd");
  entry(g_linear_fwd, addr, "ngt_linear_fwd");
  entry(g_linear_bwd_ws, addr, "ngt_linear_bwd_workspace_bytes");
  entry(g_linear_bwd, addr, "ngt_linear_bwd");
  entry(g_gated_keep, addr, "ngt_gated_keep_bytes");
  entry(g_gated_fwd_ws, addr, "ngt_gated_fwd_workspace_bytes");
  entry(g_gated_fwd, addr, "ngt_gated_fwd");
  entry(g_gated_bwd_ws, addr, "ngt_gated_bwd_workspace_bytes");
  entry(g_gated_bwd, addr, "ngt_gated_bwd");
  entry(g_rotary_fwd, addr, "ngt_norm_rotary_fwd");
  entry(g_rotary_bwd_ws, addr, "ngt_norm_rotary_bwd_workspace_bytes");
  entry(g_rotary_bwd, addr, "ngt_norm_rotary_bwd");
  entry(g_clip_ws, addr, "ngt_clip_workspace_bytes");
  entry(g_clip, addr, "ngt_clip_gradients");
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("init", &init, "{name: address} of libngt_attn.so's entry points");
  m.def("csr_struct_bytes", []() { return static_cast<int64_t>(sizeof(ngt_window_csr)); });
  m.def("abi_version", []() { return static_cast<int64_t>(NGT_ABI_VERSION); },
        "NGT_ABI_VERSION of the header this extension was compiled against");
  m.def("sparse_attention", &sparse_attention,
        "(q, k, v, k_ext, v_ext, csr, csr_mem, dst_end, scale, lo, hi, eps, fwd_bytes, "
        "bwd_bytes, interleave_grads) -> (out, node_scores); interleave_grads: dQ, dK, dV as "
        "views of one [N, 3, H, d] buffer (when q and k have the same rows)");
  m.def("linear", &linear, "(x, weight, bias) -> y: linear.py's _WgradLinearFn");
  m.def("project3", &project3,
        "(x, w0, b0, w1, b1, w2, b2, heads) -> [y0, y1, y2]: linear.py's _ProjectionGroupFn; "
        "heads > 0: outputs [..., heads, n_out / heads]");
  m.def("layernorm", &layernorm, "(x, weight, bias, eps, out_bf16) -> y: layernorm.py's _LayerNormFn");
  m.def("add_layernorm", &add_layernorm,
        "(x, y, weight, bias, eps, p, seed tensor or None, out_bf16) -> (s, out): layernorm.py's "
        "_AddLayerNormFn");
  m.def("packed_struct_bytes", []() { return static_cast<int64_t>(sizeof(ngt_packed_windows)); });
  m.def("packed_attention", &packed_attention,
        "(q, k, v, table, windows, windows_mem, by_query, by_key, scale) -> out or None: "
        "packed.py's PackedAttentionFunction; windows: the bytes of one ngt_packed_windows");
  m.def("linear_epilogue", &linear_epilogue,
        "(x, weight, bias, residual, activation) -> y or None: linear.py's LinearEpilogueFunction");
  m.def("gated_linear", &gated_linear,
        "(x, w_gate, w_up, b_gate, b_up, activation) -> y or None: linear.py's GatedLinearFunction");
  m.def("norm_rotary", &norm_rotary,
        "(q, k, q_gain, k_gain, positions, turns, interleaved, magnitude, eps) -> [q', k'] (or [q']) "
        "or None: rotary.py's NormRotaryFunction");
  m.def("clip_gradients", &clip_gradients,
        "(parameters, results or None, max_norm; negative: the norm alone) -> norm or None: "
        "gradients.py's call");
}
