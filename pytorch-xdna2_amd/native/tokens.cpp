// Host side of the token-model operators (xdna_train/tokens.py): checks, workspaces, C-ABI
// calls and autograd nodes of the embedding, the gated feed-forward, the distillation loss,
// the token log probabilities, layer norm, the linear layer and decay attention
// (csrc/embed.hip, gated.hip, vocab.hip, layer_norm.hip, decay.hip).  No call reads
// device data on the host, so all of them can be captured in a graph.
#include "xdna.h"

#include <torch/csrc/autograd/custom_function.h>

namespace xdna_backend {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool on_xdna(const at::Tensor& t) { return t.defined() && t.device().type() == kXdna; }

int float_code(const at::Tensor& t, const char* op, const char* what) {
  TORCH_CHECK(on_xdna(t), op, ": ", what, " must be an xdna tensor");
  TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, op, ": ", what,
              " must be float32 or bfloat16, got ", t.scalar_type());
  return t.scalar_type() == at::kFloat ? 1 : 2;
}

int index_bytes(const at::Tensor& t, const char* op, const char* what) {
  TORCH_CHECK(on_xdna(t), op, ": ", what, " must be an xdna tensor");
  TORCH_CHECK(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, op, ": ", what,
              " must be int64 or int32, got ", t.scalar_type());
  return t.scalar_type() == at::kLong ? 8 : 4;
}

void check_bf16(const at::Tensor& t, const char* op, const char* what) {
  TORCH_CHECK(on_xdna(t) && t.scalar_type() == at::kBFloat16, op, ": ", what, " must be a bfloat16 xdna tensor");
}

// [..., n] as [rows][n] with unit stride along n and a row stride of at least n (a copy only
// where the strides do not allow a view)
at::Tensor as_rows(const at::Tensor& t) {
  const int64_t n = t.size(-1);
  at::Tensor r = t.dim() == 2 ? t : t.reshape({n ? t.numel() / n : 0, n});
  if ((n > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < n)) r = r.contiguous();
  return r;
}

int64_t row_stride(const at::Tensor& rows) { return rows.size(0) > 1 ? rows.stride(0) : rows.size(1); }

at::Tensor workspace(size_t bytes) { return empty_xdna({int64_t(bytes)}, at::kByte); }

void* ptr_or_null(const at::Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
const void* cptr(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
const uint16_t* p16(const at::Tensor& t) { return static_cast<const uint16_t*>(t.const_data_ptr()); }
uint16_t* m16(at::Tensor& t) { return static_cast<uint16_t*>(t.data_ptr()); }
float* f32(at::Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }
const float* cf32(const at::Tensor& t) { return t.defined() ? static_cast<const float*>(t.const_data_ptr()) : nullptr; }

bool tracked(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t->requires_grad()) return true;
  return false;
}

// Raises where an operand carries a tangent (forward-mode differentiation, whatever the grad mode):
// the operators have no such rule, and a plain call would hand out a result without it.  (PyTorch
// opens one level at a time, 0.)
void no_tangents(const char* op, std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), op, ": forward-mode differentiation is not supported");
}

void once_only(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op, ": the gradient itself cannot be differentiated");
}

// whether the library's products load a matrix as whole vectors
bool vector_rows(const at::Tensor& t) {
  const int64_t ld = t.stride(1) == 1 ? t.stride(0) : t.stride(0) == 1 ? t.stride(1) : 1;
  return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0 && ld % 8 == 0;
}

// a b of two bf16 matrices, each contiguous along one dimension: on the framework's GEMM where its
// 256 x 256 tiles can load them and fill the CUs (or do with k split evenly) for long enough, else
// on the gated block's own tiles.  Measured (rows x columns x k, GEMM and own tiles in us): 8192 x
// 2048 x 4096 110 and 147, 4096 x 4096 x 1024 36 and 44, 8192 x 1024 x 8192 132 and 174; but 4800 x
// 4096 x 2048 (1.2 rounds of the CUs) 100 and 95, 8192 x 768 x 6144 (96 tiles) 121 and 105, 4096 x
// 1024 x 4096 55 and 46, 8192 x 1024 x 2048 51 and 42, 6424 x 896 x 1024 44 and 23.  Even splits begin
// where the two cross, in the mean of the three layouts (a w^T, a w, a^T b): 64 tiles 4096 x 1024 x 5120
// 60 58 58 and 52 55 57, x 6144 66 63 66 and 61 65 67, x 7168 71 69 72 and 70 74 77 (2048 x 2048 and
// 8192 x 512 the same); 128 tiles 8192 x 1024 x 3328 65 65 65 and 60 63 66, x 3840 71 71 71 and 69 72
// 75, x 5120 86 86 87 and 90 93 97 (4096 x 2048 the same).
bool on_gemm(const at::Tensor& a, const at::Tensor& b) {
  const int64_t K = a.size(1), tiles = ((a.size(0) + 255) / 256) * ((b.size(1) + 255) / 256);
  const bool fills = tiles >= 192 && 100 * tiles >= 65 * 256 * ((tiles + 255) / 256) && K * tiles >= 262144;
  const bool splits = (tiles == 64 && K >= 6144) || (tiles == 128 && K >= 3744);
  return vector_rows(a) && vector_rows(b) && K % 8 == 0 && K >= 1024 && (fills || splits);
}

at::Tensor product(const at::Tensor& a, const at::Tensor& b) {
  const int64_t M = a.size(0), K = a.size(1), N = b.size(1);
  at::Tensor c = empty_xdna({M, N}, at::kBFloat16);
  const bool b_rows = b.stride(1) == 1 && K > 1, a_rows = a.stride(0) == 1 && M > 1 && a.stride(1) != 1;
  const bool a_ok = a_rows ? b_rows : a.stride(1) == 1 || K == 1, b_ok = b_rows || b.stride(0) == 1 || K == 1;
  if (K > 0 && !on_gemm(a, b) && a_ok && b_ok && M <= int64_t(1) << 22) {
    const int64_t lda = a_rows ? a.stride(1) : M > 1 ? a.stride(0) : K, ldb = b_rows ? b.stride(0) : N > 1 ? b.stride(1) : K;
    check_abi(xdna_tile_mm_bf16(p16(b), ldb, b_rows ? 1 : 0, p16(a), lda, a_rows ? 1 : 0, N, M, K, m16(c), N,
                                current_stream()),
              "tile product");
    return c;
  }
  check_abi(xdna_gemm_bf16(p16(a), p16(b), m16(c), nullptr, 1, int(M), int(N), int(K), a.stride(0), a.stride(1), 0,
                           b.stride(0), b.stride(1), 0, N, 1, 0, 0, 0, 0, 1.0f, 0.0f, current_stream()),
            "gemm");
  return c;
}

// ---- embedding -------------------------------------------------------------------------------

at::Tensor embed_forward(const at::Tensor& ids, const at::Tensor& weight, double scale) {
  ScopedCount sc("hip_tokens.embed.fwd.run");
  const int ib = index_bytes(ids, "embed", "ids"), dt = float_code(weight, "embed", "weight");
  const at::Tensor i = ids.contiguous(), w = as_rows(weight);
  auto shape = ids.sizes().vec();
  shape.push_back(w.size(1));
  at::Tensor y = empty_xdna(shape, w.scalar_type());
  check_abi(xdna_embed(cptr(i), ib, i.numel(), cptr(w), dt, w.size(0), w.size(1), row_stride(w), float(scale),
                       ptr_or_null(y), current_stream()),
            "embed");
  return y;
}

struct EmbedFn : public torch::autograd::Function<EmbedFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& ids, const at::Tensor& weight, double scale,
                            int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->saved_data["dim"] = weight.size(1);
    return embed_forward(ids, weight, scale);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("embed");
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    ScopedCount sc("hip_tokens.embed.bwd.run");
    const at::Tensor ids = ctx->get_saved_variables()[0].contiguous();
    const int64_t V = ctx->saved_data["vocab"].toInt(), D = ctx->saved_data["dim"].toInt();
    const at::Tensor dy = as_rows(grads[0]);
    const size_t bytes = xdna_embed_bwd_workspace_bytes(ids.numel(), V, D);
    at::Tensor ws = workspace(bytes), dw = empty_xdna({V, D}, dy.scalar_type());
    check_abi(xdna_embed_bwd(cptr(ids), ids.scalar_type() == at::kLong ? 8 : 4, ids.numel(), cptr(dy),
                             float_code(dy, "embed", "the gradient"), row_stride(dy), V, D,
                             ctx->saved_data["padding"].toInt(), float(ctx->saved_data["scale"].toDouble()),
                             dw.data_ptr(), ptr_or_null(ws), bytes, current_stream()),
              "embed backward");
    return {at::Tensor(), dw, at::Tensor(), at::Tensor()};
  }
};

// ---- gated feed-forward --------------------------------------------------------------------------

struct GatedForward {
  at::Tensor x, w, h, gu;  // x and w as rows
};

GatedForward gated_forward(const at::Tensor& x, const at::Tensor& w_in, int64_t act, bool keep) {
  GatedForward r;
  r.x = as_rows(x);
  r.w = as_rows(w_in);
  const int64_t M = r.x.size(0), K = r.x.size(1), F = r.w.size(0) / 2;
  r.h = empty_xdna({M, F}, at::kBFloat16);
  if (keep) r.gu = empty_xdna({int64_t(xdna_gated_kept_bytes(M, F))}, at::kByte);
  check_abi(xdna_gated_bf16(p16(r.x), row_stride(r.x), p16(r.w), row_stride(r.w), M, K, F, int(act), m16(r.h),
                            keep ? ptr_or_null(r.gu) : nullptr, current_stream()),
            "gated");
  return r;
}

at::Tensor gated_dgu(const at::Tensor& dh, const at::Tensor& gu, int64_t act) {
  const at::Tensor d = as_rows(dh);
  const int64_t M = d.size(0), F = d.size(1);
  at::Tensor dgu = empty_xdna({M, 2 * F}, at::kBFloat16);
  check_abi(xdna_gated_bwd_bf16(p16(d), row_stride(d), cptr(gu), M, F, int(act), m16(dgu), current_stream()),
            "gated backward");
  return dgu;
}

// The gradients that follow dgu, of all inputs: one launch where that is faster, else one each.
struct GatedGrads {
  at::Tensor dx, dw_in, dw_out;
};

// Whether one launch is faster than products of which some run on the GEMM: while the block is short,
// the launch's tiles of one product fill the CUs that another leaves.  Measured, rows x K x F with N =
// K, one launch and apart in us: 6000 x 1024 x 4096 294 and 319, 7000 344 and 335; 12288 x 1024 x 2048
// 326 and 337, 16384 447 and 355; 16384 x 1024 x 1024 228 and 237; 10000 x 512 x 4096 281 and 301,
// 16384 448 and 391.  Without dw_out, whose few tiles gain most: 7000 x 1024 x 2048 142 and 148, 12288
// 241 and 237; 3500 x 1024 x 4096 143 and 166, 4096 186 and 154; 7000 x 512 x 4096 141 and 164, 10000
// 238 and 216.
bool short_block(int64_t M, int64_t K, int64_t F, int64_t N) {
  return double(M) * double(F) * double(4 * K + N) <= (N ? 129e9 : 64e9);
}

GatedGrads gated_grads(const at::Tensor& dgu, const at::Tensor& x, const at::Tensor& w, const at::Tensor& dy,
                       const at::Tensor& h) {
  const int64_t M = x.size(0), K = x.size(1), F = dgu.size(1) / 2, N = dy.defined() ? dy.size(1) : 0;
  GatedGrads r;
  const auto apart = [&] { return on_gemm(dgu, w) || on_gemm(dgu.t(), x) || (N && on_gemm(dy.t(), h)); };
  if (M > 0 && xdna_gated_grads_pick(M, K, F, N) && (short_block(M, K, F, N) || !apart())) {
    r.dx = empty_xdna({M, K}, at::kBFloat16);
    r.dw_in = empty_xdna({2 * F, K}, at::kBFloat16);
    if (N) r.dw_out = empty_xdna({N, F}, at::kBFloat16);
    check_abi(xdna_gated_grads_bf16(p16(dgu), p16(x), row_stride(x), p16(w), row_stride(w), N ? p16(dy) : nullptr,
                                    N ? row_stride(dy) : 0, N ? p16(h) : nullptr, M, K, F, N, m16(r.dx), m16(r.dw_in),
                                    N ? m16(r.dw_out) : nullptr, current_stream()),
              "gated backward");
    return r;
  }
  r.dx = product(dgu, w);
  r.dw_in = product(dgu.t(), x);
  if (N) r.dw_out = product(dy.t(), h);
  return r;
}

std::vector<int64_t> with_last(const at::Tensor& x, int64_t n) {
  auto s = x.sizes().vec();
  s.back() = n;
  return s;
}

struct GatedLinearFn : public torch::autograd::Function<GatedLinearFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w_in, int64_t act) {
    ScopedCount sc("hip_tokens.gated.fwd.run");
    const GatedForward f = gated_forward(x, w_in, act, true);
    ctx->save_for_backward({x, w_in, f.gu});
    ctx->saved_data["act"] = act;
    return f.h.view(with_last(x, f.h.size(1)));
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("gated_linear");
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor()};
    ScopedCount sc("hip_tokens.gated.bwd.run");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor dgu = gated_dgu(grads[0], saved[2], ctx->saved_data["act"].toInt());
    at::Tensor dx, dw;
    if (ctx->needs_input_grad(0) && ctx->needs_input_grad(1)) {
      const GatedGrads g = gated_grads(dgu, as_rows(saved[0]), as_rows(saved[1]), at::Tensor(), at::Tensor());
      return {g.dx.view(saved[0].sizes()), g.dw_in, at::Tensor()};
    }
    if (ctx->needs_input_grad(0)) dx = product(dgu, as_rows(saved[1])).view(saved[0].sizes());
    if (ctx->needs_input_grad(1)) dw = product(dgu.t(), as_rows(saved[0]));
    return {dx, dw, at::Tensor()};
  }
};

struct GatedMlpFn : public torch::autograd::Function<GatedMlpFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w_in,
                            const at::Tensor& w_out, int64_t act) {
    ScopedCount sc("hip_tokens.gated.fwd.run");
    const GatedForward f = gated_forward(x, w_in, act, true);
    ctx->save_for_backward({x, w_in, w_out, f.gu, f.h});
    ctx->saved_data["act"] = act;
    return product(f.h, as_rows(w_out).t()).view(with_last(x, w_out.size(0)));
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("gated_mlp");
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    ScopedCount sc("hip_tokens.gated.bwd.run");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &w_in = saved[1], &w_out = saved[2], &gu = saved[3], &h = saved[4];
    const at::Tensor dy = as_rows(grads[0]);
    at::Tensor dx, dw_in, dw_out;
    if (ctx->needs_input_grad(0) || ctx->needs_input_grad(1)) {
      const at::Tensor wo = as_rows(w_out);
      at::Tensor dgu = empty_xdna({h.size(0), 2 * h.size(1)}, at::kBFloat16);
      check_abi(xdna_gated_mlp_bwd_bf16(p16(dy), row_stride(dy), p16(wo), row_stride(wo), cptr(gu), dy.size(0), dy.size(1),
                                        h.size(1), int(ctx->saved_data["act"].toInt()), m16(dgu), current_stream()),
                "gated_mlp backward");
      if (ctx->needs_input_grad(0) && ctx->needs_input_grad(1) && ctx->needs_input_grad(2)) {
        const GatedGrads g = gated_grads(dgu, as_rows(x), as_rows(w_in), dy, h);
        return {g.dx.view(x.sizes()), g.dw_in, g.dw_out, at::Tensor()};
      }
      if (ctx->needs_input_grad(0)) dx = product(dgu, as_rows(w_in)).view(x.sizes());
      if (ctx->needs_input_grad(1)) dw_in = product(dgu.t(), as_rows(x));
    }
    if (ctx->needs_input_grad(2)) dw_out = product(dy.t(), h);
    return {dx, dw_in, dw_out, at::Tensor()};
  }
};

void check_gated(const char* op, const at::Tensor& x, const at::Tensor& w_in) {
  check_bf16(x, op, "x");
  check_bf16(w_in, op, "w_in");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, op, ": x needs a last dimension");
  TORCH_CHECK(w_in.dim() == 2 && w_in.size(0) >= 2 && w_in.size(0) % 2 == 0 && w_in.size(1) == x.size(-1), op,
              ": w_in must hold the gate rows and then the up rows, [2 F, ", x.size(-1), "], got ", w_in.sizes());
  TORCH_CHECK(x.numel() / x.size(-1) <= (int64_t(1) << 22) && w_in.size(0) <= (int64_t(1) << 30) &&
                  w_in.size(1) <= (int64_t(1) << 30),
              op, ": too many rows");
}

// ---- distillation --------------------------------------------------------------------------------

// What a call's kernels write beside the loss, in one buffer (an allocation each would cost a short
// call as much as its kernels): the pieces' workspace, [T] (m, 1 / s), [T][k] p, [T] shares,
// [T] row losses (where the loss itself is one number) and 1 / sum of the weights.
struct DistillAux {
  size_t workspace;  // bytes, a multiple of 16
  int64_t T, k;
  DistillAux(int64_t rows, int64_t V, int64_t entries)
      : workspace((xdna_distill_workspace_bytes(rows, V) + 15) / 16 * 16), T(rows), k(entries) {}
  int64_t bytes() const { return int64_t(workspace) + (T * (k + 4) + 1) * int64_t(sizeof(float)); }
  float* stats(void* p) const { return reinterpret_cast<float*>(static_cast<char*>(p) + workspace); }
  float* p(void* b) const { return stats(b) + 2 * T; }
  float* share(void* b) const { return p(b) + T * k; }
  float* row(void* b) const { return share(b) + T; }
  float* inv_weight(void* b) const { return row(b) + T; }
};

struct DistillForward {
  at::Tensor loss, ids, aux;
};

DistillForward distill_forward(const at::Tensor& logits, const at::Tensor& teacher_ids, const at::Tensor& teacher,
                               double tau, const std::optional<at::Tensor>& weight, int64_t reduction) {
  ScopedCount sc("hip_tokens.distill.fwd.run");
  DistillForward r;
  const at::Tensor z = as_rows(logits), t = as_rows(teacher).contiguous();
  r.ids = as_rows(teacher_ids).contiguous();
  at::Tensor w;
  if (weight.has_value()) w = weight->to(at::kFloat).contiguous();
  const DistillAux aux(z.size(0), z.size(1), r.ids.size(1));
  r.loss = reduction == 0 ? empty_xdna(logits.sizes().slice(0, logits.dim() - 1), at::kFloat) : empty_xdna({}, at::kFloat);
  r.aux = workspace(size_t(aux.bytes()));
  void* b = r.aux.data_ptr();
  float* loss = static_cast<float*>(ptr_or_null(r.loss));
  check_abi(xdna_distill(cptr(z), z.scalar_type() == at::kFloat ? 1 : 2, aux.T, z.size(1), row_stride(z), cptr(r.ids),
                         r.ids.scalar_type() == at::kLong ? 8 : 4, cptr(t), t.scalar_type() == at::kFloat ? 1 : 2,
                         int(aux.k), float(tau), cf32(w), int(reduction), reduction == 0 ? loss : aux.row(b), aux.share(b),
                         aux.stats(b), aux.p(b), reduction == 0 ? nullptr : loss, aux.inv_weight(b), b, aux.workspace,
                         current_stream()),
            "distill_loss");
  return r;
}

struct DistillFn : public torch::autograd::Function<DistillFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& ids,
                            const at::Tensor& teacher, double tau, const std::optional<at::Tensor>& weight,
                            int64_t reduction) {
    const DistillForward f = distill_forward(logits, ids, teacher, tau, weight, reduction);
    ctx->save_for_backward({logits, f.ids, f.aux});
    ctx->saved_data["tau"] = tau;
    ctx->saved_data["rows"] = reduction == 0;
    return f.loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("distill_loss");
    variable_list none(6);
    if (!grads[0].defined()) return none;
    ScopedCount sc("hip_tokens.distill.bwd.run");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor z = as_rows(saved[0]), go = grads[0].contiguous();
    const at::Tensor& ids = saved[1];
    const bool rows = ctx->saved_data["rows"].toBool();
    const DistillAux aux(z.size(0), z.size(1), ids.size(1));
    void* b = saved[2].data_ptr();
    at::Tensor dz = empty_xdna(saved[0].sizes(), z.scalar_type());
    check_abi(xdna_distill_bwd(cptr(z), z.scalar_type() == at::kFloat ? 1 : 2, z.size(0), z.size(1), row_stride(z),
                               cptr(ids), ids.scalar_type() == at::kLong ? 8 : 4, int(ids.size(1)),
                               float(ctx->saved_data["tau"].toDouble()), aux.share(b), aux.stats(b), aux.p(b),
                               rows ? nullptr : aux.inv_weight(b), cptr(go),
                               float_code(go, "distill_loss", "the gradient"), rows ? 1 : 0, ptr_or_null(dz),
                               current_stream()),
              "distill_loss backward");
    none[0] = dz;
    return none;
  }
};

// ---- token log probabilities -----------------------------------------------------------------------

struct LogprobForward {
  at::Tensor log_probs, entropy, top_log_probs, top_ids, targets, stats;
};

size_t logprob_workspace(int64_t T, int64_t V, int64_t top) {
  return (xdna_token_logprobs_workspace_bytes(T, V, int(top)) + 15) / 16 * 16;
}

float* stats_in(void* b, size_t workspace) {
  return b ? reinterpret_cast<float*>(static_cast<char*>(b) + workspace) : nullptr;
}

LogprobForward logprob_forward(const at::Tensor& logits, const at::Tensor& targets, int64_t top, double tau) {
  ScopedCount sc("hip_tokens.logprobs.fwd.run");
  LogprobForward r;
  const at::Tensor z = as_rows(logits);
  r.targets = targets.contiguous();
  const int64_t T = z.size(0), V = z.size(1);
  auto shape = targets.sizes().vec();
  r.log_probs = empty_xdna(shape, at::kFloat);
  r.entropy = empty_xdna(shape, at::kFloat);
  // the pieces' workspace, then [T] (m, 1 / s)
  const size_t bytes = logprob_workspace(T, V, top);
  r.stats = workspace(bytes + size_t(T) * 2 * sizeof(float));
  shape.push_back(top);
  r.top_log_probs = empty_xdna(shape, at::kFloat);
  r.top_ids = empty_xdna(shape, at::kLong);
  void* b = ptr_or_null(r.stats);
  check_abi(xdna_token_logprobs(cptr(z), z.scalar_type() == at::kFloat ? 1 : 2, T, V, row_stride(z), cptr(r.targets),
                                r.targets.scalar_type() == at::kLong ? 8 : 4, float(tau), int(top), f32(r.log_probs),
                                f32(r.entropy), stats_in(b, bytes), f32(r.top_log_probs),
                                static_cast<int64_t*>(ptr_or_null(r.top_ids)), b, bytes, current_stream()),
            "token_log_probs");
  return r;
}

struct LogprobFn : public torch::autograd::Function<LogprobFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& targets, int64_t top,
                               double tau) {
    const LogprobForward f = logprob_forward(logits, targets, top, tau);
    // entropy goes through a detached alias: as an output it carries this node
    ctx->save_for_backward({logits, f.targets, f.stats, f.entropy.detach()});
    ctx->saved_data["tau"] = tau;
    ctx->saved_data["top"] = top;
    ctx->mark_non_differentiable({f.top_log_probs, f.top_ids});
    ctx->set_materialize_grads(false);
    return {f.log_probs, f.entropy, f.top_log_probs, f.top_ids};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("token_log_probs");
    variable_list none(4);
    if (!grads[0].defined() && !grads[1].defined()) return none;
    ScopedCount sc("hip_tokens.logprobs.bwd.run");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor z = as_rows(saved[0]);
    const at::Tensor gl = grads[0].defined() ? grads[0].to(at::kFloat).contiguous() : grads[0];
    const at::Tensor gh = grads[1].defined() ? grads[1].to(at::kFloat).contiguous() : grads[1];
    at::Tensor dz = empty_xdna(saved[0].sizes(), z.scalar_type());
    check_abi(xdna_token_logprobs_bwd(cptr(z), z.scalar_type() == at::kFloat ? 1 : 2, z.size(0), z.size(1),
                                      row_stride(z), cptr(saved[1]), saved[1].scalar_type() == at::kLong ? 8 : 4,
                                      float(ctx->saved_data["tau"].toDouble()),
                                      stats_in(ptr_or_null(saved[2]), logprob_workspace(z.size(0), z.size(1), ctx->saved_data["top"].toInt())),
                                      cf32(saved[3]), cf32(gl), cf32(gh), ptr_or_null(dz), current_stream()),
              "token_log_probs backward");
    none[0] = dz;
    return none;
  }
};

// ---- layer norm ------------------------------------------------------------------------------------
// A tensor that a call leaves out is undefined here and an empty optional to its node, which has no
// edge for it: whether argument `i` of those that are there gets a gradient is asked by its place among them.
std::optional<at::Tensor> given(const at::Tensor& t) { return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt; }

struct Wanted {
  AutogradContext* ctx;
  size_t next = 0;
  bool operator()(bool there) { return there && ctx->needs_input_grad(next++); }
};

int param_code(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias) {
  const at::Tensor& p = weight.defined() ? weight : bias;
  return (p.defined() ? p : x).scalar_type() == at::kFloat ? 1 : 2;
}

struct NormForward {
  at::Tensor y, sum, stats;  // sum: undefined without a residual
};

NormForward norm_forward(const at::Tensor& x, const at::Tensor& residual, const at::Tensor& weight, const at::Tensor& bias,
                         double eps, bool keep) {
  ScopedCount sc("hip_tokens.norm.fwd.run");
  NormForward r;
  const at::Tensor xr = as_rows(x), rr = residual.defined() ? as_rows(residual) : residual;
  const at::Tensor w = weight.defined() ? weight.contiguous() : weight, b = bias.defined() ? bias.contiguous() : bias;
  r.y = empty_xdna(x.sizes(), x.scalar_type());
  if (residual.defined()) r.sum = empty_xdna(x.sizes(), x.scalar_type());
  if (keep) r.stats = empty_xdna({xr.size(0), 2}, at::kFloat);
  check_abi(xdna_layer_norm(cptr(xr), row_stride(xr), cptr(rr), rr.defined() ? row_stride(rr) : 0,
                            xr.scalar_type() == at::kFloat ? 1 : 2, xr.size(0), xr.size(1), cptr(w), cptr(b),
                            param_code(x, w, b), float(eps), ptr_or_null(r.sum), ptr_or_null(r.y),
                            static_cast<float*>(ptr_or_null(r.stats)), current_stream()),
            "layer_norm");
  return r;
}

struct LayerNormFn : public torch::autograd::Function<LayerNormFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const std::optional<at::Tensor>& residual_,
                               const std::optional<at::Tensor>& weight_, const std::optional<at::Tensor>& bias_, double eps) {
    const at::Tensor residual = residual_.value_or(at::Tensor()), weight = weight_.value_or(at::Tensor()),
                     bias = bias_.value_or(at::Tensor());
    const NormForward f = norm_forward(x, residual, weight, bias, eps, true);
    // the sum goes through a detached alias: as an output it carries this node
    ctx->save_for_backward({residual.defined() ? f.sum.detach() : x, weight, bias, f.stats});
    ctx->saved_data["add"] = residual.defined();
    ctx->set_materialize_grads(false);
    if (residual.defined()) return {f.y, f.sum};
    return {f.y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("layer_norm");
    variable_list none(5);
    const at::Tensor dsum = grads.size() > 1 ? grads[1] : at::Tensor();
    const auto saved = ctx->get_saved_variables();
    Wanted wanted{ctx};
    const bool want_x = wanted(true), want_r = wanted(ctx->saved_data["add"].toBool()), want_w = wanted(saved[1].defined()),
               want_b = wanted(saved[2].defined());
    if (!grads[0].defined()) {  // the norm has no gradient, the sum may have one
      if (want_x) none[0] = dsum;
      if (want_r) none[1] = dsum;
      return none;
    }
    ScopedCount sc("hip_tokens.norm.bwd.run");
    const at::Tensor x = as_rows(saved[0]), dy = as_rows(grads[0]), ds = dsum.defined() ? as_rows(dsum) : dsum;
    const at::Tensor w = saved[1].defined() ? saved[1].contiguous() : saved[1];
    const int64_t R = x.size(0), D = x.size(1);
    const int pt = param_code(x, saved[1], saved[2]);
    const at::ScalarType ptype = pt == 1 ? at::kFloat : at::kBFloat16;
    at::Tensor dx, dw, db, ws;
    if (want_x || want_r) dx = empty_xdna(saved[0].sizes(), x.scalar_type());
    if (want_w) dw = empty_xdna({D}, ptype);
    if (want_b) db = empty_xdna({D}, ptype);
    const size_t bytes = dw.defined() || db.defined() ? xdna_layer_norm_bwd_workspace_bytes(R, D) : 0;
    if (bytes) ws = workspace(bytes);
    check_abi(xdna_layer_norm_bwd(cptr(dy), row_stride(dy), cptr(ds), ds.defined() ? row_stride(ds) : 0, cptr(x), row_stride(x),
                                  x.scalar_type() == at::kFloat ? 1 : 2, R, D, cptr(w), pt, cf32(saved[3]), ptr_or_null(dx),
                                  ptr_or_null(dw), ptr_or_null(db), ptr_or_null(ws), bytes, current_stream()),
              "layer_norm backward");
    if (want_x) none[0] = dx;
    if (want_r) none[1] = dx;
    none[2] = dw;
    none[3] = db;
    return none;
  }
};

// ---- linear layer ------------------------------------------------------------------------------------

constexpr int64_t kNoActivation = 3;

struct LinearForward {
  at::Tensor y, kept;  // kept: undefined where no slopes are
};

LinearForward linear_forward(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, const at::Tensor& residual,
                             int64_t act, bool keep) {
  ScopedCount sc("hip_tokens.linear.fwd.run");
  LinearForward r;
  const at::Tensor xr = as_rows(x), w = as_rows(weight), b = bias.defined() ? bias.contiguous() : bias;
  const at::Tensor rr = residual.defined() ? as_rows(residual) : residual;
  const int64_t M = xr.size(0), K = xr.size(1), N = w.size(0);
  r.y = empty_xdna(with_last(x, N), at::kBFloat16);
  if (keep && act != kNoActivation) r.kept = workspace(xdna_linear_kept_bytes(M, N, int(act)));
  check_abi(xdna_linear_bf16(p16(xr), row_stride(xr), p16(w), row_stride(w), M, K, N, int(act),
                             static_cast<const uint16_t*>(cptr(b)), static_cast<const uint16_t*>(cptr(rr)),
                             rr.defined() ? row_stride(rr) : 0, static_cast<uint16_t*>(ptr_or_null(r.y)),
                             ptr_or_null(r.kept), current_stream()),
            "linear");
  return r;
}

struct LinearFn : public torch::autograd::Function<LinearFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                            const std::optional<at::Tensor>& bias_, const std::optional<at::Tensor>& residual_, int64_t act) {
    const at::Tensor bias = bias_.value_or(at::Tensor()), residual = residual_.value_or(at::Tensor());
    // only the gradient of what comes before the activation takes its slopes
    const auto wants = [](const at::Tensor& t) { return t.defined() && t.requires_grad(); };
    const LinearForward f = linear_forward(x, weight, bias, residual, act, wants(x) || wants(weight) || wants(bias));
    ctx->save_for_backward({x, weight, f.kept});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = bias.defined();
    ctx->saved_data["residual"] = residual.defined();
    return f.y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("linear");
    variable_list out(5);
    if (!grads[0].defined()) return out;
    Wanted wanted{ctx};
    const bool want_x = wanted(true), want_w = wanted(true), want_b = wanted(ctx->saved_data["bias"].toBool());
    if (wanted(ctx->saved_data["residual"].toBool())) out[3] = grads[0];
    if (!want_x && !want_w && !want_b) return out;
    ScopedCount sc("hip_tokens.linear.bwd.run");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor x = as_rows(saved[0]), w = as_rows(saved[1]), dy = as_rows(grads[0]), &kept = saved[2];
    const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
    at::Tensor dp = dy, db, ws;
    const bool slopes = kept.defined(), own_dp = slopes && (want_x || want_w);
    if (own_dp) dp = empty_xdna({M, N}, at::kBFloat16);
    if (want_b) db = empty_xdna({N}, at::kBFloat16);
    if (slopes || want_b) {
      const size_t bytes = want_b ? xdna_linear_bwd_workspace_bytes(M, N) : 0;
      if (bytes) ws = workspace(bytes);
      check_abi(xdna_linear_bwd_bf16(p16(dy), row_stride(dy), ptr_or_null(kept), int(ctx->saved_data["act"].toInt()), M, N,
                                     own_dp ? static_cast<uint16_t*>(ptr_or_null(dp)) : nullptr,
                                     static_cast<uint16_t*>(ptr_or_null(db)), ptr_or_null(ws), bytes, current_stream()),
                "linear backward");
      out[2] = db;
    }
    const int how = want_x && want_w && M > 0
                        ? xdna_linear_grads_pick(p16(dp), row_stride(dp), p16(x), row_stride(x), p16(w), row_stride(w), M, K, N)
                        : 0;
    if (how == 2 || (how == 1 && (short_block(M, K, N, 0) || !(on_gemm(dp, w) || on_gemm(dp.t(), x))))) {
      at::Tensor dx = empty_xdna({M, K}, at::kBFloat16), dw = empty_xdna({N, K}, at::kBFloat16);
      check_abi(xdna_linear_grads_bf16(p16(dp), row_stride(dp), p16(x), row_stride(x), p16(w), row_stride(w), M, K, N, m16(dx),
                                       m16(dw), current_stream()),
                "linear backward");
      out[0] = dx.view(saved[0].sizes());
      out[1] = dw;
      return out;
    }
    if (want_x) out[0] = product(dp, w).view(saved[0].sizes());
    if (want_w) out[1] = product(dp.t(), x);
    return out;
  }
};

// ---- decay attention ---------------------------------------------------------------------------------

// [B, T, H, D] as the C ABI takes it: unit stride along the head, no negative stride (a copy only
// where the strides are others)
at::Tensor as_heads(const at::Tensor& t) { return t.size(-1) > 1 && t.stride(-1) != 1 ? t.contiguous() : t; }

xdna_heads_bf16 heads_of(const at::Tensor& t) { return {p16(t), t.stride(0), t.stride(1), t.stride(2)}; }

struct DecaySizes {
  int64_t B, T, H, G, dk, dv;
  DecaySizes(const at::Tensor& q, const at::Tensor& v)
      : B(q.size(0)), T(q.size(1)), H(q.size(2)), G(v.size(2)), dk(q.size(3)), dv(v.size(3)) {}
  bool none() const { return B == 0 || T == 0; }
};

int index_size(const at::Tensor& t) { return t.defined() && t.scalar_type() == at::kInt ? 4 : 8; }

struct DecayForward {
  at::Tensor out, state;
};

DecayForward decay_forward(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& state_,
                           const at::Tensor& log_decay, const at::Tensor& lengths, double scale) {
  ScopedCount sc("hip_tokens.decay.fwd.run");
  const DecaySizes n(q_, v_);
  DecayForward r;
  const at::Tensor q = as_heads(q_), k = as_heads(k_), v = as_heads(v_), state = state_.defined() ? state_.contiguous() : state_;
  r.out = empty_xdna({n.B, n.T, n.H, n.dv}, at::kBFloat16);
  r.state = empty_xdna({n.B, n.H, n.dk, n.dv}, at::kFloat);
  if (n.none()) {
    if (state.defined()) r.state.copy_(state);
    else r.state.zero_();
    return r;
  }
  const size_t bytes = xdna_decay_workspace_bytes(n.B, n.T, n.H, n.dk, n.dv);
  at::Tensor ws;
  if (bytes) ws = workspace(bytes);
  const xdna_heads_bf16 hq = heads_of(q), hk = heads_of(k), hv = heads_of(v);
  check_abi(xdna_decay_attention(&hq, &hk, &hv, n.B, n.T, n.H, n.G, n.dk, n.dv, cf32(log_decay), cptr(lengths),
                                 index_size(lengths), float(scale), cf32(state), m16(r.out), f32(r.state), ptr_or_null(ws), bytes,
                                 current_stream()),
            "decay_attention");
  return r;
}

struct DecayFn : public torch::autograd::Function<DecayFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                               const std::optional<at::Tensor>& state_, const at::Tensor& log_decay,
                               const std::optional<at::Tensor>& lengths_, double scale) {
    const at::Tensor state = state_.value_or(at::Tensor()), lengths = lengths_.value_or(at::Tensor());
    const DecayForward f = decay_forward(q, k, v, state, log_decay, lengths, scale);
    ctx->save_for_backward({q, k, v, state, log_decay, lengths});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    return {f.out, f.state};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("decay_attention");
    variable_list none(7);
    if (!grads[0].defined() && !grads[1].defined()) return none;
    ScopedCount sc("hip_tokens.decay.bwd.run");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor q = as_heads(saved[0]), k = as_heads(saved[1]), v = as_heads(saved[2]);
    const at::Tensor state = saved[3].defined() ? saved[3].contiguous() : saved[3];
    const at::Tensor &log_decay = saved[4], &lengths = saved[5];
    const DecaySizes n(q, v);
    at::Tensor dout = grads[0].defined() ? as_heads(grads[0]) : empty_xdna({n.B, n.T, n.H, n.dv}, at::kBFloat16).zero_();
    const at::Tensor ds = grads[1].defined() ? grads[1].contiguous() : grads[1];
    at::Tensor dq = empty_xdna(q.sizes(), at::kBFloat16), dk = empty_xdna(k.sizes(), at::kBFloat16),
               dv = empty_xdna(v.sizes(), at::kBFloat16), d_state;
    if (state.defined() && ctx->needs_input_grad(3)) d_state = empty_xdna({n.B, n.H, n.dk, n.dv}, at::kFloat);
    if (n.none()) {
      if (d_state.defined() && ds.defined()) d_state.copy_(ds);
      else if (d_state.defined()) d_state.zero_();
    } else {
      const size_t bytes = xdna_decay_bwd_workspace_bytes(n.B, n.T, n.H, n.G, n.dk, n.dv);
      at::Tensor ws;
      if (bytes) ws = workspace(bytes);
      const xdna_heads_bf16 ho = heads_of(dout), hq = heads_of(q), hk = heads_of(k), hv = heads_of(v);
      check_abi(xdna_decay_attention_bwd(&ho, cf32(ds), &hq, &hk, &hv, n.B, n.T, n.H, n.G, n.dk, n.dv, cf32(log_decay),
                                         cptr(lengths), index_size(lengths), float(ctx->saved_data["scale"].toDouble()),
                                         cf32(state), m16(dq), m16(dk), m16(dv), f32(d_state), ptr_or_null(ws), bytes,
                                         current_stream()),
                "decay_attention backward");
    }
    none[0] = dq;
    none[1] = dk;
    none[2] = dv;
    none[3] = d_state;
    return none;
  }
};

// q, k, v of heads after `lead` dimensions (2: batch, tokens; 1: batch), log_decay and scale
void check_decay(const char* op, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay,
                 int64_t lead, double scale) {
  check_bf16(q, op, "q");
  check_bf16(k, op, "k");
  check_bf16(v, op, "v");
  TORCH_CHECK(q.dim() == lead + 2 && k.dim() == lead + 2 && v.dim() == lead + 2 &&
                  q.sizes().slice(0, lead) == k.sizes().slice(0, lead) && q.sizes().slice(0, lead) == v.sizes().slice(0, lead),
              op, ": q, k and v must be [", lead == 2 ? "batch, tokens" : "batch", ", heads, size], got ", q.sizes(), ", ", k.sizes(),
              " and ", v.sizes());
  const int64_t H = q.size(lead), G = k.size(lead);
  TORCH_CHECK(q.size(-1) == k.size(-1), op, ": q and k have heads of ", q.size(-1), " and ", k.size(-1));
  TORCH_CHECK(q.size(-1) >= 1 && q.size(-1) <= 128 && v.size(-1) >= 1 && v.size(-1) <= 128, op, ": heads of 1 to 128, got ",
              q.size(-1), " and ", v.size(-1));
  TORCH_CHECK(G >= 1 && v.size(lead) == G && H >= G && H % G == 0, op, ": k and v must have as many heads, a divisor of q's ", H,
              ", got ", G, " and ", v.size(lead));
  TORCH_CHECK(on_xdna(log_decay) && log_decay.scalar_type() == at::kFloat && log_decay.dim() == 1 && log_decay.size(0) == H, op,
              ": log_decay must be a float32 xdna tensor of ", H, " heads");
  TORCH_CHECK(!(at::GradMode::is_enabled() && log_decay.requires_grad()), op, ": log_decay is a constant, it gets no gradient");
  TORCH_CHECK(std::isfinite(float(scale)), op, ": scale must be finite in fp32, got ", scale);
}

void check_tau(const char* op, double tau) {
  // the kernels divide by tau in base 2: log2(e) / tau has to be a finite fp32 number
  TORCH_CHECK(float(tau) > 0.0f && std::isfinite(float(tau)) && std::isfinite(1.0f / float(tau) * 1.442695041f), op,
              ": temperature must be positive and finite (in fp32, and log2(e) / temperature too), got ", tau);
}

void check_logits(const char* op, const at::Tensor& logits) {
  float_code(logits, op, "logits");
  TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1 && logits.size(-1) <= (int64_t(1) << 22), op,
              ": logits need a last dimension of 1 .. 2^22 tokens, got ", logits.sizes());
}

}  // namespace

at::Tensor token_embed(const at::Tensor& ids, const at::Tensor& weight, double scale, std::optional<int64_t> padding) {
  no_tangents("embed", {&weight});
  index_bytes(ids, "embed", "ids");
  float_code(weight, "embed", "weight");
  TORCH_CHECK(weight.dim() == 2 && weight.size(0) >= 1 && weight.size(1) >= 1, "embed: weight must be [tokens, width], got ",
              weight.sizes());
  TORCH_CHECK(std::isfinite(float(scale)), "embed: scale must be finite in fp32, got ", scale);
  const int64_t V = weight.size(0);
  int64_t pad = -1;
  if (padding.has_value()) {
    pad = *padding < 0 ? *padding + V : *padding;
    TORCH_CHECK(pad >= 0 && pad < V, "embed: padding_idx ", *padding, " outside a table of ", V, " rows");
  }
  if (tracked({&weight})) return EmbedFn::apply(ids, weight, scale, pad);
  return embed_forward(ids, weight, scale);
}

at::Tensor token_gated_linear(const at::Tensor& x, const at::Tensor& w_in, int64_t act) {
  no_tangents("gated_linear", {&x, &w_in});
  check_gated("gated_linear", x, w_in);
  if (tracked({&x, &w_in})) return GatedLinearFn::apply(x, w_in, act);
  ScopedCount sc("hip_tokens.gated.fwd.run");
  const GatedForward f = gated_forward(x, w_in, act, false);
  return f.h.view(with_last(x, f.h.size(1)));
}

at::Tensor token_gated_mlp(const at::Tensor& x, const at::Tensor& w_in, const at::Tensor& w_out, int64_t act) {
  no_tangents("gated_mlp", {&x, &w_in, &w_out});
  check_gated("gated_mlp", x, w_in);
  check_bf16(w_out, "gated_mlp", "w_out");
  TORCH_CHECK(w_out.dim() == 2 && w_out.size(0) >= 1 && w_out.size(0) <= (int64_t(1) << 30) &&
                  w_out.size(1) == w_in.size(0) / 2,
              "gated_mlp: w_out must be [N, ", w_in.size(0) / 2, "], got ", w_out.sizes());
  if (tracked({&x, &w_in, &w_out})) return GatedMlpFn::apply(x, w_in, w_out, act);
  ScopedCount sc("hip_tokens.gated.fwd.run");
  const GatedForward f = gated_forward(x, w_in, act, false);
  return product(f.h, as_rows(w_out).t()).view(with_last(x, w_out.size(0)));
}

std::tuple<at::Tensor, at::Tensor> token_layer_norm(const at::Tensor& x, const std::optional<at::Tensor>& residual,
                                                    const std::optional<at::Tensor>& weight,
                                                    const std::optional<at::Tensor>& bias, double eps) {
  const char* op = residual.has_value() ? "add_layer_norm" : "layer_norm";
  const at::Tensor r = residual.value_or(at::Tensor()), w = weight.value_or(at::Tensor()), b = bias.value_or(at::Tensor());
  no_tangents(op, {&x, &r, &w, &b});
  float_code(x, op, "x");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= (int64_t(1) << 24) && x.numel() / x.size(-1) <= (int64_t(1) << 30),
              op, ": x must be [..., width], width 1 .. 2^24 and up to 2^30 rows, got ", x.sizes());
  if (r.defined())
    TORCH_CHECK(on_xdna(r) && r.scalar_type() == x.scalar_type() && r.sizes() == x.sizes(), op, ": residual must be an xdna tensor like x, ",
                x.scalar_type(), " ", x.sizes());
  for (const at::Tensor* p : {&w, &b})
    TORCH_CHECK(!p->defined() || (on_xdna(*p) && (p->scalar_type() == at::kFloat || p->scalar_type() == x.scalar_type()) &&
                                  p->dim() == 1 && p->size(0) == x.size(-1)),
                op, ": weight and bias must be xdna tensors [", x.size(-1), "] of float32 or of x's type");
  TORCH_CHECK(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), op, ": weight and bias must be of one type");
  TORCH_CHECK(float(eps) >= 0.0f && std::isfinite(float(eps)), op, ": eps must be finite and not negative, got ", eps);
  const auto wants = [](const at::Tensor& t) { return t.defined() && t.requires_grad(); };
  if (at::GradMode::is_enabled() && (wants(x) || wants(r) || wants(w) || wants(b))) {
    const variable_list v = LayerNormFn::apply(x, given(r), given(w), given(b), eps);
    return {v[0], v.size() > 1 ? v[1] : at::Tensor()};
  }
  const NormForward f = norm_forward(x, r, w, b, eps, false);
  return {f.y, f.sum};
}

at::Tensor token_linear(const at::Tensor& x, const at::Tensor& weight, const std::optional<at::Tensor>& bias,
                        const std::optional<at::Tensor>& residual, int64_t act) {
  const char* op = "linear";
  const at::Tensor b = bias.value_or(at::Tensor()), r = residual.value_or(at::Tensor());
  no_tangents(op, {&x, &weight, &b, &r});
  check_bf16(x, op, "x");
  check_bf16(weight, op, "weight");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= (int64_t(1) << 30), op, ": x needs a last dimension");
  TORCH_CHECK(weight.dim() == 2 && weight.size(0) >= 1 && weight.size(0) <= (int64_t(1) << 22) && weight.size(1) == x.size(-1), op,
              ": weight must be [units, ", x.size(-1), "], up to 2^22 units, got ", weight.sizes());
  TORCH_CHECK(x.numel() / x.size(-1) <= (int64_t(1) << 22), op, ": more than 2^22 rows");
  if (b.defined()) {
    check_bf16(b, op, "bias");
    TORCH_CHECK(b.dim() == 1 && b.size(0) == weight.size(0), op, ": bias must be [", weight.size(0), "], got ", b.sizes());
  }
  if (r.defined()) {
    check_bf16(r, op, "residual");
    const std::vector<int64_t> want = with_last(x, weight.size(0));
    TORCH_CHECK(r.sizes() == at::IntArrayRef(want), op, ": residual must be ", at::IntArrayRef(want), ", got ", r.sizes());
  }
  const auto wants = [](const at::Tensor& t) { return t.defined() && t.requires_grad(); };
  if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(b) || wants(r)))
    return LinearFn::apply(x, weight, given(b), given(r), act);
  return linear_forward(x, weight, b, r, act, false).y;
}

std::tuple<at::Tensor, at::Tensor> token_decay(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                               const at::Tensor& log_decay, const std::optional<at::Tensor>& state,
                                               const std::optional<at::Tensor>& lengths, double scale) {
  const char* op = "decay_attention";
  const at::Tensor s = state.value_or(at::Tensor()), l = lengths.has_value() ? lengths->contiguous() : at::Tensor();
  no_tangents(op, {&q, &k, &v, &log_decay, &s});
  check_decay(op, q, k, v, log_decay, 2, scale);
  if (s.defined()) {
    const std::vector<int64_t> want = {q.size(0), q.size(2), q.size(3), v.size(3)};
    TORCH_CHECK(on_xdna(s) && s.scalar_type() == at::kFloat && s.sizes() == at::IntArrayRef(want), op,
                ": state must be a float32 xdna tensor ", at::IntArrayRef(want));
  }
  if (l.defined()) {
    index_bytes(l, op, "lengths");
    TORCH_CHECK(l.dim() == 1 && l.size(0) == q.size(0), op, ": lengths must be [", q.size(0), "], got ", l.sizes());
  }
  const at::Tensor g = log_decay.contiguous();
  if (tracked({&q, &k, &v}) || (s.defined() && tracked({&s}))) {
    const variable_list r = DecayFn::apply(q, k, v, given(s), g, given(l), scale);
    return {r[0], r[1]};
  }
  const DecayForward f = decay_forward(q, k, v, s, g, l, scale);
  return {f.out, f.state};
}

at::Tensor token_decay_step(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& log_decay,
                            at::Tensor state, const std::optional<at::Tensor>& slots, double scale) {
  const char* op = "decay_attention_step";
  const at::Tensor l = slots.has_value() ? slots->contiguous() : at::Tensor();
  no_tangents(op, {&q_, &k_, &v_, &log_decay, &state});
  check_decay(op, q_, k_, v_, log_decay, 1, scale);
  TORCH_CHECK(!tracked({&q_, &k_, &v_, &state}), op, " writes the state in place and has no gradient: call it under no_grad");
  const int64_t B = q_.size(0), H = q_.size(1), G = k_.size(1), dk = q_.size(2), dv = v_.size(2);
  TORCH_CHECK(on_xdna(state) && state.scalar_type() == at::kFloat && state.dim() == 4 && state.is_contiguous() &&
                  state.size(1) == H && state.size(2) == dk && state.size(3) == dv,
              op, ": state must be a contiguous float32 xdna tensor [slots, ", H, ", ", dk, ", ", dv, "], got ", state.sizes());
  if (l.defined()) {
    index_bytes(l, op, "slots");
    TORCH_CHECK(l.dim() == 1 && l.size(0) == B, op, ": slots must be [", B, "], got ", l.sizes());
  } else {
    TORCH_CHECK(state.size(0) == B, op, ": without slots the states must be the batch's ", B, ", got ", state.size(0));
  }
  ScopedCount sc("hip_tokens.decay.step.run");
  at::Tensor out = empty_xdna({B, H, dv}, at::kBFloat16);
  if (B == 0) return out;
  const at::Tensor q = as_heads(q_), k = as_heads(k_), v = as_heads(v_), g = log_decay.contiguous();
  const auto heads = [](const at::Tensor& t) { return xdna_heads_bf16{p16(t), t.stride(0), 0, t.stride(1)}; };
  const xdna_heads_bf16 hq = heads(q), hk = heads(k), hv = heads(v);
  check_abi(xdna_decay_step(&hq, &hk, &hv, B, H, G, dk, dv, cf32(g), static_cast<float*>(ptr_or_null(state)), state.size(0), cptr(l),
                            index_size(l), float(scale), m16(out), current_stream()),
            op);
  bump_write_epoch(state);
  state.unsafeGetTensorImpl()->bump_version();
  return out;
}

at::Tensor token_distill(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& teacher, double tau,
                         const std::optional<at::Tensor>& weight, int64_t reduction) {
  const char* op = "distill_loss";
  no_tangents(op, {&logits, &teacher});
  if (weight.has_value()) no_tangents(op, {&*weight});
  check_logits(op, logits);
  index_bytes(ids, op, "teacher_ids");
  float_code(teacher, op, "teacher_logits");
  check_tau(op, tau);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK(ids.dim() == logits.dim() && ids.sizes().slice(0, ids.dim() - 1) == lead && ids.sizes() == teacher.sizes(),
              op, ": teacher_ids and teacher_logits must be [..., k] beside logits ", logits.sizes(), ", got ", ids.sizes(),
              " and ", teacher.sizes());
  TORCH_CHECK(ids.size(-1) >= 1 && ids.size(-1) <= 1024, op, ": 1 to 1024 teacher entries a row, got ", ids.size(-1));
  if (weight.has_value())
    TORCH_CHECK(on_xdna(*weight) && weight->sizes() == lead, op, ": weight must be an xdna tensor of shape ", lead);
  if (tracked({&logits})) return DistillFn::apply(logits, ids, teacher, tau, weight, reduction);
  return distill_forward(logits, ids, teacher, tau, weight, reduction).loss;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> token_log_probs(const at::Tensor& logits,
                                                                           const at::Tensor& targets, int64_t top,
                                                                           double tau) {
  const char* op = "token_log_probs";
  no_tangents(op, {&logits});
  check_logits(op, logits);
  index_bytes(targets, op, "targets");
  check_tau(op, tau);
  TORCH_CHECK(targets.sizes() == logits.sizes().slice(0, logits.dim() - 1), op, ": targets must be ",
              logits.sizes().slice(0, logits.dim() - 1), ", got ", targets.sizes());
  TORCH_CHECK(top >= 0 && top <= 64 && top <= logits.size(-1), op, ": top_k must be 0 .. min(64, vocabulary), got ", top);
  if (tracked({&logits})) {
    const variable_list v = LogprobFn::apply(logits, targets, top, tau);
    return {v[0], v[1], v[2], v[3]};
  }
  const LogprobForward f = logprob_forward(logits, targets, top, tau);
  return {f.log_probs, f.entropy, f.top_log_probs, f.top_ids};
}

}  // namespace xdna_backend
