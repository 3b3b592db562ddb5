// Host side of the token-model operators (xdna_train/tokens.py): checks, workspaces, C-ABI
// calls and autograd nodes of the embedding, the gated feed-forward, the distillation loss
// and the token log probabilities (csrc/embed.hip, gated.hip, vocab.hip).  No call reads
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
