// dl::ops -- tensor-level operations.  Names, argument meaning, defaults and error strings
// follow fast_dl's include/dl/ops/*.hpp; each op validates, allocates the result, selects the
// device, calls dl::kernels / the C ABI and checks the launch, in the order of
// run_elementwise (src/ops/Elementwise.cpp:36-50).
//
// Extensions, all API-compatible with what was there:
//   * add/sub/mul/div (and operators) accept NumPy-broadcastable shapes; equal shapes behave
//     exactly as before, non-broadcastable ones raise the reference's
//     "... tensors must have the same shape" error;
//   * sum / mean / max / argmax along an axis, full sum (fast_dl has none, FUTURE_WORK.md:84-92
//     gives the pattern new ops should follow);
//   * layernorm with gamma and beta; mul_add_relu; linear with a fused ReLU epilogue;
//   * training a model from a teacher and serving with a draft model: distill_topk, norm_residual
//     (both with their gradients) and verify_draft.
#pragma once

#include <cstdint>

#include <dl/tensor/Tensor.hpp>

namespace dl::ops {

// ---- Elementwise.hpp ----
Tensor add(const Tensor& a, const Tensor& b);
Tensor sub(const Tensor& a, const Tensor& b);
Tensor mul(const Tensor& a, const Tensor& b);
Tensor div(const Tensor& a, const Tensor& b);
/// relu(a*b + c) in one pass, bit-identical to relu(add(mul(a, b), c)).
Tensor mul_add_relu(const Tensor& a, const Tensor& b, const Tensor& c);

// ---- Activation.hpp ----
Tensor relu(const Tensor& a);
Tensor leaky_relu(const Tensor& a, float alpha = 0.01f);
Tensor gelu(const Tensor& a);
Tensor sigmoid(const Tensor& a);
Tensor tanh(const Tensor& a);

// ---- Softmax.hpp / LayerNorm.hpp (rank-2 inputs, along the last axis) ----
Tensor softmax(const Tensor& input);
Tensor layernorm(const Tensor& input, float eps = 1.0e-5f);
/// (x - mean) * rstd * gamma + beta; gamma and beta have shape [cols].
Tensor layernorm(const Tensor& input, const Tensor& gamma, const Tensor& beta, float eps = 1.0e-5f);

// ---- reductions (new).  `axis` may be negative; the reduced axis is removed. ----
/// Sum of all elements, shape {1} (fast_dl has no rank-0 tensors: src/core/Shape.cpp:17-20).
Tensor sum(const Tensor& input);
Tensor sum(const Tensor& input, int axis);
Tensor mean(const Tensor& input, int axis);
Tensor max(const Tensor& input, int axis);
/// Int64 indices of the maximum along the LAST axis; ties go to the lowest index.
Tensor argmax(const Tensor& input, int axis);

// ---- Matmul.hpp / Linear.hpp / CrossEntropy.hpp ----
Tensor matmul(const Tensor& a, const Tensor& b);
Tensor linear(const Tensor& input, const Tensor& weight, const Tensor& bias);
/// relu(linear(...)) with bias add and ReLU fused into one pass over the GEMM output.
Tensor linear_relu(const Tensor& input, const Tensor& weight, const Tensor& bias);
Tensor cross_entropy(const Tensor& logits, const Tensor& labels);

// ---- training a model from a teacher, serving with a draft model (new) ----
// Tensors are Float32 or Float16 (weights, statistics, losses and random numbers Float32, indices and
// tokens Int64); an undefined tensor stands for one that is not given.  The formulas are those of the
// entry points in fdl_kernels.h.

struct DistillTarget {
    Tensor teacher;      ///< [rows, k]: the teacher's highest logits
    Tensor index;        ///< [rows, k] Int64: their columns; outside [0, vocab): padding
    Tensor teacher_lse;  ///< [rows] or undefined: log-sum-exp of all its logits / temperature
    Tensor row_weight;   ///< [rows] or undefined (1)
    float temperature = 1.0f;
};
struct DistillLoss {
    Tensor loss;       ///< {1}: the weighted mean over the rows
    Tensor row_loss;   ///< [rows]
    Tensor row_stats;  ///< [rows, 2], for the backward call
    Tensor grad;       ///< [rows, vocab]: distill_topk_with_grad only
};
/// Mean over the rows of the divergence of softmax(logits / T) from the teacher's distribution.
DistillLoss distill_topk(const Tensor& logits, const DistillTarget& target);
/// The same with its gradient, in one pass over the logits.
DistillLoss distill_topk_with_grad(const Tensor& logits, const DistillTarget& target);
/// The gradient of grad_loss * loss (grad_loss {1}, or undefined for 1) from the forward call's row_stats.
Tensor distill_topk_backward(const Tensor& logits, const DistillTarget& target, const Tensor& row_stats,
                             const Tensor& grad_loss = Tensor());

enum class NormKind { None, Rms, Layer };
enum class GateAct { Plain, Sigmoid, Tanh };
struct NormResidualParams {
    NormKind post = NormKind::Rms, pre = NormKind::Rms;
    Tensor post_gamma, post_beta, pre_gamma, pre_beta;  ///< [cols] or undefined
    Tensor gate;                                        ///< [gate_rows, cols] or undefined; gate_rows divides rows
    GateAct gate_act = GateAct::Plain;
    float residual_scale = 1.0f, block_scale = 1.0f, eps = 1.0e-5f;
};
struct NormResidual {
    Tensor y;      ///< residual_scale * x + block_scale * act(gate) * norm_post(h)
    Tensor n;      ///< norm_pre(y); undefined with NormKind::None
    Tensor stats;  ///< [rows, 4], for the backward call
};
NormResidual norm_residual(const Tensor& x, const Tensor& h, const NormResidualParams& params);
/// Gradients of all that `params` defines; dy or dn may be undefined (no gradient there).
struct NormResidualGrads {
    Tensor x, h, gate, post_gamma, post_beta, pre_gamma, pre_beta;
};
NormResidualGrads norm_residual_backward(const Tensor& dy, const Tensor& dn, const NormResidual& forward, const Tensor& h,
                                         const NormResidualParams& params);

struct VerifiedDraft {
    Tensor tokens;    ///< [batch, drafted + 1] Int64: those that stand, the next one, then -1
    Tensor accepted;  ///< [batch] Int64
};
/// target [batch, drafted + 1, vocab] and draft [batch, drafted, vocab] (or undefined) are probabilities,
/// accept_u [batch, drafted] and sample_u [batch] numbers in [0, 1), draft_len [batch] Int64 or undefined.
VerifiedDraft verify_draft(const Tensor& target, const Tensor& draft, const Tensor& draft_tokens, const Tensor& accept_u,
                           const Tensor& sample_u, const Tensor& draft_len = Tensor());

}  // namespace dl::ops

namespace dl {
Tensor operator+(const Tensor& a, const Tensor& b);
Tensor operator-(const Tensor& a, const Tensor& b);
Tensor operator*(const Tensor& a, const Tensor& b);
Tensor operator/(const Tensor& a, const Tensor& b);
}  // namespace dl
