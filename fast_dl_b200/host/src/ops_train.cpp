// Training a model from a teacher and serving with a draft model: distillation, gated residual norms,
// verification of drafted tokens.  Each op checks, allocates, selects the device and calls the C ABI on the
// legacy default stream, like the rest of dl::ops.
#include <dl/ops/Ops.hpp>

#include <dl/core/CudaUtils.hpp>
#include <dl/ops/OpUtils.hpp>

#include <fdl_kernels.h>

#include <algorithm>
#include <stdexcept>
#include <string>

namespace dl::ops {

namespace {

[[noreturn]] void fail(const char* op, const std::string& what) { throw std::runtime_error(std::string(op) + ": " + what); }

int code_of(const Tensor& t, const char* op, const char* name) {
    if (t.dtype() == DType::Float32) return FDL_F32;
    if (t.dtype() == DType::Float16) return FDL_F16;
    fail(op, std::string(name) + " tensor must be float32 or float16");
}

// A tensor beside `like`, of this type and shape; `optional`: it may be undefined.
void check_beside(const Tensor& like, const Tensor& t, DType dtype, const Shape& shape, const char* op, const char* name,
                  bool optional = false) {
    if (optional && !t.defined()) return;
    check_defined(t, op, name);
    check_dtype(t, dtype, op, name);
    check_cuda(t, op, name);
    check_same_device(like, t, op, "input", name);
    if (t.shape() != shape) fail(op, std::string(name) + " tensor must have shape " + shape.str());
}

const float* floats(const Tensor& t) { return static_cast<const float*>(t.data()); }
const int64_t* ints(const Tensor& t) { return static_cast<const int64_t*>(t.data()); }

void check_distill(const Tensor& logits, const DistillTarget& d, const char* op) {
    check_defined(logits, op, "logits");
    check_rank(logits, 2, op, "logits");
    check_cuda(logits, op, "logits");
    code_of(logits, op, "logits");
    check_defined(d.index, op, "index");
    check_rank(d.index, 2, op, "index");
    const int64_t rows = logits.shape()[0], k = d.index.shape()[1];
    check_beside(logits, d.index, DType::Int64, Shape({rows, k}), op, "index");
    check_defined(d.teacher, op, "teacher");
    code_of(d.teacher, op, "teacher");
    check_beside(logits, d.teacher, d.teacher.dtype(), Shape({rows, k}), op, "teacher");
    check_beside(logits, d.teacher_lse, DType::Float32, Shape({rows}), op, "teacher_lse", true);
    check_beside(logits, d.row_weight, DType::Float32, Shape({rows}), op, "row_weight", true);
}

DistillLoss distill(const Tensor& logits, const DistillTarget& d, bool with_grad, const char* op) {
    check_distill(logits, d, op);
    const int64_t rows = logits.shape()[0], vocab = logits.shape()[1], k = d.index.shape()[1];
    const int type = code_of(logits, op, "logits"), teacher_type = code_of(d.teacher, op, "teacher");
    DistillLoss out;
    out.loss = Tensor(Shape({1}), DType::Float32, logits.device());
    out.row_loss = Tensor(Shape({rows}), DType::Float32, logits.device());
    out.row_stats = Tensor(Shape({rows, 2}), DType::Float32, logits.device());
    const float scale = 1.0f / static_cast<float>(rows);
    cuda::set_device(logits.device().index);
    int status;
    if (with_grad) {
        out.grad = Tensor(logits.shape(), logits.dtype(), logits.device());
        status = fdl_distill_topk_with_grad(logits.data(), vocab, type, d.teacher.data(), teacher_type, ints(d.index),
                                            floats(d.teacher_lse), floats(d.row_weight), rows, vocab, k, d.temperature, scale,
                                            static_cast<float*>(out.loss.data()), static_cast<float*>(out.row_loss.data()),
                                            static_cast<float*>(out.row_stats.data()), out.grad.data(), vocab, nullptr);
    } else {
        status = fdl_distill_topk(logits.data(), vocab, type, d.teacher.data(), teacher_type, ints(d.index), floats(d.teacher_lse),
                                  floats(d.row_weight), rows, vocab, k, d.temperature, scale,
                                  static_cast<float*>(out.loss.data()), static_cast<float*>(out.row_loss.data()),
                                  static_cast<float*>(out.row_stats.data()), nullptr);
    }
    cuda::check_fdl(status, (std::string(op) + " kernel launch failed").c_str());
    return out;
}

int kind_of(NormKind kind) { return kind == NormKind::None ? FDL_NORM_NONE : kind == NormKind::Rms ? FDL_NORM_RMS : FDL_NORM_LAYER; }
int act_of(GateAct act) { return act == GateAct::Plain ? FDL_GATE_PLAIN : act == GateAct::Sigmoid ? FDL_GATE_SIGMOID : FDL_GATE_TANH; }

// h is [rows, cols] and the parameters fit it.
void check_norm(const Tensor& h, const NormResidualParams& p, const char* op) {
    check_defined(h, op, "block");
    check_rank(h, 2, op, "block");
    check_cuda(h, op, "block");
    code_of(h, op, "block");
    const Shape col({h.shape()[1]});
    check_beside(h, p.post_gamma, DType::Float32, col, op, "post_gamma", true);
    check_beside(h, p.post_beta, DType::Float32, col, op, "post_beta", true);
    check_beside(h, p.pre_gamma, DType::Float32, col, op, "pre_gamma", true);
    check_beside(h, p.pre_beta, DType::Float32, col, op, "pre_beta", true);
    if (p.gate.defined()) {
        check_rank(p.gate, 2, op, "gate");
        check_beside(h, p.gate, h.dtype(), Shape({p.gate.shape()[0], h.shape()[1]}), op, "gate");
        if (h.shape()[0] % p.gate.shape()[0] != 0) fail(op, "gate rows must divide the rows");
    }
}

int64_t gate_rows(const NormResidualParams& p) { return p.gate.defined() ? p.gate.shape()[0] : 0; }

Tensor like(const Tensor& t) { return t.defined() ? Tensor(t.shape(), t.dtype(), t.device()) : Tensor(); }

}  // namespace

DistillLoss distill_topk(const Tensor& logits, const DistillTarget& target) {
    return distill(logits, target, false, "distill_topk");
}

DistillLoss distill_topk_with_grad(const Tensor& logits, const DistillTarget& target) {
    return distill(logits, target, true, "distill_topk_with_grad");
}

Tensor distill_topk_backward(const Tensor& logits, const DistillTarget& d, const Tensor& row_stats, const Tensor& grad_loss) {
    const char* op = "distill_topk_backward";
    check_distill(logits, d, op);
    const int64_t rows = logits.shape()[0], vocab = logits.shape()[1];
    check_beside(logits, row_stats, DType::Float32, Shape({rows, 2}), op, "row_stats");
    check_beside(logits, grad_loss, DType::Float32, Shape({1}), op, "grad_loss", true);
    Tensor grad(logits.shape(), logits.dtype(), logits.device());
    cuda::set_device(logits.device().index);
    cuda::check_fdl(fdl_distill_topk_backward(logits.data(), vocab, code_of(logits, op, "logits"), d.teacher.data(),
                                              code_of(d.teacher, op, "teacher"), ints(d.index), floats(d.teacher_lse),
                                              floats(d.row_weight), floats(row_stats), floats(grad_loss), rows, vocab,
                                              d.index.shape()[1], d.temperature, 1.0f / static_cast<float>(rows), grad.data(),
                                              vocab, nullptr),
                    "distill_topk_backward kernel launch failed");
    return grad;
}

NormResidual norm_residual(const Tensor& x, const Tensor& h, const NormResidualParams& p) {
    const char* op = "norm_residual";
    check_norm(h, p, op);
    check_beside(h, x, h.dtype(), h.shape(), op, "residual");
    const int64_t rows = h.shape()[0], cols = h.shape()[1];
    NormResidual out;
    out.y = Tensor(x.shape(), x.dtype(), x.device());
    if (p.pre != NormKind::None) out.n = Tensor(x.shape(), x.dtype(), x.device());
    out.stats = Tensor(Shape({rows, 4}), DType::Float32, x.device());
    cuda::set_device(x.device().index);
    cuda::check_fdl(fdl_norm_residual(x.data(), h.data(), p.gate.data(), gate_rows(p), act_of(p.gate_act), kind_of(p.post),
                                      floats(p.post_gamma), floats(p.post_beta), kind_of(p.pre), floats(p.pre_gamma),
                                      floats(p.pre_beta), out.y.data(), out.n.data(), static_cast<float*>(out.stats.data()), rows,
                                      cols, p.residual_scale, p.block_scale, p.eps, code_of(x, op, "residual"), nullptr),
                    "norm_residual kernel launch failed");
    return out;
}

NormResidualGrads norm_residual_backward(const Tensor& dy, const Tensor& dn, const NormResidual& f, const Tensor& h,
                                         const NormResidualParams& p) {
    const char* op = "norm_residual_backward";
    check_norm(h, p, op);
    if (!dy.defined() && !dn.defined()) fail(op, "a gradient of y or of n is needed");
    check_beside(h, dy, h.dtype(), h.shape(), op, "dy", true);
    check_beside(h, dn, h.dtype(), h.shape(), op, "dn", true);
    check_beside(h, f.y, h.dtype(), h.shape(), op, "y");
    const int64_t rows = h.shape()[0], cols = h.shape()[1];
    check_beside(h, f.stats, DType::Float32, Shape({rows, 4}), op, "stats");
    NormResidualGrads g;
    g.x = like(h);
    g.h = like(h);
    g.gate = like(p.gate);
    g.post_gamma = like(p.post_gamma);
    g.post_beta = like(p.post_beta);
    g.pre_gamma = like(p.pre_gamma);
    g.pre_beta = like(p.pre_beta);
    cuda::set_device(h.device().index);
    const std::size_t bytes = fdl_norm_residual_backward_scratch_bytes(rows, cols, gate_rows(p));
    Tensor scratch(Shape({static_cast<int64_t>(std::max<std::size_t>(bytes, 1) + 3) / 4}), DType::Float32, h.device());
    cuda::check_fdl(fdl_norm_residual_backward(dy.data(), dn.data(), f.y.data(), h.data(), floats(f.stats), p.gate.data(),
                                               gate_rows(p), act_of(p.gate_act), kind_of(p.post), floats(p.post_gamma),
                                               floats(p.post_beta), kind_of(p.pre), floats(p.pre_gamma), g.x.data(), g.h.data(),
                                               g.gate.data(), static_cast<float*>(g.post_gamma.data()),
                                               static_cast<float*>(g.post_beta.data()), static_cast<float*>(g.pre_gamma.data()),
                                               static_cast<float*>(g.pre_beta.data()), rows, cols, p.residual_scale,
                                               p.block_scale, code_of(h, op, "block"), scratch.data(), scratch.nbytes(), nullptr),
                    "norm_residual_backward kernel launch failed");
    return g;
}

VerifiedDraft verify_draft(const Tensor& target, const Tensor& draft, const Tensor& draft_tokens, const Tensor& accept_u,
                           const Tensor& sample_u, const Tensor& draft_len) {
    const char* op = "verify_draft";
    check_defined(target, op, "target");
    check_rank(target, 3, op, "target");
    check_cuda(target, op, "target");
    const int type = code_of(target, op, "target");
    const int64_t batch = target.shape()[0], drafted = target.shape()[1] - 1, vocab = target.shape()[2];
    // (a tensor without elements is undefined: with nothing drafted there are no tokens and no accept_u)
    check_beside(target, draft, target.dtype(), Shape({batch, drafted, vocab}), op, "draft", true);
    check_beside(target, draft_tokens, DType::Int64, Shape({batch, drafted}), op, "draft_tokens", drafted == 0);
    check_beside(target, accept_u, DType::Float32, Shape({batch, drafted}), op, "accept_u", drafted == 0);
    check_beside(target, sample_u, DType::Float32, Shape({batch}), op, "sample_u");
    check_beside(target, draft_len, DType::Int64, Shape({batch}), op, "draft_len", true);
    VerifiedDraft out;
    out.tokens = Tensor(Shape({batch, drafted + 1}), DType::Int64, target.device());
    out.accepted = Tensor(Shape({batch}), DType::Int64, target.device());
    cuda::set_device(target.device().index);
    cuda::check_fdl(fdl_verify_draft(target.data(), (drafted + 1) * vocab, vocab, draft.data(), drafted * vocab, vocab, type,
                                     ints(draft_tokens), ints(draft_len), floats(accept_u), floats(sample_u), batch, drafted, vocab,
                                     static_cast<int64_t*>(out.tokens.data()), static_cast<int64_t*>(out.accepted.data()), nullptr),
                    "verify_draft kernel launch failed");
    return out;
}

}  // namespace dl::ops
