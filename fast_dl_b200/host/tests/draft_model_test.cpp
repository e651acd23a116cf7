// A draft model through dl::ops, in the style of the reference's own tests: its residual block, its head, the
// distillation loss and gradients, and the verification of what it drafts, against CPU loops in double.
// Needs a GPU (device 0).
#include <dl/dl.hpp>

#include <algorithm>
#include <cmath>
#include <iostream>
#include <random>
#include <string>
#include <vector>

namespace {

int g_failed = 0;

void report(const char* name, bool ok) {
    std::cout << name << " : " << (ok ? "passed" : "not passed") << "\n";
    if (!ok) ++g_failed;
}

std::vector<float> randoms(std::size_t n, unsigned seed, float lo, float hi) {
    std::mt19937 gen(seed);
    std::uniform_real_distribution<float> dist(lo, hi);
    std::vector<float> v(n);
    for (float& x : v) x = dist(gen);
    return v;
}

// |a - b| <= tol * max(1, |b|): sums here have at most a few hundred terms of size ten in 32 bits.
bool close(const std::vector<float>& a, const std::vector<double>& b, double tol = 2e-5) {
    if (a.size() != b.size()) return false;
    for (std::size_t i = 0; i < a.size(); ++i) {
        if (!(std::fabs(a[i] - b[i]) <= tol * std::max(1.0, std::fabs(b[i])))) return false;
    }
    return true;
}

template <class Fn>
bool throws_with(Fn fn, const std::string& text) {
    try {
        fn();
    } catch (const std::runtime_error& e) {
        return std::string(e.what()).find(text) != std::string::npos;
    }
    return false;
}

}  // namespace

int main() {
    const dl::Device dev(dl::DeviceType::CUDA, 0);
    const int64_t R = 6, C = 40, V = 97, K = 5;
    const double eps = 1e-5;
    const auto x = randoms(R * C, 1, -2, 2), h = randoms(R * C, 2, -1, 3), g1 = randoms(C, 3, 0.5f, 1.5f), g2 = randoms(C, 4, 0.5f, 1.5f),
               gate = randoms(2 * C, 5, -1, 2), wt = randoms(C * V, 6, -0.5f, 0.5f), bias = randoms(V, 7, -0.1f, 0.1f);
    const auto from = [&](const std::vector<float>& v, const dl::Shape& s) { return dl::Tensor::from_host<float>(v, s, dev); };
    dl::Tensor tx = from(x, dl::Shape({R, C})), th = from(h, dl::Shape({R, C}));
    dl::ops::NormResidualParams p;
    p.post_gamma = from(g1, dl::Shape({C}));
    p.pre_gamma = from(g2, dl::Shape({C}));
    p.gate = from(gate, dl::Shape({2, C}));
    p.gate_act = dl::ops::GateAct::Sigmoid;
    p.block_scale = 0.5f;

    // block -> head
    dl::ops::NormResidual block = dl::ops::norm_residual(tx, th, p);
    std::vector<double> y(R * C), n(R * C);
    for (int64_t r = 0; r < R; ++r) {
        double q = 0, s = 0;
        for (int64_t c = 0; c < C; ++c) q += static_cast<double>(h[r * C + c]) * h[r * C + c];
        const double r1 = 1 / std::sqrt(q / C + eps);
        for (int64_t c = 0; c < C; ++c) {
            const double a = 1 / (1 + std::exp(-static_cast<double>(gate[(r / 3) * C + c])));
            y[r * C + c] = x[r * C + c] + 0.5 * a * h[r * C + c] * r1 * g1[c];
            s += y[r * C + c] * y[r * C + c];
        }
        const double r2 = 1 / std::sqrt(s / C + eps);
        for (int64_t c = 0; c < C; ++c) n[r * C + c] = y[r * C + c] * r2 * g2[c];
    }
    report("norm_residual", close(block.y.to_host<float>(), y) && close(block.n.to_host<float>(), n));
    dl::Tensor logits = dl::ops::linear(block.n, from(wt, dl::Shape({C, V})), from(bias, dl::Shape({V})));

    // the loss and its gradient, from the logits that the head gave
    std::vector<int64_t> index(R * K);
    for (int64_t i = 0; i < R * K; ++i) index[i] = (i * 37 + 11) % V;
    index[3 * K + 4] = -1;  // padding
    const auto teacher = randoms(R * K, 8, 0, 4);
    dl::ops::DistillTarget target;
    target.teacher = from(teacher, dl::Shape({R, K}));
    target.index = dl::Tensor::from_host<int64_t>(index, dl::Shape({R, K}), dev);
    target.temperature = 2.0f;
    const auto z = logits.to_host<float>();
    std::vector<double> want(R), grad(R * V);
    double mean = 0;
    for (int64_t r = 0; r < R; ++r) {
        double tsum = 0, zsum = 0;
        for (int64_t j = 0; j < K; ++j) tsum += index[r * K + j] < 0 ? 0 : std::exp(teacher[r * K + j] / 2.0);
        for (int64_t v = 0; v < V; ++v) zsum += std::exp(z[r * V + v] / 2.0);
        for (int64_t v = 0; v < V; ++v) grad[r * V + v] = std::exp(z[r * V + v] / 2.0) / zsum / (2.0 * R);
        for (int64_t j = 0; j < K; ++j) {
            if (index[r * K + j] < 0) continue;
            const double pj = std::exp(teacher[r * K + j] / 2.0) / tsum;
            want[r] += pj * (std::log(pj) - (z[r * V + index[r * K + j]] / 2.0 - std::log(zsum)));
            grad[r * V + index[r * K + j]] -= pj / (2.0 * R);
        }
        mean += want[r] / R;
    }
    dl::ops::DistillLoss loss = dl::ops::distill_topk(logits, target);
    dl::ops::DistillLoss both = dl::ops::distill_topk_with_grad(logits, target);
    report("distill_topk", close(loss.row_loss.to_host<float>(), want) && close(loss.loss.to_host<float>(), {mean}) &&
                               close(both.row_loss.to_host<float>(), want) && !loss.grad.defined());
    dl::Tensor back = dl::ops::distill_topk_backward(logits, target, loss.row_stats);
    report("distill_topk gradients", close(both.grad.to_host<float>(), grad, 1e-6) && close(back.to_host<float>(), grad, 1e-6));

    // through the head and the block: differences of the whole run's loss along the residual stream
    {
        std::vector<float> wtt(V * C);
        for (int64_t c = 0; c < C; ++c)
            for (int64_t v = 0; v < V; ++v) wtt[v * C + c] = wt[c * V + v];
        dl::Tensor dn = dl::ops::matmul(both.grad, from(wtt, dl::Shape({V, C})));
        dl::ops::NormResidualGrads g = dl::ops::norm_residual_backward(dl::Tensor(), dn, block, th, p);
        const auto run = [&](const std::vector<float>& at) {
            dl::ops::NormResidual b = dl::ops::norm_residual(from(at, dl::Shape({R, C})), th, p);
            dl::Tensor zz = dl::ops::linear(b.n, from(wt, dl::Shape({C, V})), from(bias, dl::Shape({V})));
            double s = 0;
            for (float v : dl::ops::distill_topk(zz, target).row_loss.to_host<float>()) s += v / R;
            return s;
        };
        const auto gx = g.x.to_host<float>();
        const auto along = randoms(R * C, 9, -1, 1);
        const double step = 1.0 / 64;
        std::vector<float> up = x, down = x;
        double dot = 0;
        for (int64_t i = 0; i < R * C; ++i) {
            up[i] += static_cast<float>(step) * along[i];
            down[i] -= static_cast<float>(step) * along[i];
            dot += static_cast<double>(gx[i]) * along[i];
        }
        // third derivatives of order one: step^2 / 6 of them; losses are good to 1e-5
        report("gradient of the whole run against differences",
               std::fabs((run(up) - run(down)) / (2 * step) - dot) < step * step + 1e-5 / step);
        report("gradients of all parameters", g.gate.defined() && g.post_gamma.defined() && g.pre_gamma.defined() &&
                                                  !g.post_beta.defined() && g.gate.shape() == p.gate.shape());
    }

    // verification: the target's rows stand for both models (everything stands), then a draft that is wrong
    {
        const int64_t B = 2, D = 2;
        dl::Tensor probs = dl::ops::softmax(logits).reshaped(dl::Shape({B, D + 1, V}));
        const auto pr = probs.to_host<float>();
        std::vector<int64_t> drawn(B * D);
        std::vector<float> qv(B * D * V, 0.0f), accept(B * D, 0.25f);
        for (int64_t b = 0; b < B; ++b) {
            for (int64_t i = 0; i < D; ++i) {
                drawn[b * D + i] = (b * 7 + i * 3) % V;
                for (int64_t v = 0; v < V; ++v) qv[(b * D + i) * V + v] = pr[(b * (D + 1) + i) * V + v];
            }
        }
        accept[1 * D + 1] = 1.0f;  // falls: p < 1 * p does not hold, and nothing is left of p - q: the row itself
        dl::ops::VerifiedDraft got = dl::ops::verify_draft(
            probs, from(qv, dl::Shape({B, D, V})), dl::Tensor::from_host<int64_t>(drawn, dl::Shape({B, D}), dev),
            from(accept, dl::Shape({B, D})), from({0.5f, 0.5f}, dl::Shape({B})));
        const auto tokens = got.tokens.to_host<int64_t>(), count = got.accepted.to_host<int64_t>();
        const auto median = [&](int64_t row) {
            double total = 0, sum = 0;
            for (int64_t v = 0; v < V; ++v) total += pr[row * V + v];
            for (int64_t v = 0; v < V; ++v) {
                sum += pr[row * V + v];
                if (sum > 0.5 * total) return v;
            }
            return int64_t{-1};
        };
        report("verify_draft", count == std::vector<int64_t>({2, 1}) &&
                                   tokens == std::vector<int64_t>({drawn[0], drawn[1], median(2), drawn[2], median(4), -1}));
    }

    {   // refusals
        dl::ops::DistillTarget bad = target;
        bad.index = dl::Tensor();
        report("distill_topk without an index", throws_with([&] { dl::ops::distill_topk(logits, bad); }, "distill_topk: index tensor is not defined"));
        bad = target;
        bad.row_weight = from(teacher, dl::Shape({R, K}));
        report("distill_topk with a weight of another shape", throws_with([&] { dl::ops::distill_topk(logits, bad); }, "row_weight tensor must have shape"));
        bad = target;
        bad.temperature = 0.0f;
        report("distill_topk at temperature 0", throws_with([&] { dl::ops::distill_topk(logits, bad); }, "invalid argument"));
        dl::ops::NormResidualParams q = p;
        q.gate = from(randoms(4 * C, 1, 0, 1), dl::Shape({4, C}));
        report("a gate whose rows do not divide", throws_with([&] { dl::ops::norm_residual(tx, th, q); }, "gate rows must divide the rows"));
        report("norm_residual_backward without a gradient",
               throws_with([&] { dl::ops::norm_residual_backward(dl::Tensor(), dl::Tensor(), block, th, p); }, "is needed"));
        report("verify_draft on a matrix", throws_with([&] { dl::ops::verify_draft(logits, dl::Tensor(), target.index, logits, logits); },
                                                       "verify_draft: target tensor has incorrect rank"));
    }

    std::cout << "draft_model_test : " << (g_failed == 0 ? "passed" : "not passed") << "\n";
    return g_failed == 0 ? 0 : 1;
}
