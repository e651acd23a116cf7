"""A draft model as a user runs it: its residual block, head, distillation loss and all gradients, a step on its
weights, and the verification of what it drafts -- through the Python binding against 64-bit autograd, and
through dl::ops (the C++ test program).

Tolerances: each operator's own tests hold it to a derived bound of a few hundred half steps of 2^-24 on the sum of
absolute values; through the chain (two matrix products of 32-bit floats with at most 1000 terms, the norms, the
softmax) the gradients are compared at 2^-13 of the largest entry of each, i.e. 2048 half steps."""
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
pytestmark = pytest.mark.gpu


def test_host_library(cuda):
    exe = ROOT / "fast_dl_b200" / "lib" / "draft_model_test"
    assert exe.exists(), "run python -m fast_dl_b200.build core"
    proc = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120, cwd=str(ROOT))
    assert proc.returncode == 0 and "not passed" not in proc.stdout, proc.stdout + proc.stderr


class Draft(torch.autograd.Function):
    """block -> n -> logits -> loss, with the framework's gradients."""

    @staticmethod
    def forward(ctx, fdl, x, h, gate, post_gamma, pre_gamma, head, teacher, index, weight):
        y, n, stats = fdl.norm_residual(x, h, gate=gate, gate_act=fdl.GATE_TANH, post_gamma=post_gamma, pre_gamma=pre_gamma)
        logits = n @ head
        loss, _, row_stats = fdl.distill_topk(logits, teacher, index, row_weight=weight)
        ctx.fdl = fdl
        ctx.save_for_backward(y, n, stats, h, gate, post_gamma, pre_gamma, head, logits, row_stats, teacher, index, weight)
        return loss

    @staticmethod
    def backward(ctx, grad_loss):
        fdl = ctx.fdl
        y, n, stats, h, gate, post_gamma, pre_gamma, head, logits, row_stats, teacher, index, weight = ctx.saved_tensors
        dz = fdl.distill_topk_backward(logits, teacher, index, row_stats, row_weight=weight, grad_loss=grad_loss.contiguous())
        g = fdl.norm_residual_backward(None, dz @ head.t(), y, h, stats, gate=gate, gate_act=fdl.GATE_TANH, post_gamma=post_gamma,
                                       pre_gamma=pre_gamma)
        return (None, g["x"], g["h"], g["gate"], g["post_gamma"], g["pre_gamma"], n.t() @ dz, None, None, None)


def reference(x, h, gate, post_gamma, pre_gamma, head, teacher, index, weight):
    def rms(v, g):
        return v / torch.sqrt(v.pow(2).mean(1, keepdim=True) + 1e-5) * g

    y = x + torch.tanh(gate).repeat_interleave(x.shape[0] // gate.shape[0], 0) * rms(h, post_gamma)
    logq = torch.log_softmax(rms(y, pre_gamma) @ head, 1)
    counts = index >= 0
    p = torch.softmax(teacher.masked_fill(~counts, -float("inf")), 1)
    each = torch.where(counts, p * (p.clamp(min=1e-300).log() - logq.gather(1, index.clamp(min=0))), torch.zeros_like(p)).sum(1)
    return (weight * each).mean().reshape(1)


@pytest.mark.parametrize("rows,cols,vocab,k,gates", [(12, 64, 1000, 8, 3), (33, 257, 997, 16, 1), (500, 128, 9001, 32, 5)])
def test_training_step(fdl, cuda, rows, cols, vocab, k, gates):
    g = torch.Generator().manual_seed(rows)
    leaves = [torch.randn(rows, cols, generator=g), torch.randn(rows, cols, generator=g), torch.randn(gates, cols, generator=g),
              1 + 0.1 * torch.randn(cols, generator=g), 1 + 0.1 * torch.randn(cols, generator=g),
              torch.randn(cols, vocab, generator=g) / cols ** 0.5]
    teacher = (torch.randn(rows, k, generator=g) * 2).sort(1, descending=True).values
    index = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)])
    index[::3, k // 2:] = -1
    weight = (torch.arange(rows) % 5 != 4).float()
    tf32 = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        own = [t.cuda().requires_grad_() for t in leaves]
        loss = Draft.apply(fdl, *own, teacher.cuda(), index.cuda(), weight.cuda())
        (3.0 * loss).backward()
    finally:
        torch.backends.cuda.matmul.allow_tf32 = tf32
    exact = [t.double().requires_grad_() for t in leaves]
    want = reference(*exact, teacher.double(), index, weight.double())
    (3.0 * want).backward()
    assert abs(loss.item() - want.item()) <= 2.0 ** -13 * max(1.0, abs(want.item()))
    for a, b in zip(own, exact):
        assert (a.grad.double().cpu() - b.grad).abs().max() <= 2.0 ** -13 * b.grad.abs().max()


def test_drafts_and_their_verification(fdl, cuda):
    """Softmax rows of a draft head and a target head, drafted tokens, verification: accepted tokens stand where
    they were drafted, and the rest of a row is -1."""
    batch, drafted, cols, vocab = 40, 4, 96, 3001
    g = torch.Generator(device="cuda").manual_seed(3)
    hidden = torch.randn(batch * (drafted + 1), cols, device="cuda", generator=g)
    head = torch.randn(cols, vocab, device="cuda", generator=g) / 4
    y, n, _ = fdl.norm_residual(hidden, hidden)
    target = fdl.softmax_rows(n @ head).view(batch, drafted + 1, vocab)
    noisy = head + 0.05 * torch.randn(cols, vocab, device="cuda", generator=g)
    draft = fdl.softmax_rows((n @ noisy).contiguous()).view(batch, drafted + 1, vocab)[:, :drafted]
    tokens = torch.multinomial(draft.reshape(-1, vocab), 1, generator=g).view(batch, drafted)
    accept = torch.rand(batch, drafted, device="cuda", generator=g)
    out, count = fdl.verify_draft(target, tokens, accept, torch.rand(batch, device="cuda", generator=g), draft=draft)
    ratio = target[:, :drafted].gather(2, tokens[..., None])[..., 0] > accept * draft.gather(2, tokens[..., None])[..., 0]
    assert torch.equal(count, ratio.long().cumprod(1).sum(1)) and 0 < count.sum() < batch * drafted
    for b in range(batch):
        c = count[b].item()
        row = out[b].tolist()
        assert row[:c] == tokens[b, :c].tolist() and 0 <= row[c] < vocab and row[c + 1:] == [-1] * (drafted - c)
        if c < drafted:  # what was put in its place had more of the target than of the draft
            assert target[b, c, row[c]] > draft[b, c, row[c]]
