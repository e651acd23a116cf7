"""Distillation from a teacher's top logits against the definition in 64 bits.

Tolerances, derived before the first run.  A step of half a unit is eps/2 relative (f32 2^-24, f16
2^-11, bf16 2^-8).  The sum S of the exponentials: each term carries 2^-22 (the hardware's exp2) and an
exponent off by 3 roundings of its size, on average at most log2(vocab) -- 3 ln 2 * 18 * 2^-24 -- and
the additions at most ADDS * 2^-24, ADDS being the longest chain of additions (a thread's share of
the row, at least 128 threads on it, and 64 for the tree).  That is `rel_sum` below.  A teacher
probability carries the same kinds of error on at most 1024 terms (`REL_P`, 2^-18).  Then
  |d row_loss| <= P rel_sum + sum p |log p - log q| REL_P + 2^-24 |row_loss|   (differences are taken in 64 bits)
  |d grad_v|   <= |coef| (P q_v (rel_sum + 2^-22 + 3 |log2 q_v| 2^-24 + 2^-21) + p_v REL_P) + eps/2 |grad_v| + the
                  smallest step of the type.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -24, "bf16": 2.0 ** -126}
REL_P = 2.0 ** -18


def definition(z, t, index, lse, weight, temperature, scale):
    """row_loss, loss, grad, and what the tolerances need, in 64 bits (CPU)."""
    z, t = z.double().cpu() / temperature, t.double().cpu() / temperature
    index = index.cpu()
    rows, vocab = z.shape
    weight = torch.ones(rows, dtype=torch.float64) if weight is None else weight.double().cpu()
    counts = (index >= 0) & (index < vocab) & (t > -math.inf)
    live = counts.any(1) & (weight != 0)
    row_loss = torch.zeros(rows, dtype=torch.float64)
    spread = torch.zeros(rows, dtype=torch.float64)
    mass = torch.zeros(rows, dtype=torch.float64)
    grad, q_all, p_all = (torch.zeros(rows, vocab, dtype=torch.float64) for _ in range(3))
    for r in range(rows):
        if not live[r]:
            continue
        at = index[r][counts[r]]
        logp = t[r][counts[r]]
        logp = logp - (torch.logsumexp(logp, 0) if lse is None else lse[r].double().cpu())
        p = logp.exp()
        logq = torch.log_softmax(z[r], 0)
        delta = torch.where(p > 0, logp - logq[at], torch.zeros_like(p))
        row_loss[r] = (p * delta).sum()
        spread[r] = (p * delta.abs()).sum()
        mass[r] = p.sum()
        q_all[r] = logq.exp()
        p_all[r].index_add_(0, at, p)
        grad[r] = scale * weight[r] / temperature * (mass[r] * q_all[r] - p_all[r])
    loss = scale * (weight * row_loss)[live].sum()
    coef = torch.where(live, (scale * weight / temperature).abs(), torch.zeros_like(weight))
    return row_loss, loss, grad, dict(spread=spread, mass=mass, q=q_all, p=p_all, coef=coef, live=live)


def rel_sum(vocab):
    return 2.0 ** -22 + (3 * math.log(2) * 18 + math.ceil(vocab / 128) + 64) * 2.0 ** -24


def check_loss(row_loss, loss, want_rows, want, info, vocab, weight, scale):
    tol = info["mass"] * rel_sum(vocab) + info["spread"] * REL_P + 2.0 ** -24 * want_rows.abs()
    off = (row_loss.double().cpu() - want_rows).abs()
    assert bool((off <= tol).all()), (off - tol).max()
    w = torch.ones_like(tol) if weight is None else weight.double().cpu().abs()
    assert abs(loss.item() - want.item()) <= abs(scale) * (w * tol).sum().item() + 2.0 ** -24 * abs(want.item())


def check_grad(grad, want, info, vocab, kind):
    q, p = info["q"], info["p"]
    size = torch.where(q > 0, -torch.log2(q.clamp(min=1e-300)), torch.zeros_like(q))
    each = rel_sum(vocab) + 2.0 ** -22 + 3 * size * 2.0 ** -24 + 2.0 ** -21
    tol = info["coef"][:, None] * (info["mass"][:, None] * q * each + p * REL_P) + HALF[kind] * want.abs() + TINY[kind]
    off = (grad.double().cpu() - want).abs()
    assert bool((off <= tol).all()), (off - tol).max()


def make(rows, vocab, k, kind, seed=0, stride=None, tail=False, teacher_kind=None, repeat=False):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, stride or vocab, generator=g) * 3
    index = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)])
    if repeat and k > 1:
        index[:, -1] = index[:, 0]
    t = (torch.randn(rows, k, generator=g) * 2 + 6).sort(1, descending=True).values
    for r in range(rows):
        z[r, index[r]] += 0.6 * t[r]
    lse = torch.logsumexp(t, 1) + torch.rand(rows, generator=g) if tail else None
    kind_t = TYPES[teacher_kind or kind]
    return (z.to(TYPES[kind]).cuda()[:, :vocab], t.to(kind_t).cuda(), index.cuda(), None if lse is None else lse.cuda())


SHAPES = [(1, 1, 1), (1, 7, 3), (3, 33, 33), (5, 1000, 8), (2, 1027, 64), (9, 4099, 5), (4, 16384, 100), (2, 50257, 128),
          (1, 131072, 1024), (3, 100003, 17), (700, 129, 4), (2, 262145, 33), (160, 9001, 12), (400, 16385, 40), (90, 40000, 3), (2, 400001, 30),
          (1, 1000003, 5), (20, 1024, 9), (11, 2049, 1), (300, 512, 7)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,k", SHAPES)
def test_against_the_definition(fdl, cuda, rows, vocab, k, kind):
    for tail, temperature in ((False, 1.0), (True, 2.5)):
        z, t, index, lse = make(rows, vocab, k, kind, seed=rows + vocab, tail=tail)
        weight = torch.linspace(0.5, 2.0, rows).cuda() if tail else None
        scale = 1.0 / rows if not tail else 3.0
        want_rows, want, want_grad, info = definition(z, t, index, lse, weight, temperature, scale)
        more = dict(teacher_lse=lse, row_weight=weight, temperature=temperature, scale=scale)
        loss, row_loss, stats = fdl.distill_topk(z, t, index, **more)
        check_loss(row_loss, loss, want_rows, want, info, vocab, weight, scale)
        grad = fdl.distill_topk_backward(z, t, index, stats, **more)
        check_grad(grad, want_grad, info, vocab, kind)
        loss2, row_loss2, grad2 = fdl.distill_topk_with_grad(z, t, index, **more)
        check_loss(row_loss2, loss2, want_rows, want, info, vocab, weight, scale)
        check_grad(grad2, want_grad, info, vocab, kind)
        again = fdl.distill_topk_with_grad(z, t, index, **more)  # no order that depends on timing
        for a, b in zip((loss2, row_loss2, grad2), again):
            assert torch.equal(a, b)
    fdl.take_device_error()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_padding_entries_rows_and_weights(fdl, cuda, kind):
    """Padding entries hold NaN and infinities, left-out rows hold NaN logits: none of it reaches a result."""
    rows, vocab, k = 8, 1003, 12
    z, t, index, _ = make(rows, vocab, k, kind, seed=4)
    index[0, 5:] = -1
    t[0, 5:] = float("nan")
    index[1, 0] = vocab          # beyond the vocabulary
    t[1, 0] = float("inf")
    index[2] = -1                # nothing counts
    t[3] = -float("inf")         # nothing counts
    t[4, 3:] = -float("inf")
    t[5, 2:] = torch.finfo(t.dtype).min
    z[2], z[3], z[6] = float("nan"), float("nan"), float("nan")
    weight = torch.ones(rows).cuda()
    weight[6] = 0.0
    want_rows, want, want_grad, info = definition(z, t, index, None, weight, 1.0, 0.25)
    loss, row_loss, stats = fdl.distill_topk(z, t, index, row_weight=weight, scale=0.25)
    check_loss(row_loss, loss, want_rows, want, info, vocab, weight, 0.25)
    for grad in (fdl.distill_topk_backward(z, t, index, stats, row_weight=weight, scale=0.25),
                 fdl.distill_topk_with_grad(z, t, index, row_weight=weight, scale=0.25)[2]):
        check_grad(grad, want_grad, info, vocab, kind)
        for r in (2, 3, 6):
            assert row_loss[r].item() == 0.0 and not grad[r].any()
            assert not stats[r].any()


@pytest.mark.parametrize("kind,rows,vocab", [("f32", 1300, 4200), ("bf16", 1100, 8200), ("f16", 2500, 300), ("f32", 600, 20000)])
def test_many_rows_with_some_left_out(fdl, cuda, kind, rows, vocab):
    """Many rows a CTA, single rows and runs of rows left out, in each of the three calls."""
    k = 6
    z, t, index, _ = make(rows, vocab, k, kind, seed=rows)
    g = torch.Generator().manual_seed(5)
    weight = torch.ones(rows)
    weight[torch.rand(rows, generator=g) < 0.3] = 0.0
    weight[rows // 2:] = (torch.rand(rows - rows // 2, generator=g) < 0.2).float()
    weight = weight.cuda()
    index[::7] = -1
    z[::7] = float("nan")
    want_rows, want, want_grad, info = definition(z, t, index, None, weight, 1.0, 0.5)
    for _ in range(3):
        loss, row_loss, stats = fdl.distill_topk(z, t, index, row_weight=weight, scale=0.5)
        check_loss(row_loss, loss, want_rows, want, info, vocab, weight, 0.5)
        check_grad(fdl.distill_topk_backward(z, t, index, stats, row_weight=weight, scale=0.5), want_grad, info, vocab, kind)
        loss, row_loss, grad = fdl.distill_topk_with_grad(z, t, index, row_weight=weight, scale=0.5)
        check_loss(row_loss, loss, want_rows, want, info, vocab, weight, 0.5)
        check_grad(grad, want_grad, info, vocab, kind)
    fdl.take_device_error()


@pytest.mark.parametrize("kind,rows,vocab", [("f32", 601, 72472), ("bf16", 901, 100001), ("f32", 3000, 8200), ("f16", 5000, 1500)])
def test_many_runs_give_the_same_bits(fdl, cuda, kind, rows, vocab):
    """Chunks that are overwritten too early, or taken for another round's, would show in some runs of a hundred."""
    g = torch.Generator(device="cuda").manual_seed(2)
    z = torch.empty(rows, vocab, dtype=TYPES[kind], device="cuda").normal_(0.0, 2.0, generator=g)
    index = torch.randint(0, vocab, (rows, 24), device="cuda", generator=g)
    t = torch.randn(rows, 24, device="cuda", generator=g)
    loss, row_loss, stats = fdl.distill_topk(z, t, index)
    grad = fdl.distill_topk_backward(z, t, index, stats)
    both = fdl.distill_topk_with_grad(z, t, index)
    for _ in range(60):
        again = fdl.distill_topk(z, t, index)
        assert torch.equal(again[0], loss) and torch.equal(again[1], row_loss) and torch.equal(again[2], stats)
        assert torch.equal(fdl.distill_topk_backward(z, t, index, stats), grad)
        assert all(torch.equal(a, b) for a, b in zip(fdl.distill_topk_with_grad(z, t, index), both))


def test_no_row_at_all_counts_and_no_rows(fdl, cuda):
    z, t, index, _ = make(3, 100, 4, "f32")
    loss, row_loss, grad = fdl.distill_topk_with_grad(z, t, torch.full_like(index, -1))
    assert loss.item() == 0.0 and not row_loss.any() and not grad.any()
    empty = torch.empty(0, 100).cuda()
    loss, row_loss, grad = fdl.distill_topk_with_grad(empty, torch.empty(0, 4).cuda(), torch.empty(0, 4, dtype=torch.int64).cuda())
    assert loss.item() == 0.0 and row_loss.numel() == 0 and grad.shape == (0, 100)


@pytest.mark.parametrize("k", [2, 40, 1024])
def test_the_same_index_twice(fdl, cuda, k):
    vocab = 5000
    z, t, index, _ = make(4, vocab, k, "f32", seed=k, repeat=True)
    index[1, :] = 17            # every entry names one column
    want_rows, want, want_grad, info = definition(z, t, index, None, None, 1.0, 1.0)
    loss, row_loss, grad = fdl.distill_topk_with_grad(z, t, index, scale=1.0)
    check_loss(row_loss, loss, want_rows, want, info, vocab, None, 1.0)
    check_grad(grad, want_grad, info, vocab, "f32")


def test_masked_and_huge_student_logits(fdl, cuda):
    vocab, k = 2051, 6
    z, t, index, _ = make(6, vocab, k, "f32", seed=8)
    free = [v for v in range(vocab) if v not in index[0].tolist()]
    z[0, free[::2]] = -float("inf")                    # a masked half
    z[1] = torch.finfo(torch.float32).min              # the lowest value as a mask, but for the teacher's places
    z[1, index[1]] = t[1]
    z[2] += 30000.0                                    # a large offset cancels
    z[3, index[3, 0]] = -float("inf")                  # the teacher believes in it: infinite loss
    z[4] = -float("inf")                               # no distribution
    z[5, 77] = float("nan")
    loss, row_loss, grad = fdl.distill_topk_with_grad(z, t, index, scale=1.0)
    assert math.isnan(loss.item())
    want_rows, want, want_grad, info = definition(z[:3], t[:3], index[:3], None, None, 1.0, 1.0)
    check_loss(row_loss[:3], fdl.distill_topk(z[:3], t[:3], index[:3], scale=1.0)[0], want_rows, want, info, vocab, None, 1.0)
    check_grad(grad[:3], want_grad, info, vocab, "f32")
    assert row_loss[3].item() == math.inf and bool(torch.isfinite(grad[3]).all())
    assert math.isnan(row_loss[4].item()) and bool(torch.isnan(grad[4]).all())
    assert math.isnan(row_loss[5].item()) and bool(torch.isnan(grad[5]).all())


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab,stride", [(1000, 1003), (1003, 1008), (30001, 30016), (60001, 60002)])
def test_padded_rows_shifted_starts_and_in_place(fdl, cuda, kind, vocab, stride):
    rows, k = 5, 9
    z, t, index, _ = make(rows, vocab, k, kind, seed=vocab, stride=stride)
    want_rows, want, want_grad, info = definition(z, t, index, None, None, 1.0, 1.0)
    loss, row_loss, grad = fdl.distill_topk_with_grad(z, t, index, scale=1.0)
    check_loss(row_loss, loss, want_rows, want, info, vocab, None, 1.0)
    check_grad(grad, want_grad, info, vocab, kind)
    # a gradient with rows at another phase, its padding left as it was
    buf = torch.full((rows * (stride + 5) + 1,), 7.0, dtype=TYPES[kind], device="cuda")
    out = buf[1:].view(rows, stride + 5)[:, :vocab]
    fdl.distill_topk_with_grad(z, t, index, scale=1.0, out=out)
    check_grad(out, want_grad, info, vocab, kind)
    assert bool((buf[1:].view(rows, stride + 5)[:, vocab:] == 7.0).all()) and buf[0].item() == 7.0
    # logits off the 16-byte grid
    moved = torch.zeros(rows * vocab + 1, dtype=TYPES[kind], device="cuda")
    moved[1:] = z.reshape(-1)
    shifted = moved[1:].view(rows, vocab)
    check_grad(fdl.distill_topk_with_grad(shifted, t, index, scale=1.0)[2], want_grad, info, vocab, kind)
    # in place, from the one call and from the backward call
    stats = fdl.distill_topk(z, t, index, scale=1.0)[2]
    for one_call in (True, False):
        base = torch.full((rows, stride), 5.0, dtype=TYPES[kind], device="cuda")
        own = base[:, :vocab]
        own.copy_(z)
        if one_call:
            fdl.distill_topk_with_grad(own, t, index, scale=1.0, out=own)
        else:
            fdl.distill_topk_backward(own, t, index, stats, scale=1.0, out=own)
        check_grad(own, want_grad, info, vocab, kind)
        assert bool((base[:, vocab:] == 5.0).all())


def test_teacher_of_another_type_and_upstream_gradient(fdl, cuda):
    z, t, index, _ = make(4, 3001, 20, "bf16", teacher_kind="f32")
    up = torch.tensor([0.125], device="cuda")
    _, _, want_grad, info = definition(z, t, index, None, None, 1.0, 0.125)
    stats = fdl.distill_topk(z, t, index, scale=1.0)[2]
    grad = fdl.distill_topk_backward(z, t, index, stats, scale=1.0, grad_loss=up)
    check_grad(grad, want_grad, info, 3001, "bf16")


def test_gradient_against_differences_of_the_loss(fdl, cuda):
    """Central differences along a direction of entries of size at most 1.  The third derivative of a
    row's loss along it is a third central moment of values in [-1, 1]: at most 8 / (6 sqrt 3)."""
    rows, vocab, k, h = 6, 900, 7, 2.0 ** -5
    z, t, index, _ = make(rows, vocab, k, "f32", seed=21)
    g = torch.Generator().manual_seed(3)
    direction = (torch.rand(rows, vocab, generator=g) * 2 - 1).cuda()
    _, _, grad = fdl.distill_topk_with_grad(z, t, index, scale=1.0)
    up = fdl.distill_topk(z + h * direction, t, index, scale=1.0)[1].double()
    down = fdl.distill_topk(z - h * direction, t, index, scale=1.0)[1].double()
    got = (grad.double() * direction.double()).sum(1)
    want = (up - down) / (2 * h)
    info = definition(z, t, index, None, None, 1.0, 1.0)[3]
    loss_tol = info["mass"] * rel_sum(vocab) + info["spread"] * 2 * REL_P
    # the shifted logits themselves are rounded: half a step of numbers below 32
    tol = h * h / 6 * 8 / (6 * math.sqrt(3)) + loss_tol / h + 2 * 2.0 ** -24 * 32 / h + 2.0 ** -18
    assert bool(((got - want).abs().cpu() <= tol).all())


def test_rows_beyond_32_bit_offsets(fdl, cuda):
    """The last rows of a matrix of more than 2^32 bytes, in place."""
    rows, vocab, k = 17000, 131080, 3
    free, _ = cuda.cuda.mem_get_info()
    if free < rows * vocab * 2 + (2 << 30):
        pytest.skip("not enough free device memory")
    z = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    z[-2:] = torch.randn(2, vocab, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    index = torch.zeros(rows, k, dtype=torch.int64, device="cuda")
    index += torch.tensor([5, 131079, 70000], device="cuda")
    t = torch.zeros(rows, k, device="cuda") + torch.tensor([1.0, 0.5, -1.0], device="cuda")
    want_rows, _, want_grad, info = definition(z[-2:], t[-2:], index[-2:], None, None, 1.0, 1.0)
    loss, row_loss, grad = fdl.distill_topk_with_grad(z, t, index, scale=1.0, out=z)
    check_grad(grad[-2:], want_grad, info, vocab, "bf16")
    # rows of zeros: log q = -log vocab
    p = torch.softmax(t[0].double().cpu(), 0)
    first = (p * (p.log() + math.log(vocab))).sum().item()
    assert abs(row_loss[0].item() - first) <= rel_sum(vocab) + 2.0 ** -24 * first + REL_P * first
    assert abs(row_loss[-1].item() - want_rows[-1].item()) <= rel_sum(vocab) + (REL_P + 2.0 ** -24) * info["spread"][-1].item()


def test_streams_and_graph_capture(fdl, cuda):
    """Two calls on two streams at once, and a captured call that follows its inputs when replayed."""
    za, ta, ia, _ = make(40, 30000, 16, "bf16", seed=1)
    zb, tb, ib, _ = make(33, 20011, 16, "f32", seed=2)
    want_a = fdl.distill_topk_with_grad(za, ta, ia)
    want_b = fdl.distill_topk_with_grad(zb, tb, ib)
    cuda.cuda.synchronize()
    one, two = cuda.cuda.Stream(), cuda.cuda.Stream()
    for _ in range(5):
        with cuda.cuda.stream(one):
            got_a = fdl.distill_topk_with_grad(za, ta, ia)
        with cuda.cuda.stream(two):
            got_b = fdl.distill_topk_with_grad(zb, tb, ib)
        cuda.cuda.synchronize()
        for got, want in ((got_a, want_a), (got_b, want_b)):
            assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        loss, row_loss, stats = fdl.distill_topk(za, ta, ia)
        grad = fdl.distill_topk_backward(za, ta, ia, stats)
    for seed in (5, 6):
        z, t, i, _ = make(40, 30000, 16, "bf16", seed=seed)
        za.copy_(z), ta.copy_(t), ia.copy_(i)
        graph.replay()
        cuda.cuda.synchronize()
        want = fdl.distill_topk(z, t, i)
        assert all(torch.equal(x, y) for x, y in zip((loss, row_loss, stats), want))
        assert torch.equal(grad, fdl.distill_topk_backward(z, t, i, want[2]))
