"""Verification of drafted tokens against the definition, sums in 80-bit floats: tokens and counts are equal.

A token is decided by sum <= sample_u * total: with sums in 64 bits the kernel could differ from the
definition only where the two are within a few 2^-53 of each other, which none of the seeded inputs is
(and where sums are exact, as with equal probabilities, there is no difference at all)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def definition(target, draft, tokens, lens, accept, sample):
    target = target.double().cpu().numpy()
    draft = None if draft is None else draft.double().cpu().numpy()
    tokens, accept, sample = tokens.cpu().numpy(), accept.cpu().numpy(), sample.cpu().numpy()
    batch, drafted = tokens.shape
    vocab = target.shape[2]
    out = np.full((batch, drafted + 1), -1, np.int64)
    counts = np.zeros(batch, np.int64)

    def mass(w):
        return np.where((w > 0) & (w < np.inf), w, 0.0)

    for b in range(batch):
        n = drafted if lens is None else min(max(int(lens[b]), 0), drafted)
        i = 0
        while i < n:
            d = tokens[b, i]
            if not 0 <= d < vocab:
                break
            q = 1.0 if draft is None else draft[b, i, d]
            if not np.float32(accept[b, i]) * np.float32(q) < np.float32(target[b, i, d]):
                break
            out[b, i] = d
            i += 1
        with np.errstate(invalid="ignore"):
            w = target[b, i]
            if i < n and draft is not None:
                w = target[b, i] - draft[b, i]
            elif i < n and 0 <= tokens[b, i] < vocab:
                w = target[b, i].copy()
                w[tokens[b, i]] = 0.0
            w = mass(w)
            if not w.any():
                w = mass(target[b, i])
        counts[b] = i
        if not w.any():
            continue
        reach = np.cumsum(w.astype(np.longdouble))
        some = np.flatnonzero(w)
        goal = np.longdouble(np.float64(sample[b])) * reach[-1]
        over = np.flatnonzero(reach > goal)
        out[b, i] = over[0] if over.size else some[-1]
    return out, counts


def make(batch, drafted, vocab, kind, seed, with_draft=True, near=0.5):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(batch, drafted + 1, vocab, generator=g) * 2.5
    target = torch.softmax(logits, -1).to(TYPES[kind])
    q = torch.softmax(logits[:, :drafted] + near * torch.randn(batch, drafted, vocab, generator=g), -1)
    if drafted:
        tokens = torch.multinomial(q.reshape(-1, vocab), 1, generator=g).view(batch, drafted)
    else:
        tokens = torch.empty(batch, 0, dtype=torch.int64)
    accept = torch.rand(batch, drafted, generator=g)
    if not with_draft:
        accept = accept * 2 * target[:, :drafted].float().gather(2, tokens[..., None])[..., 0]
    return dict(target=target.cuda(), draft=q.to(TYPES[kind]).cuda() if with_draft else None, tokens=tokens.cuda(),
                accept=accept.cuda(), sample=torch.rand(batch, generator=g).cuda())


def check(fdl, s, lens=None):
    want, counts = definition(s["target"], s["draft"], s["tokens"], lens, s["accept"], s["sample"])
    got, got_counts = fdl.verify_draft(s["target"], s["tokens"], s["accept"], s["sample"], draft=s["draft"],
                                       draft_len=None if lens is None else lens.cuda())
    assert np.array_equal(got_counts.cpu().numpy(), counts)
    assert np.array_equal(got.cpu().numpy(), want)
    return counts


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("batch,drafted,vocab", [(1, 1, 1), (2, 3, 2), (5, 4, 17), (1, 4, 32000), (3, 2, 4097), (64, 5, 1001),
                                                 (2, 40, 513), (7, 3, 50257), (200, 1, 600), (1, 2, 262147), (33, 2, 9000)])
def test_against_the_definition(fdl, cuda, batch, drafted, vocab, kind):
    for with_draft in (True, False):
        for near in (0.05, 1.0):
            check(fdl, make(batch, drafted, vocab, kind, batch + vocab, with_draft, near))


def test_some_stand_some_fall_all_stand(fdl, cuda):
    counts = check(fdl, make(300, 4, 257, "f32", 5, near=0.4))
    assert set(counts.tolist()) == {0, 1, 2, 3, 4}


def test_lengths_of_sequences(fdl, cuda):
    s = make(9, 6, 3000, "f32", 3, near=0.1)
    lens = torch.tensor([0, 1, 2, 3, 4, 5, 6, -4, 99])
    counts = check(fdl, s, lens)
    assert counts[0] == 0 and counts[7] == 0
    s["tokens"][0] = 1 << 40                  # what lies behind a sequence's length is not looked at
    s["accept"][0] = float("nan")
    check(fdl, s, lens)


def test_nothing_drafted_at_all(fdl, cuda):
    s = make(6, 0, 777, "f32", 1)
    s["draft"] = None
    check(fdl, s)


def test_tokens_outside_the_vocabulary_fall(fdl, cuda):
    for with_draft in (True, False):
        s = make(4, 3, 900, "f32", 9, with_draft)
        s["tokens"][0, 0] = -1
        s["tokens"][1, 1] = 900
        s["tokens"][2, 0] = 1 << 62
        check(fdl, s)


@pytest.mark.parametrize("vocab", [64, 5000, 40000])
def test_the_draft_covers_the_target(fdl, cuda, vocab):
    """p <= q everywhere and yet a rejection: the target's own row serves.  No mass anywhere: -1."""
    s = make(3, 2, vocab, "f32", 2)
    s["draft"][:, :] = s["target"][:, :2]
    s["accept"][:] = 1.0
    s["draft"][0, 0] *= 2
    s["target"][2] = 0.0
    got, counts = fdl.verify_draft(s["target"], s["tokens"], s["accept"], s["sample"], draft=s["draft"])
    check(fdl, s)
    assert counts.tolist() == [0, 0, 0] and got[2].tolist() == [-1, -1, -1]
    one = make(2, 1, vocab, "f32", 4, with_draft=False)   # the only possible token fell: it is drawn again
    one["target"].zero_()
    one["target"][:, 0].scatter_(1, one["tokens"], 1.0)
    one["accept"][:] = 1.0
    check(fdl, one)
    assert fdl.verify_draft(one["target"], one["tokens"], one["accept"], one["sample"])[0][:, 0].tolist() == one["tokens"][:, 0].tolist()


@pytest.mark.parametrize("vocab", [8, 1024, 65536])
def test_borders_of_equal_probabilities(fdl, cuda, vocab):
    """Sums of equal powers of two are exact: sample_u on a border belongs to the next token."""
    batch = 64
    target = torch.full((batch, 1, vocab), 1.0 / vocab, device="cuda")
    picks = torch.randint(0, vocab, (batch,), generator=torch.Generator().manual_seed(1))
    sample = (picks.double() / vocab).float().cuda()
    none = torch.empty(batch, 0, dtype=torch.int64, device="cuda")
    got, _ = fdl.verify_draft(target, none, torch.empty(batch, 0, device="cuda"), sample)
    assert torch.equal(got[:, 0].cpu(), picks)


def test_sample_at_its_ends_and_weights_that_do_not_count(fdl, cuda):
    s = make(5, 1, 4099, "f32", 6)
    s["accept"][:] = 1.0
    s["target"][:, :, ::3] = 0.0
    s["target"][0, :, 5] = float("nan")
    s["target"][1, :, 7] = float("inf")
    s["draft"][2, :, 11] = float("nan")
    s["target"][3, :, -7:] = 0.0
    s["sample"][:] = torch.tensor([0.0, 1.0, 1.0, 1.0, 0.0])
    check(fdl, s)
    got, _ = fdl.verify_draft(s["target"], s["tokens"], s["accept"], torch.full((5,), float("nan"), device="cuda"), draft=s["draft"])
    high, _ = fdl.verify_draft(s["target"], s["tokens"], s["accept"], torch.ones(5, device="cuda"), draft=s["draft"])
    assert torch.equal(got, high)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_strides_and_shifted_starts(fdl, cuda, kind):
    s = make(5, 3, 2001, kind, 12)
    big = torch.zeros(5, 6, 2011, dtype=TYPES[kind], device="cuda")
    big[:, 1:5, 3:2004] = s["target"]
    moved = torch.zeros(3, 5, 2003, dtype=TYPES[kind], device="cuda")
    moved[..., 1:2002] = s["draft"].transpose(0, 1)
    t = dict(s, target=big[:, 1:5, 3:2004], draft=moved[..., 1:2002].transpose(0, 1))
    check(fdl, t)
    a = fdl.verify_draft(s["target"], s["tokens"], s["accept"], s["sample"], draft=s["draft"])
    b = fdl.verify_draft(t["target"], t["tokens"], t["accept"], t["sample"], draft=t["draft"])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    same = dict(s, target=s["target"][:1].expand(5, -1, -1), draft=s["draft"][:1].expand(5, -1, -1))  # stride 0
    check(fdl, same)


def test_distribution_is_the_targets(fdl, cuda):
    """Whatever the draft proposes, the first token is distributed as the target's row (a chi-square of 7
    degrees of freedom exceeds 40.5 once in a million)."""
    batch, vocab = 200000, 8
    g = torch.Generator(device="cuda").manual_seed(7)
    p = torch.tensor([0.3, 0.2, 0.15, 0.1, 0.1, 0.08, 0.05, 0.02], device="cuda")
    q = torch.tensor([0.05, 0.3, 0.1, 0.2, 0.05, 0.1, 0.1, 0.1], device="cuda")
    tokens = torch.multinomial(q, batch, replacement=True, generator=g)[:, None]
    got, _ = fdl.verify_draft(p.expand(batch, 2, vocab), tokens, torch.rand(batch, 1, device="cuda", generator=g),
                              torch.rand(batch, device="cuda", generator=g), draft=q.expand(batch, 1, vocab))
    seen = torch.bincount(got[:, 0], minlength=vocab).double().cpu()
    want = p.double().cpu() / p.double().cpu().sum() * batch
    assert ((seen - want) ** 2 / want).sum().item() < 40.5


def test_offsets_beyond_32_bits(fdl, cuda):
    vocab, batch = 131072, 9000
    free, _ = cuda.cuda.mem_get_info()
    if free < vocab * batch * 4 + (2 << 30):
        pytest.skip("not enough free device memory")
    base = torch.zeros(batch, 2, vocab, dtype=torch.float16, device="cuda")
    base[-1, 0, 5] = 1.0
    base[-1, 1, vocab - 3] = 1.0
    base[:-1, :, 9] = 1.0
    tokens = torch.full((batch, 1), 9, device="cuda")
    tokens[-1] = 5
    got, counts = fdl.verify_draft(base, tokens, torch.full((batch, 1), 0.5, device="cuda"), torch.full((batch,), 0.5, device="cuda"))
    assert bool((counts == 1).all()) and got[-1].tolist() == [5, vocab - 3] and bool((got[:-1] == 9).all())


def test_streams_and_graph_capture(fdl, cuda):
    a, b = make(16, 4, 32000, "f32", 1), make(5, 3, 50257, "bf16", 2)

    def call(s):
        return fdl.verify_draft(s["target"], s["tokens"], s["accept"], s["sample"], draft=s["draft"])

    want_a, want_b = call(a), call(b)
    cuda.cuda.synchronize()
    one, two = cuda.cuda.Stream(), cuda.cuda.Stream()
    for _ in range(5):
        with cuda.cuda.stream(one):
            got_a = call(a)
        with cuda.cuda.stream(two):
            got_b = call(b)
        cuda.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got_a + got_b, want_a + want_b))
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        got = call(a)
    for seed in (3, 4):
        s = make(16, 4, 32000, "f32", seed)
        for name in a:
            a[name].copy_(s[name])
        graph.replay()
        cuda.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, call(s)))
