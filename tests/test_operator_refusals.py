"""Calls that the distillation, gated norm and draft verification entry points refuse: an error code before
anything is launched (no GPU needed: arguments are checked first), ValueError from the Python binding."""
import ctypes as C

import pytest
import torch

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3
P = 4096  # stands for a device pointer: it is not looked at


def call(fn, names, defaults, **changes):
    args = dict(defaults, **changes)
    assert set(changes) <= set(names)
    return fn(*[args[n] for n in names])


DISTILL = ["logits", "stride", "dtype", "teacher", "teacher_dtype", "index", "lse", "weight", "rows", "vocab", "k", "temperature",
           "scale", "loss", "row_loss", "stats", "stream"]
DISTILL_OK = dict(logits=P, stride=100, dtype=0, teacher=P, teacher_dtype=0, index=P, lse=None, weight=None, rows=4, vocab=100, k=5,
                  temperature=1.0, scale=1.0, loss=P, row_loss=P, stats=P, stream=None)
BAD_DISTILL = [(dict(logits=None), INVALID), (dict(teacher=None), INVALID), (dict(index=None), INVALID), (dict(stride=99), INVALID),
               (dict(dtype=3), INVALID), (dict(dtype=-1), INVALID), (dict(teacher_dtype=7), INVALID), (dict(rows=-1), INVALID),
               (dict(vocab=0), INVALID), (dict(k=0), INVALID), (dict(k=1025), UNSUPPORTED), (dict(temperature=0.0), INVALID),
               (dict(temperature=-1.0), INVALID), (dict(temperature=float("nan")), INVALID), (dict(temperature=float("inf")), INVALID),
               (dict(rows=1 << 31), UNSUPPORTED), (dict(vocab=1 << 31, stride=1 << 31), UNSUPPORTED)]


@pytest.mark.parametrize("change,status", BAD_DISTILL + [(dict(loss=None), INVALID), (dict(row_loss=None), INVALID), (dict(stats=None), INVALID)])
def test_distill_loss(fdl, change, status):
    assert call(fdl.lib().fdl_distill_topk, DISTILL, DISTILL_OK, **change) == status


@pytest.mark.parametrize("change,status", BAD_DISTILL + [(dict(grad=None), INVALID), (dict(grad_stride=99), INVALID),
                                                         (dict(grad=P, grad_stride=101), INVALID), (dict(stats=None), INVALID)])
def test_distill_gradients(fdl, change, status):
    names = DISTILL[:-1] + ["grad", "grad_stride", "stream"]
    ok = dict(DISTILL_OK, grad=2 * P, grad_stride=100)
    assert call(fdl.lib().fdl_distill_topk_with_grad, names, ok, **change) == status
    back = DISTILL[:8] + ["stats", "grad_loss"] + DISTILL[8:13] + ["grad", "grad_stride", "stream"]
    ok = dict(ok, grad_loss=None)
    assert call(fdl.lib().fdl_distill_topk_backward, back, ok, **change) == status


NORM = ["x", "h", "gate", "gate_rows", "gate_act", "post", "post_gamma", "post_beta", "pre", "pre_gamma", "pre_beta", "y", "n", "stats",
        "rows", "cols", "residual_scale", "block_scale", "eps", "dtype", "stream"]
NORM_OK = dict(x=P, h=2 * P, gate=None, gate_rows=0, gate_act=0, post=1, post_gamma=None, post_beta=None, pre=1, pre_gamma=None,
               pre_beta=None, y=3 * P, n=4 * P, stats=None, rows=6, cols=64, residual_scale=1.0, block_scale=1.0, eps=1e-5, dtype=0,
               stream=None)
BAD_NORM = [(dict(h=None), INVALID), (dict(gate=P), INVALID), (dict(gate_rows=1), INVALID), (dict(gate=P, gate_rows=4), INVALID),
            (dict(gate=P, gate_rows=7), INVALID), (dict(gate_act=3), INVALID), (dict(gate_act=-1), INVALID), (dict(post=3), INVALID),
            (dict(pre=-1), INVALID), (dict(rows=-1), INVALID), (dict(cols=0), INVALID), (dict(cols=32769), UNSUPPORTED),
            (dict(rows=1 << 31), UNSUPPORTED), (dict(dtype=4), INVALID), (dict(stats=P + 8), INVALID), (dict(post=0, post_gamma=P), INVALID)]


@pytest.mark.parametrize("change,status", BAD_NORM + [
    (dict(x=None), INVALID), (dict(y=None), INVALID), (dict(n=None), INVALID), (dict(pre=0), INVALID), (dict(n=3 * P), INVALID),
    (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(post=0, post_beta=P), INVALID),
    (dict(pre=0, n=None, pre_gamma=P), INVALID), (dict(pre=0, n=None, pre_beta=P), INVALID)])
def test_norm_forward(fdl, change, status):
    assert call(fdl.lib().fdl_norm_residual, NORM, NORM_OK, **change) == status


@pytest.mark.parametrize("change,status", BAD_NORM + [
    (dict(stats=None), INVALID), (dict(dy=None, dn=None), INVALID), (dict(y=None), INVALID), (dict(dgate=P), INVALID),
    (dict(pre=0), INVALID), (dict(pre=0, dn=None, dpre_beta=P), INVALID), (dict(post=0, dpost_gamma=P), INVALID),
    (dict(scratch=None), WORKSPACE), (dict(scratch=P + 16), WORKSPACE), (dict(scratch_bytes=0), WORKSPACE)])
def test_norm_backward(fdl, change, status):
    names = ["dy", "dn", "y", "h", "stats", "gate", "gate_rows", "gate_act", "post", "post_gamma", "post_beta", "pre", "pre_gamma", "dx",
             "dh", "dgate", "dpost_gamma", "dpost_beta", "dpre_gamma", "dpre_beta", "rows", "cols", "residual_scale", "block_scale",
             "dtype", "scratch", "scratch_bytes", "stream"]
    ok = dict(NORM_OK, dy=P, dn=2 * P, stats=5 * P, dx=6 * P, dh=7 * P, dgate=None, dpost_gamma=None, dpost_beta=None, dpre_gamma=None,
              dpre_beta=None, scratch=P, scratch_bytes=1 << 40)
    assert call(fdl.lib().fdl_norm_residual_backward, names, ok, **change) == status


def test_norm_scratch_bytes(fdl):
    size = fdl.lib().fdl_norm_residual_backward_scratch_bytes
    for rows, cols, gates in ((1, 1, 0), (100, 64, 0), (100, 4096, 4), (70000, 8192, 7), (12, 32768, 12)):
        assert size(rows, cols, gates) % 256 == 0 and size(rows, cols, gates) > 0
    for bad in ((0, 64, 0), (10, 0, 0), (10, 64, 3), (10, 64, -1), (10, 64, 11), (10, 32769, 0), (-1, 64, 0)):
        assert size(*bad) == 0


@pytest.mark.parametrize("change,status", [
    (dict(target=None), INVALID), (dict(tokens=None), INVALID), (dict(drawn=None), INVALID), (dict(accept=None), INVALID),
    (dict(sample=None), INVALID), (dict(accepted=None), INVALID), (dict(dtype=5), INVALID), (dict(batch=-1), INVALID),
    (dict(drafted=-1), INVALID), (dict(vocab=0), INVALID), (dict(tb=-1), INVALID), (dict(tr=-1), INVALID), (dict(db=-1), INVALID),
    (dict(dr=-1), INVALID), (dict(drafted=65536), UNSUPPORTED), (dict(vocab=1 << 31), UNSUPPORTED), (dict(batch=1 << 31), UNSUPPORTED)])
def test_verify(fdl, change, status):
    names = ["target", "tb", "tr", "draft", "db", "dr", "dtype", "drawn", "len", "accept", "sample", "batch", "drafted", "vocab", "tokens",
             "accepted", "stream"]
    ok = dict(target=P, tb=500, tr=100, draft=P, db=400, dr=100, dtype=0, drawn=P, len=None, accept=P, sample=P, batch=2, drafted=4,
              vocab=100, tokens=P, accepted=P, stream=None)
    assert call(fdl.lib().fdl_verify_draft, names, ok, **change) == status


def test_empty_calls_are_fine_without_pointers(fdl):
    lib = fdl.lib()
    assert call(lib.fdl_norm_residual, NORM, NORM_OK, rows=0, x=None, h=None, y=None, n=None) == 0
    assert lib.fdl_verify_draft(None, 0, 0, None, 0, 0, 0, None, None, None, None, 0, 3, 10, None, None, None) == 0
    assert lib.fdl_distill_topk_backward(None, 10, 0, None, 0, None, None, None, None, None, 0, 10, 2, C.c_float(1), C.c_float(1), None,
                                         10, None) == 0


def test_binding_refuses_tensors_off_the_current_device(fdl):
    z, t, i = torch.zeros(2, 8), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int64)
    for fn in (fdl.distill_topk, fdl.distill_topk_with_grad):
        with pytest.raises(ValueError, match="current CUDA device"):
            fn(z, t, i)
    with pytest.raises(ValueError, match="current CUDA device"):
        fdl.distill_topk_backward(z, t, i, torch.zeros(2, 2))
    with pytest.raises(ValueError, match="current CUDA device"):
        fdl.norm_residual(z, z)
    with pytest.raises(ValueError, match="current CUDA device"):
        fdl.norm_residual_backward(z, z, z, z, torch.zeros(2, 4))
    with pytest.raises(ValueError, match="current CUDA device"):
        fdl.verify_draft(torch.zeros(2, 4, 9), i, torch.zeros(2, 3), torch.zeros(2))
    with pytest.raises(ValueError, match="batch"):
        fdl.verify_draft(torch.zeros(2, 9), i, torch.zeros(2, 3), torch.zeros(2))


@pytest.mark.gpu
def test_binding_refuses_wrong_shapes_types_and_strides(fdl, cuda):
    z, t = torch.zeros(4, 32, device="cuda"), torch.zeros(4, 3, device="cuda")
    i = torch.zeros(4, 3, dtype=torch.int64, device="cuda")
    bad = [lambda: fdl.distill_topk(z.double(), t, i), lambda: fdl.distill_topk(z, t, i.int()), lambda: fdl.distill_topk(z, t[:, :2], i), lambda: fdl.distill_topk(z, t, i[:1]), lambda: fdl.distill_topk(z[0], t, i),
           lambda: fdl.distill_topk(z, t, i[:, :2]),
           lambda: fdl.distill_topk(z.t(), t, i), lambda: fdl.distill_topk(z[:1].expand(4, 32), t, i),
           lambda: fdl.distill_topk(z, t, i, row_weight=torch.zeros(3, device="cuda")),
           lambda: fdl.distill_topk(z, t, i, teacher_lse=torch.zeros(4, device="cuda").half()),
           lambda: fdl.distill_topk_with_grad(z, t, i, out=z.half()), lambda: fdl.distill_topk_with_grad(z, t, i, out=z[:, :16]),
           lambda: fdl.distill_topk_backward(z, t, i, torch.zeros(4, device="cuda")),
           lambda: fdl.distill_topk_backward(z, t, i, torch.zeros(4, 2, device="cuda"), grad_loss=torch.zeros(2, device="cuda")),
           lambda: fdl.norm_residual(z, z.half()), lambda: fdl.norm_residual(z.t(), z.t()), lambda: fdl.norm_residual(z, z[:2]),
           lambda: fdl.norm_residual(z, z, gate=z[:, :3].contiguous()), lambda: fdl.norm_residual(z, z, post_gamma=t[0]),
           lambda: fdl.norm_residual(z, z, post_gamma=z[0].half()), lambda: fdl.norm_residual(z, z, out=z.half()),
           lambda: fdl.norm_residual_backward(z, z, z, z, torch.zeros(4, 2, device="cuda")),
           lambda: fdl.verify_draft(torch.zeros(4, 3, 9, device="cuda"), i, t, t[:, 0].contiguous()),
           lambda: fdl.verify_draft(torch.zeros(4, 4, 9, device="cuda"), i, t, t[:, 0]),
           lambda: fdl.verify_draft(torch.zeros(4, 9, 4, device="cuda").transpose(1, 2), i, t, t[:, 0].contiguous()),
           lambda: fdl.verify_draft(torch.zeros(4, 4, 9, device="cuda"), i, t, t[:, 0].contiguous(),
                                    draft=torch.zeros(4, 3, 9, device="cuda").half()),
           lambda: fdl.verify_draft(torch.zeros(4, 4, 9, device="cuda"), i, t, t[:, 0].contiguous(),
                                    draft=torch.zeros(4, 3, 1, device="cuda").expand(4, 3, 9))]
    for k, fn in enumerate(bad):
        with pytest.raises(ValueError):
            fn()
            pytest.fail(f"call {k} was accepted")
    with pytest.raises(fdl.FdlError):
        fdl.norm_residual(z, z, gate=torch.zeros(3, 32, device="cuda"))
    with pytest.raises(fdl.FdlError):
        fdl.distill_topk(z, t, i, temperature=0.0)
