"""The measured cases of the operators for training a draft model from a teacher and serving with it:

  distill   the distillation loss on a teacher's top logits, its gradient, and both in one call
  norm      the norms after and before a block, its gate and its residual scale, forward and backward
  verify    the verification of drafted tokens against the target's probabilities

Each operator stands here in its plain form (elementary torch operations in 32 bits, rounded once at
the end; 64 bits where the position of a sampled token depends on a long sum), and as the call that a
user of the framework makes.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases -----------------------------------------------------------------------------------------


def listed():
    return [
        # The loss alone on a short validation batch: a few sequences' last tokens, latency counts.
        {"name": "distill loss small", "op": "distill", "mode": "loss", "rows": 8, "vocab": 32000, "k": 8, "type": "f32",
         "temperature": 1.0, "tail": False},
        # The gradient for a graph that kept the forward pass's statistics; an odd vocabulary.
        {"name": "distill backward odd", "op": "distill", "mode": "backward", "rows": 1000, "vocab": 50257, "k": 64,
         "type": "f32", "temperature": 2.0, "tail": False},
        # A training step's loss and gradient in one call: 2048 tokens, a large vocabulary, 16-bit logits.
        {"name": "distill train bf16", "op": "distill", "mode": "train", "rows": 2048, "vocab": 131072, "k": 64,
         "type": "bf16", "temperature": 1.0, "tail": True},
        # The same in 32 bits, with many entries a token and a vocabulary that is no multiple of four.
        {"name": "distill train f32", "op": "distill", "mode": "train", "rows": 4096, "vocab": 65537, "k": 128,
         "type": "f32", "temperature": 1.5, "tail": False},
        # One new token at a time: a decoding step between two blocks.
        {"name": "norm decode", "op": "norm", "mode": "forward", "rows": 1, "cols": 4096, "type": "bf16",
         "post": "rms", "pre": "rms", "gate": "shared", "act": "none"},
        # A prompt's tokens with a gate for each token and channel.
        {"name": "norm prompt", "op": "norm", "mode": "forward", "rows": 16384, "cols": 4096, "type": "bf16",
         "post": "rms", "pre": "rms", "gate": "full", "act": "sigmoid"},
        # Training in 32 bits with layer norms, an odd width and no gate.
        {"name": "norm backward odd", "op": "norm", "mode": "backward", "rows": 2049, "cols": 1001, "type": "f32",
         "post": "layer", "pre": "layer", "gate": "none", "act": "none"},
        # Training on long sequences: a gate for each sequence's channels, shared by its tokens.
        {"name": "norm backward", "op": "norm", "mode": "backward", "rows": 16384, "cols": 8192, "type": "bf16",
         "post": "rms", "pre": "rms", "gate": "sequence", "act": "tanh"},
        # A single user's decoding step: four drafted tokens.
        {"name": "verify one", "op": "verify", "batch": 1, "drafted": 4, "vocab": 32000, "type": "f32", "draft": True},
        # A serving batch, an odd vocabulary.
        {"name": "verify batch odd", "op": "verify", "batch": 64, "drafted": 5, "vocab": 50257, "type": "f32", "draft": True},
        # Tokens drafted by looking them up in the text (no draft probabilities), 16-bit target.
        {"name": "verify lookup", "op": "verify", "batch": 32, "drafted": 8, "vocab": 100003, "type": "bf16", "draft": False},
        # The largest batch and vocabulary.
        {"name": "verify large", "op": "verify", "batch": 256, "drafted": 7, "vocab": 131072, "type": "f32", "draft": True},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["distill", "norm", "verify"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "distill":
        vocab = _spread(rng, 500, 200000)
        rows = _spread(rng, 1, max(2, min(16384, 2.5e8 / vocab)))
        return {"op": op, "mode": rng.choice(["loss", "backward", "train"]), "rows": rows, "vocab": vocab,
                "k": min(_spread(rng, 1, 256), vocab), "type": kind, "temperature": rng.choice([0.7, 1.0, 2.0]),
                "tail": rng.random() < 0.5}
    if op == "norm":
        cols = _spread(rng, 64, 16384)
        if rng.random() < 0.6:
            cols = max(64, cols // 64 * 64)
        rows = _spread(rng, 1, max(2, min(65536, 6e7 / cols)))
        gate = rng.choice(["none", "shared", "sequence", "full"])
        if gate == "sequence":
            rows = max(8, rows // 8 * 8)
        return {"op": op, "mode": rng.choice(["forward", "backward"]), "rows": rows, "cols": cols, "type": kind,
                "post": rng.choice(["rms", "layer"]), "pre": rng.choice(["rms", "layer"]), "gate": gate,
                "act": "none" if gate == "none" else rng.choice(["none", "sigmoid", "tanh"])}
    vocab = _spread(rng, 500, 200000)
    drafted = _spread(rng, 1, 16)
    return {"op": op, "batch": _spread(rng, 1, max(2, min(512, 2.5e8 / (vocab * drafted)))), "drafted": drafted,
            "vocab": vocab, "type": kind, "draft": rng.random() < 0.7}


# ---- inputs ----------------------------------------------------------------------------------------


def _distill_inputs(case, g):
    rows, vocab, k, kind = case["rows"], case["vocab"], case["k"], TYPES[case["type"]]
    dev = "cuda"
    logits = torch.empty(rows, vocab, dtype=kind, device=dev).normal_(0.0, 2.0, generator=g)
    # The teacher's k entries: other places for each row, values in falling order; the student knows them in part.
    first = torch.randint(0, vocab, (rows, 1), device=dev, generator=g)
    index = (first + torch.arange(k, device=dev) * max(1, vocab // k)) % vocab
    teacher = (torch.randn(rows, k, device=dev, generator=g) * 2.0 + 8.0).sort(-1, descending=True).values
    seen = 0.7 * teacher + torch.randn(rows, k, device=dev, generator=g)
    logits.scatter_(1, index, seen.to(kind))
    # The tail of some rows is padding (a shorter list), and some rows are padding altogether.
    short = torch.rand(rows, 1, device=dev, generator=g) < 0.2
    cut = torch.arange(k, device=dev) >= max(1, k - k // 4)
    index = torch.where(short & cut, torch.full_like(index, -1), index)
    weight = (torch.rand(rows, device=dev, generator=g) >= 0.05).float()
    lse = None
    if case["tail"]:  # the teacher's own normaliser: what is not among the k holds some of the mass
        lse = torch.logsumexp(teacher / case["temperature"], -1) + 0.1 * torch.rand(rows, device=dev, generator=g)
    return {"logits": logits, "teacher": teacher.to(kind), "index": index, "lse": lse, "weight": weight,
            "temperature": case["temperature"], "scale": 1.0 / rows, "mode": case["mode"]}


def _norm_inputs(case, g):
    rows, cols, kind = case["rows"], case["cols"], TYPES[case["type"]]
    dev = "cuda"

    def normal(*shape, mean=0.0, std=1.0):
        return torch.empty(*shape, dtype=kind, device=dev).normal_(mean, std, generator=g)

    def weight(mean):
        return mean + 0.1 * torch.randn(cols, device=dev, generator=g)

    s = {"mode": case["mode"], "post": case["post"], "pre": case["pre"], "act": case["act"],
         "h": normal(rows, cols, mean=0.2, std=1.5), "post_gamma": weight(1.0), "pre_gamma": weight(1.0),
         "post_beta": weight(0.0) if case["post"] == "layer" else None,
         "pre_beta": weight(0.0) if case["pre"] == "layer" else None,
         "residual_scale": 1.0, "block_scale": 0.5, "eps": 1e-5}
    gates = {"none": 0, "shared": 1, "sequence": 8, "full": rows}[case["gate"]]
    s["gate"] = normal(gates, cols, mean=0.5) if gates else None
    x = normal(rows, cols, std=2.0)
    if case["mode"] == "forward":
        s["x"] = x
        return s
    s["x"] = x
    y, _, stats = _norm_forward(s)
    del s["x"]
    s["y"], s["stats"] = y, stats
    s["dy"], s["dn"] = normal(rows, cols), normal(rows, cols)
    return s


def _verify_inputs(case, g):
    batch, drafted, vocab, kind = case["batch"], case["drafted"], case["vocab"], TYPES[case["type"]]
    dev = "cuda"
    logits = torch.empty(batch, drafted + 1, vocab, device=dev).normal_(0.0, 3.0, generator=g)
    draft = None
    if case["draft"]:  # the draft model's opinion: the target's with noise
        near = torch.empty(batch, drafted, vocab, device=dev).normal_(0.0, 0.5, generator=g)
        near += logits[:, :drafted]
        draft = torch.softmax(near, -1)
        del near
        tokens = torch.multinomial(draft.view(-1, vocab), 1, generator=g).view(batch, drafted)
        draft = draft.to(kind)
    target = torch.softmax(logits, -1)
    if not case["draft"]:  # a continuation that the target often agrees with
        tokens = torch.multinomial(target[:, :drafted].reshape(-1, vocab), 1, generator=g).view(batch, drafted)
        target[:, :drafted] *= 0.2
        target[:, :drafted].scatter_add_(2, tokens[..., None], torch.full((batch, drafted, 1), 0.8, device=dev))
    return {"target": target.to(kind), "draft": draft, "tokens": tokens,
            "accept": torch.rand(batch, drafted, device=dev, generator=g),
            "sample": torch.rand(batch, device=dev, generator=g)}


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed))
    s = {"distill": _distill_inputs, "norm": _norm_inputs, "verify": _verify_inputs}[case["op"]](case, g)
    s["op"] = case["op"]
    if case["op"] == "distill" and case["mode"] == "backward":
        m = s["logits"].amax(-1, keepdim=True).float()
        total = torch.exp((s["logits"].float() - m) / s["temperature"]).sum(-1, keepdim=True)
        s["stats"] = torch.cat([m, total], 1)
    return s


# ---- plain forms -------------------------------------------------------------------------------------


def _teacher(s, vocab):
    """The teacher's probabilities (0 for entries that do not count), their logarithms, which rows count, their mass."""
    t = s["teacher"].float() / s["temperature"]
    counts = (s["index"] >= 0) & (s["index"] < vocab) & (t > -math.inf)
    t = torch.where(counts, t, torch.full_like(t, -math.inf))
    rows = counts.any(-1) & (s["weight"] != 0)
    top = torch.where(rows, t.amax(-1), torch.zeros_like(t[:, 0]))[:, None]
    if s["lse"] is None:
        norm = top + torch.log(torch.exp(t - top).sum(-1, keepdim=True))
    else:
        norm = s["lse"][:, None]
    keep = counts & rows[:, None]
    logp = torch.where(keep, t - norm, torch.zeros_like(t))
    p = torch.where(keep, torch.exp(logp), torch.zeros_like(t))
    mass = rows.float() if s["lse"] is None else p.sum(-1)
    return p, logp, rows, mass


def _distill(s):
    z, vocab = s["logits"].float(), s["logits"].shape[1]
    p, logp, rows, mass = _teacher(s, vocab)
    at = s["index"].clamp(0, vocab - 1)
    if s["mode"] == "backward":
        m, total = s["stats"][:, :1], s["stats"][:, 1:]
        e = torch.exp((z - m) / s["temperature"])
    else:
        m = z.amax(-1, keepdim=True)
        e = torch.exp((z - m) / s["temperature"])
        total = e.sum(-1, keepdim=True)
        logq = (z.gather(1, at) - m) / s["temperature"] - torch.log(total)
        row_loss = (p * (logp - logq)).sum(-1)
        loss = s["scale"] * (s["weight"] * row_loss).double().sum().float().reshape(1)
        if s["mode"] == "loss":
            return loss, row_loss
    e *= (mass[:, None] / total)
    e.scatter_add_(1, at, -p)
    e *= torch.where(rows, s["weight"] * (s["scale"] / s["temperature"]), torch.zeros_like(mass))[:, None]
    grad = e.to(s["logits"].dtype)
    return grad if s["mode"] == "backward" else (loss, row_loss, grad)


def _act(name, g):
    return torch.sigmoid(g) if name == "sigmoid" else torch.tanh(g) if name == "tanh" else g


def _by_rows(gate):
    """[gates, 1, cols] against a view of [rows, cols] as [gates, rows of a gate, cols]."""
    return gate.float()[:, None, :]


def _moments(v, kind, eps):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    c = v - mean
    return c, mean, torch.rsqrt((c * c).mean(-1, keepdim=True) + eps)


def _norm_forward(s):
    h, x = s["h"].float(), s["x"].float()
    rows, cols = h.shape
    c, mean1, r1 = _moments(h, s["post"], s["eps"])
    u = c * r1 * s["post_gamma"]
    if s["post_beta"] is not None:
        u = u + s["post_beta"]
    if s["gate"] is not None:
        u = (u.view(s["gate"].shape[0], -1, cols) * _act(s["act"], _by_rows(s["gate"]))).view(rows, cols)
    y = s["residual_scale"] * x + s["block_scale"] * u
    c, mean2, r2 = _moments(y, s["pre"], s["eps"])
    n = c * r2 * s["pre_gamma"]
    if s["pre_beta"] is not None:
        n = n + s["pre_beta"]
    return y.to(s["x"].dtype), n.to(s["x"].dtype), torch.cat([mean1, r1, mean2, r2], 1)


def _norm_grad(d, hat, rstd, kind):
    """Gradient of (v - mean) * rstd from that of its result."""
    d2 = d - hat * (d * hat).mean(-1, keepdim=True)
    if kind == "layer":
        d2 = d2 - d.mean(-1, keepdim=True)
    return rstd * d2


def _norm_backward(s):
    kind, st = s["h"].dtype, s["stats"]
    dy, dn, y, h = s["dy"].float(), s["dn"].float(), s["y"].float(), s["h"].float()
    rows, cols = h.shape
    hat = (y - st[:, 2:3]) * st[:, 3:4]
    out = {"pre_gamma": (dn * hat).sum(0)}
    if s["pre_beta"] is not None:
        out["pre_beta"] = dn.sum(0)
    d = dy + _norm_grad(dn * s["pre_gamma"], hat, st[:, 3:4], s["pre"])
    out["x"] = (s["residual_scale"] * d).to(kind)
    d = s["block_scale"] * d
    hat = (h - st[:, 0:1]) * st[:, 1:2]
    if s["gate"] is not None:
        u = hat * s["post_gamma"]
        if s["post_beta"] is not None:
            u = u + s["post_beta"]
        gates = s["gate"].shape[0]
        a = _act(s["act"], _by_rows(s["gate"]))
        slope = a * (1 - a) if s["act"] == "sigmoid" else 1 - a * a if s["act"] == "tanh" else torch.ones_like(a)
        out["gate"] = ((d * u).view(gates, -1, cols).sum(1, keepdim=True) * slope).view(gates, cols).to(kind)
        d = (d.view(gates, -1, cols) * a).view(rows, cols)
    out["post_gamma"] = (d * hat).sum(0)
    if s["post_beta"] is not None:
        out["post_beta"] = d.sum(0)
    out["h"] = _norm_grad(d * s["post_gamma"], hat, st[:, 1:2], s["post"]).to(kind)
    return out


def _verify(s):
    target, draft, tokens = s["target"], s["draft"], s["tokens"]
    batch, drafted = tokens.shape
    each = torch.arange(batch, device=target.device)
    pd = target[:, :drafted].gather(2, tokens[..., None])[..., 0].float()
    qd = torch.ones_like(pd) if draft is None else draft.gather(2, tokens[..., None])[..., 0].float()
    taken = (s["accept"] * qd < pd).long().cumprod(1)
    accepted = taken.sum(1)
    p = target[each, accepted].double()
    last = accepted.clamp(max=drafted - 1)
    if draft is None:
        q = torch.zeros_like(p).scatter_(1, tokens[each, last][:, None], math.inf)
    else:
        q = draft[each, last].double()
    rejected = (accepted < drafted)[:, None]
    w = torch.where(rejected, (p - q).clamp(min=0.0), p)
    w = torch.where(w.sum(1, keepdim=True) > 0, w, p)
    total = w.cumsum(1)
    token = (total <= s["sample"].double()[:, None] * total[:, -1:]).sum(1)
    at = torch.arange(w.shape[1], device=w.device)
    token = torch.minimum(token, torch.where(w > 0, at, torch.full_like(at, -1)).amax(1))
    place = torch.arange(drafted + 1, device=target.device)[None, :]
    out = torch.cat([tokens, torch.zeros_like(tokens[:, :1])], 1)
    out = torch.where(place < accepted[:, None], out, torch.where(place == accepted[:, None], token[:, None], torch.full_like(out, -1)))
    return out, accepted


# ---- one pass --------------------------------------------------------------------------------------


def _own(s):
    from fast_dl_b200 import capi

    if s["op"] == "distill":
        more = dict(teacher_lse=s["lse"], row_weight=s["weight"], temperature=s["temperature"], scale=s["scale"])
        if s["mode"] == "loss":
            loss, row_loss, _ = capi.distill_topk(s["logits"], s["teacher"], s["index"], **more)
            return loss, row_loss
        if s["mode"] == "backward":
            return capi.distill_topk_backward(s["logits"], s["teacher"], s["index"], s["stats"], **more)
        return capi.distill_topk_with_grad(s["logits"], s["teacher"], s["index"], **more)
    if s["op"] == "verify":
        return capi.verify_draft(s["target"], s["tokens"], s["accept"], s["sample"], draft=s["draft"])
    kinds = {"rms": capi.NORM_RMS, "layer": capi.NORM_LAYER}
    acts = {"none": capi.GATE_PLAIN, "sigmoid": capi.GATE_SIGMOID, "tanh": capi.GATE_TANH}
    more = dict(post=kinds[s["post"]], pre=kinds[s["pre"]], gate=s["gate"], gate_act=acts[s["act"]],
                post_gamma=s["post_gamma"], post_beta=s["post_beta"], pre_gamma=s["pre_gamma"],
                residual_scale=s["residual_scale"], block_scale=s["block_scale"])
    if s["mode"] == "forward":
        return capi.norm_residual(s["x"], s["h"], pre_beta=s["pre_beta"], eps=s["eps"], **more)
    grads = capi.norm_residual_backward(s["dy"], s["dn"], s["y"], s["h"], s["stats"],
                                        want_post_beta=s["post_beta"] is not None,
                                        want_pre_beta=s["pre_beta"] is not None, **more)
    return {name: g for name, g in grads.items() if g is not None}


def run(state):
    if own:
        return _own(state)
    if state["op"] == "distill":
        return _distill(state)
    if state["op"] == "verify":
        return _verify(state)
    return _norm_forward(state) if state["mode"] == "forward" else _norm_backward(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------


def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "distill":
        n = case["rows"] * case["vocab"] * 0.95  # rows of weight 0 need no reading
        moved = {"loss": n, "backward": n + case["rows"] * case["vocab"], "train": n + case["rows"] * case["vocab"]}
        flops = {"loss": 4, "backward": 4, "train": 7}[case["mode"]] * n
        return {"bytes": moved[case["mode"]] * size + case["rows"] * (case["k"] * (size + 8) + 16), "flops": flops}
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        gate = {"none": 0, "shared": 1, "sequence": 8, "full": case["rows"]}[case["gate"]] * case["cols"]
        if case["mode"] == "forward":
            return {"bytes": (4 * n + gate) * size + 8 * case["cols"] + 16 * case["rows"], "flops": 12 * n}
        return {"bytes": (6 * n + 2 * gate) * size + 16 * case["cols"] + 16 * case["rows"], "flops": 30 * n}
    rows = 1.0 + (0.8 if case["draft"] else 0.0)  # the target's row, and the draft's after a rejection
    read = case["batch"] * case["vocab"] * rows
    small = case["batch"] * case["drafted"] * (2 * size + 8 + 4 + 8)
    return {"bytes": read * size + small, "flops": 3 * read}


# ---- from the definitions, in 64 bits -------------------------------------------------------------------


def _exact_distill(case, s):
    f8 = torch.float64
    rows, vocab = s["logits"].shape
    grads = case["mode"] != "loss"
    temperature = float(s["temperature"])
    loss = torch.zeros(rows, dtype=f8, device="cuda")
    grad = torch.zeros(rows, vocab, dtype=f8, device="cuda") if grads else None
    step = max(1, 100_000_000 // vocab)
    for a in range(0, rows, step):  # some rows at a time: 64 bits take room
        b = min(rows, a + step)
        index, weight = s["index"][a:b], s["weight"][a:b].to(f8)
        known = (index >= 0) & (index < vocab) & torch.isfinite(s["teacher"][a:b])
        live = known.any(1) & (weight != 0)
        t = (s["teacher"][a:b].to(f8) / temperature).masked_fill(~known, -math.inf)
        if s["lse"] is None:
            logp = torch.log_softmax(t.masked_fill(~live[:, None], 0.0), 1)
        else:
            logp = t - s["lse"][a:b, None].to(f8)
        use = known & live[:, None]
        p = torch.exp(logp).masked_fill(~use, 0.0)
        logq = torch.log_softmax(s["logits"][a:b].to(f8) / temperature, 1)
        here = logq.gather(1, index.masked_fill(~known, 0))
        loss[a:b] = (p * (logp - here).masked_fill(~use, 0.0)).sum(1)
        if grads:
            dense = torch.exp(logq) * p.sum(1, keepdim=True)
            dense.scatter_add_(1, index.masked_fill(~known, 0), -p)
            grad[a:b] = dense * (weight * live * float(s["scale"]) / temperature)[:, None]
    total = (loss * s["weight"].to(f8)).sum().reshape(1) * float(s["scale"])
    return {"loss": (total, loss), "backward": grad, "train": (total, loss, grad)}[case["mode"]]


def _exact_norm(case, s):
    f8 = torch.float64

    def leaf(t):
        return None if t is None else t.to(f8)

    def normed(v, kind, gamma, beta):
        if kind == "layer":
            v = v - v.mean(1, keepdim=True)
        v = v / torch.sqrt(v.pow(2).mean(1, keepdim=True) + s["eps"]) * gamma.to(f8)
        return v if beta is None else v + beta.to(f8)

    rows, cols = s["h"].shape
    gate = leaf(s["gate"])
    act = {"none": lambda v: v, "sigmoid": lambda v: 1 / (1 + torch.exp(-v)), "tanh": torch.tanh}[case["act"]]
    if case["mode"] == "forward":
        branch = normed(leaf(s["h"]), s["post"], s["post_gamma"], s["post_beta"])
        if gate is not None:
            branch = branch * act(gate).repeat_interleave(rows // gate.shape[0], 0)
        y = s["residual_scale"] * leaf(s["x"]) + s["block_scale"] * branch
        h = leaf(s["h"])
        parts = []
        for v, kind in ((h, s["post"]), (y, s["pre"])):
            mean = v.mean(1) if kind == "layer" else torch.zeros(rows, dtype=f8, device="cuda")
            parts += [mean, 1 / torch.sqrt((v - mean[:, None]).pow(2).mean(1) + s["eps"])]
        return y, normed(y, s["pre"], s["pre_gamma"], s["pre_beta"]), torch.stack(parts, 1)

    # Backward: the statistics are inputs; the projection that a norm's gradient is, row by row.
    st = s["stats"].to(f8)
    out = {"x": torch.empty(rows, cols, dtype=f8, device="cuda"), "h": torch.empty(rows, cols, dtype=f8, device="cuda"),
           "pre_gamma": torch.zeros(cols, dtype=f8, device="cuda"), "post_gamma": torch.zeros(cols, dtype=f8, device="cuda")}
    if s["pre_beta"] is not None:
        out["pre_beta"] = torch.zeros(cols, dtype=f8, device="cuda")
    if s["post_beta"] is not None:
        out["post_beta"] = torch.zeros(cols, dtype=f8, device="cuda")
    if gate is not None:
        out["gate"] = torch.zeros(gate.shape, dtype=f8, device="cuda")
    step = max(1, 50_000_000 // cols)
    for a in range(0, rows, step):
        b = min(rows, a + step)
        n_hat = (s["y"][a:b].to(f8) - st[a:b, 2, None]) * st[a:b, 3, None]
        h_hat = (s["h"][a:b].to(f8) - st[a:b, 0, None]) * st[a:b, 1, None]
        dn = s["dn"][a:b].to(f8)

        def through(d, hat, rstd, kind):
            along = (d * hat).sum(1, keepdim=True) / cols
            level = d.sum(1, keepdim=True) / cols if kind == "layer" else 0.0
            return (d - level - along * hat) * rstd[:, None]

        out["pre_gamma"] += torch.einsum("rc,rc->c", dn, n_hat)
        if "pre_beta" in out:
            out["pre_beta"] += dn.sum(0)
        whole = s["dy"][a:b].to(f8) + through(dn * s["pre_gamma"].to(f8), n_hat, st[a:b, 3], s["pre"])
        out["x"][a:b] = whole * s["residual_scale"]
        branch = whole * s["block_scale"]
        if gate is not None:
            of = torch.arange(a, b, device="cuda") // (rows // gate.shape[0])
            u = h_hat * s["post_gamma"].to(f8)
            if s["post_beta"] is not None:
                u = u + s["post_beta"].to(f8)
            value = act(gate)
            slope = {"none": torch.ones_like(value), "sigmoid": value - value * value, "tanh": 1 - value * value}[case["act"]]
            out["gate"].index_add_(0, of, branch * u * slope[of])
            branch = branch * value[of]
        out["post_gamma"] += torch.einsum("rc,rc->c", branch, h_hat)
        if "post_beta" in out:
            out["post_beta"] += branch.sum(0)
        out["h"][a:b] = through(branch * s["post_gamma"].to(f8), h_hat, st[a:b, 1], s["post"])
    return out


def _exact_verify(case, s):
    tokens = s["tokens"].cpu().numpy()
    accept, sample = s["accept"].cpu().numpy().astype(np.float64), s["sample"].cpu().numpy().astype(np.float64)
    batch, drafted = tokens.shape
    out = np.full((batch, drafted + 1), -1, dtype=np.int64)
    counts = np.zeros(batch, dtype=np.int64)
    for b in range(batch):
        i = 0
        while i < drafted:
            d = int(tokens[b, i])
            q = 1.0 if s["draft"] is None else float(s["draft"][b, i, d])
            if not np.float32(accept[b, i]) * np.float32(q) < np.float32(float(s["target"][b, i, d])):
                break
            out[b, i] = d
            i += 1
        p = s["target"][b, i].double().cpu().numpy()
        w = p
        if i < drafted and s["draft"] is None:
            w = p.copy()
            w[int(tokens[b, i])] = 0.0
        elif i < drafted:
            w = np.maximum(p - s["draft"][b, i].double().cpu().numpy(), 0.0)
        if not w.sum() > 0:
            w = p
        reach = np.cumsum(w.astype(np.longdouble))
        some = np.flatnonzero(w > 0)
        out[b, i] = min(int(np.searchsorted(reach, sample[b] * reach[-1], side="right")), int(some[-1]))
        counts[b] = i
    return torch.from_numpy(out), torch.from_numpy(counts)


def exact(case, seed):
    s = prepare(case, seed)
    return {"distill": _exact_distill, "norm": _exact_norm, "verify": _exact_verify}[case["op"]](case, s)
