"""The operators of continued pre-training, as cases that can be timed and compared.

Adapting an encoder to a domain trains it on masked tokens: the hidden states at the masked positions are scored
against the whole (tied) embedding table, and the encoder's matrices move by orthogonalised momentum. A case is a dict
of plain values with a "kind":

* ``loss``: softmax cross entropy of hidden states over the vocabulary (``ops.vocab_ce``): the rows' losses, their
  log-sum-exps (both 0 where a row has no label) and the weighted total;
* ``train``: the same and its backward (``ops.vocab_ce_backward``): the hidden states' gradient, and the table's and
  the bias's, accumulated;
* ``orthogonalize``: the Newton-Schulz orthogonalisation of ``count`` matrices (``ops.orthogonalize``);
* ``muon``: one Muon step of the four matrices of each of ``layers`` encoder layers (``ops.muon``): parameters and
  momentum, updated in place.

Sizes are those of ``laya_amd.config`` (ModernBERT-base: width 768, GeGLU 1152, vocabulary 50368; ModernBERT-large:
1024, 2624; mmBERT-base: vocabulary 256000) and odd ones between. Rows are a batch's real tokens, or those of them that
carry a label (15 to 30 %); a target of -100 carries none. Hidden states are unit normal (what a LayerNorm leaves) with
a part along the target's embedding, so that the probabilities of the targets run from 1/vocabulary to nearly 1; targets
follow Zipf's law.
"""
from __future__ import annotations

import math

import torch

own = False

IGNORED = -100
# The quintic iteration's coefficients (a, b, c): X <- aX + (bA + cA²)X with A = XXᵀ.
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
MU, DECAY, RATE = 0.95, 0.01, 2e-3


def _ce(kind, name, rows, hidden, vocab, bias, labelled=1.0, weighted=False, bf16=False):
    return {"name": name, "kind": kind, "rows": rows, "hidden": hidden, "vocab": vocab, "bias": bias,
            "labelled": labelled, "weighted": weighted, "bf16": bf16}


def listed():
    return [
        # Scoring one short document's masked tokens: latency, and one pass over the table.
        _ce("loss", "loss 19x768x50368", 19, 768, 50368, True),
        # Evaluation on the real tokens of a batch of 32 x 512, 15 % of them labelled.
        _ce("loss", "loss 13871x768x50368 15%", 13871, 768, 50368, True, labelled=0.15),
        # The smallest training batch: 15 % of 4 x 128 tokens.
        _ce("train", "train 77x768x50368", 77, 768, 50368, True),
        # A micro-batch's labelled rows at ModernBERT-large's width.
        _ce("train", "train 1213x1024x50368", 1213, 1024, 50368, False),
        # 30 % of 32 x 512 tokens, gathered.
        _ce("train", "train 4915x768x50368", 4915, 768, 50368, True),
        # The same batch ungathered: every real token, most without a label.
        _ce("train", "train 13871x768x50368 30%", 13871, 768, 50368, True, labelled=0.3, weighted=True),
        # 30 % of 32 x 1024 tokens with bf16 weights (mixed precision).
        _ce("train", "train bf16 9830x768x50368", 9830, 768, 50368, False, bf16=True),
        # mmBERT's vocabulary.
        _ce("train", "train 2458x768x256000", 2458, 768, 256000, False),
        # One square matrix: latency.
        {"name": "orthogonalize 768x768", "kind": "orthogonalize", "count": 1, "rows": 768, "cols": 768},
        # The MLP input projections of six ModernBERT-large layers: tall matrices.
        {"name": "orthogonalize 6x5248x1024", "kind": "orthogonalize", "count": 6, "rows": 5248, "cols": 1024},
        # One layer's four matrices (a model trained in its last layer only).
        {"name": "muon 1 layer 768", "kind": "muon", "layers": 1, "hidden": 768, "inter": 1152},
        # Every encoder layer of ModernBERT-base.
        {"name": "muon 22 layers 768", "kind": "muon", "layers": 22, "hidden": 768, "inter": 1152},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["loss", "train", "train", "train", "orthogonalize", "muon"])
    if kind in ("loss", "train"):
        hidden = rng.choice([768, 768, 1024, 1024, rng.randint(33, 1100)])
        vocab = rng.choice([50368, 50368, 256000, _log(rng, 1000, 60000)])
        rows = _log(rng, 1, min(16384, 4.8e11 / (vocab * hidden)))
        return {k: v for k, v in _ce(kind, "", rows, hidden, vocab, rng.random() < 0.5,
                                     labelled=rng.choice([1.0, 1.0, 0.3, 0.15]), weighted=rng.random() < 0.3,
                                     bf16=rng.random() < 0.3).items() if k != "name"}
    if kind == "orthogonalize":
        rows, cols = rng.choice([(768, 768), (2304, 768), (768, 1152), (1024, 1024), (5248, 1024), (1024, 2624),
                                 (_log(rng, 17, 2000), _log(rng, 17, 2000)), (_log(rng, 17, 2000), _log(rng, 17, 2000))])
        return {"kind": kind, "count": _log(rng, 1, min(28, max(1, 3.0e10 / (rows * cols * min(rows, cols))))),
                "rows": rows, "cols": cols}
    hidden = rng.choice([768, 768, 64 * rng.randint(2, 12)])
    return {"kind": kind, "layers": _log(rng, 1, 22), "hidden": hidden, "inter": hidden * 3 // 2}


# ------------------------------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 6151 + 29)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _ce_inputs(case, seed):
    g = _generator(seed)
    rows, hidden, vocab = case["rows"], case["hidden"], case["vocab"]
    weight = _normal(g, vocab, hidden) * 0.02
    if case["bf16"]:
        weight = weight.bfloat16()
    zipf = torch.exp(_rand(g, rows) * math.log(vocab + 1)).long() - 1
    targets = zipf.clamp_(0, vocab - 1)
    # A logit gains c·|w|² from c·w along its own row: between nothing and a little over log(vocabulary).
    along = _rand(g, rows, 1) * (1.2 * math.log(vocab) / (hidden * 0.02 ** 2))
    x = _normal(g, rows, hidden) + along * weight[targets].float()
    targets = torch.where(_rand(g, rows) < case["labelled"], targets, IGNORED)
    labels = max(1, int((targets >= 0).sum()))
    return {"x": x, "weight": weight, "bias": 0.05 * _normal(g, vocab) if case["bias"] else None,
            "targets": targets.int(), "scale": 1.0 / labels,
            "row_weights": 0.25 + _rand(g, rows) if case["weighted"] else None}


def _update(g, *shape):
    """A gradient-like matrix: a few strong directions over noise, columns of unequal size."""
    count, rows, cols = shape
    rank = max(1, min(rows, cols) // 16)
    strong = torch.bmm(_normal(g, count, rows, rank), _normal(g, count, rank, cols)) / math.sqrt(rank)
    return 1e-4 * (0.5 * strong + _normal(g, *shape)) * torch.exp(0.5 * _normal(g, 1, 1, cols))


def _matrix_shapes(case):
    h, i = case["hidden"], case["inter"]
    return [(3 * h, h), (h, h), (2 * i, h), (h, i)]  # Wqkv, Wo, mlp.Wi, mlp.Wo


def _muon_inputs(case, seed):
    g, layers = _generator(seed), case["layers"]
    shapes = _matrix_shapes(case)
    total = layers * sum(r * c for r, c in shapes)
    d = {k: torch.empty(total, device="cuda") for k in ("params", "grads", "momentum")}
    at, offsets, rows, cols = 0, [], [], []
    for r, c in shapes:  # the layers' matrices of one shape lie together
        n = layers * r * c
        d["params"][at:at + n] = (0.02 * _normal(g, layers, r, c)).view(-1)
        d["grads"][at:at + n] = _update(g, layers, r, c).view(-1)
        d["momentum"][at:at + n] = 4 * _update(g, layers, r, c).view(-1)
        offsets += [at + k * r * c for k in range(layers)]
        rows += [r] * layers
        cols += [c] * layers
        at += n
    return {**d, "offsets": offsets, "rows": rows, "cols": cols,
            "multipliers": [0.2 * math.sqrt(max(r, c)) for r, c in zip(rows, cols)]}


def _inputs(case, seed):
    if case["kind"] in ("loss", "train"):
        return _ce_inputs(case, seed)
    if case["kind"] == "muon":
        return _muon_inputs(case, seed)
    return {"x": _update(_generator(seed), case["count"], case["rows"], case["cols"])}


# ------------------------------------------------------------------------------------ the framework

_contexts = {}


def _context():
    from laya_amd.device import Context
    if not _contexts:
        _contexts[0] = Context(0)
    return _contexts[0]


def _array(ctx, t):
    """A tensor's memory as the library's functions take it."""
    import numpy as np
    from laya_amd.device import DeviceArray
    kinds = {torch.float32: np.float32, torch.int32: np.int32, torch.bfloat16: np.uint16}
    return None if t is None else DeviceArray.borrow(ctx, t.data_ptr(), tuple(t.shape), kinds[t.dtype], owner=t)


def prepare(case, seed):
    kind = case["kind"]
    s = {"kind": kind, "case": case, **_inputs(case, seed)}
    if kind in ("loss", "train"):
        rows, hidden, vocab = case["rows"], case["hidden"], case["vocab"]
        s["row_loss"], s["lse"] = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
        s["loss"] = torch.zeros(1, device="cuda")
        if kind == "train":
            s["dx"] = torch.zeros(rows, hidden, device="cuda")
            s["dweight"] = torch.zeros(vocab, hidden, device="cuda")
            s["dbias"] = torch.zeros(vocab, device="cuda") if case["bias"] else None
    elif kind == "orthogonalize":
        s["out"] = torch.zeros_like(s["x"])
    if own:
        from laya_amd import ops
        ctx = _context()
        a = {k: _array(ctx, v) for k, v in s.items() if isinstance(v, torch.Tensor)}
        s["arrays"] = a
        if kind in ("loss", "train"):
            values = None if case["bf16"] else a["weight"]
            s["W"] = ops.Parameter.borrow(ctx, "decoder.weight", (case["vocab"], case["hidden"]), values,
                                          a.get("dweight"))
            s["b"] = ops.Parameter.borrow(ctx, "decoder.bias", (case["vocab"],), a["bias"],
                                          a.get("dbias")) if case["bias"] else None
            s["weight16"] = a["weight"] if case["bf16"] else None
        elif kind == "muon":
            s["matrices"] = ops.MuonMatrices(ctx, s["offsets"], s["rows"], s["cols"], s["multipliers"])
    return s


def _run_own(s):
    from laya_amd import ops
    kind, case, a = s["kind"], s["case"], s["arrays"]
    if kind in ("loss", "train"):
        ops.vocab_ce(s["W"], s["b"], a["x"], a["targets"], case["rows"], a["row_loss"], a["lse"],
                     row_weights=a.get("row_weights"), scale=s["scale"], loss=a["loss"], weight16=s["weight16"])
        out = {k: s[k] for k in ("row_loss", "lse", "loss")}
        if kind == "train":
            ops.vocab_ce_backward(s["W"], s["b"], a["x"], a["targets"], case["rows"], a["lse"], a["dx"],
                                  row_weights=a.get("row_weights"), scale=s["scale"], weight16=s["weight16"])
            out.update({k: s[k] for k in ("dx", "dweight", "dbias") if s[k] is not None})
        return out
    if kind == "orthogonalize":
        ops.orthogonalize(_context(), a["x"], case["count"], case["rows"], case["cols"], a["out"], steps=STEPS)
        return {"out": s["out"]}
    ops.muon(s["matrices"], a["params"], a["grads"], a["momentum"], learning_rate=RATE, mu=MU, nesterov=True,
             weight_decay=DECAY, steps=STEPS)
    return {"params": s["params"], "momentum": s["momentum"]}


# ----------------------------------------------------------------------------------- the plain form

def _plain_ce(s):
    x, targets, w = s["x"], s["targets"].long(), s["weight"].float()
    labelled = targets >= 0
    at = targets.clamp(min=0)[:, None]
    logits = x @ w.t()
    if s["bias"] is not None:
        logits += s["bias"]
    top = logits.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(logits - top).sum(1, keepdim=True))
    row_loss = torch.where(labelled, (lse - logits.gather(1, at))[:, 0], 0.0)
    each = torch.full_like(row_loss, s["scale"]) if s["row_weights"] is None else s["row_weights"] * s["scale"]
    each = torch.where(labelled, each, 0.0)
    s["row_loss"].copy_(row_loss)
    s["lse"].copy_(torch.where(labelled, lse[:, 0], 0.0))
    s["loss"].copy_((each.double() * row_loss.double()).sum())
    out = {"row_loss": s["row_loss"], "lse": s["lse"], "loss": s["loss"]}
    if s["kind"] == "train":
        d = torch.exp(logits - lse)
        d.scatter_add_(1, at, torch.full_like(lse, -1.0))
        d *= each[:, None]
        s["dx"].copy_(d @ w)
        s["dweight"] += d.t() @ x
        out.update(dx=s["dx"], dweight=s["dweight"])
        if s["bias"] is not None:
            s["dbias"] += d.sum(0)
            out["dbias"] = s["dbias"]
    return out


def _orthogonal(u):
    """The orthogonalisation of a batch of matrices, in u's precision (the norms in 64 bits)."""
    a, b, c = COEFFICIENTS
    tall = u.shape[1] > u.shape[2]
    norm = u.double().square().sum((1, 2), keepdim=True).sqrt()
    x = (u / torch.where(norm > 0, norm, 1.0)).to(u.dtype)
    x = x.transpose(1, 2).contiguous() if tall else x
    for _ in range(STEPS):
        g = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * g + c * torch.bmm(g, g), x)
    return x.transpose(1, 2) if tall else x


def _muon_groups(s):
    """(first element, matrices, rows, cols) of each shape's run of matrices."""
    layers, at, groups = s["case"]["layers"], 0, []
    for r, c in _matrix_shapes(s["case"]):
        groups.append((at, layers, r, c))
        at += layers * r * c
    return groups


def _plain_muon(s):
    m, g, p = s["momentum"], s["grads"], s["params"]
    m.mul_(MU).add_(g)
    u = g + MU * m
    for at, n, r, c in _muon_groups(s):
        here = slice(at, at + n * r * c)
        step = RATE * 0.2 * math.sqrt(max(r, c))
        p[here] = p[here] * (1 - RATE * DECAY) - step * _orthogonal(u[here].view(n, r, c)).reshape(-1)
    return {"params": p, "momentum": m}


def run(state):
    if own:
        return _run_own(state)
    if state["kind"] in ("loss", "train"):
        return _plain_ce(state)
    if state["kind"] == "orthogonalize":
        state["out"].copy_(_orthogonal(state["x"]))
        return {"out": state["out"]}
    return _plain_muon(state)


# ------------------------------------------------------------------------------------------- exact

def _exact_ce(case, seed):
    """By pieces of rows, in 64 bits."""
    i = _ce_inputs(case, seed)
    x, w, t = i["x"].double(), i["weight"].double(), i["targets"].long()
    rows, train = case["rows"], case["kind"] == "train"
    has = t != IGNORED
    weight = torch.zeros(rows, dtype=torch.float64, device="cuda")
    weight[has] = i["scale"]
    if i["row_weights"] is not None:
        weight *= i["row_weights"].double()
    row_loss, lse = torch.zeros_like(weight), torch.zeros_like(weight)
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(w[:, 0])
    piece = max(1, (1 << 29) // case["vocab"])
    for r0 in range(0, rows, piece):
        r = slice(r0, min(rows, r0 + piece))
        z = torch.matmul(x[r], w.t())
        if i["bias"] is not None:
            z = z + i["bias"].double()
        norm = torch.logsumexp(z, 1)
        lse[r] = torch.where(has[r], norm, 0.0)
        n = torch.arange(z.shape[0], device="cuda")
        picked = z[n, t[r].clamp(min=0)]
        row_loss[r] = torch.where(has[r], norm - picked, 0.0)
        if train:
            z = torch.exp(z - norm[:, None])
            z[n, t[r].clamp(min=0)] -= 1.0
            z = z * weight[r, None]
            dx[r] = torch.matmul(z, w)
            dw += torch.matmul(z.t(), x[r])
            db += z.sum(0)
    out = {"row_loss": row_loss, "lse": lse, "loss": (weight * row_loss).sum().view(1)}
    if train:
        out.update(dx=dx, dweight=dw)
        if i["bias"] is not None:
            out["dbias"] = db
    return out


def _exact_orthogonal(u):
    """One matrix in 64 bits, the iteration on its own side: X <- X(aI + bS + cS²) with S = XᵀX when tall."""
    a, b, c = COEFFICIENTS
    x = u.double()
    norm = torch.linalg.norm(x)
    x = x / norm if norm > 0 else x
    for _ in range(STEPS):
        if x.shape[0] > x.shape[1]:
            s = x.t() @ x
            x = a * x + x @ (b * s + c * (s @ s))
        else:
            s = x @ x.t()
            x = a * x + (b * s + c * (s @ s)) @ x
    return x


def exact(case, seed):
    if case["kind"] in ("loss", "train"):
        return _exact_ce(case, seed)
    if case["kind"] == "orthogonalize":
        return {"out": torch.stack([_exact_orthogonal(u) for u in _inputs(case, seed)["x"]])}
    i = _muon_inputs(case, seed)
    m = i["momentum"].double() * MU + i["grads"].double()
    u = i["grads"].double() + MU * m
    p = i["params"].double()
    for at, r, c, k in zip(i["offsets"], i["rows"], i["cols"], i["multipliers"]):
        here = slice(at, at + r * c)
        p[here] = p[here] * (1 - RATE * DECAY) - RATE * k * _exact_orthogonal(u[here].view(r, c)).reshape(-1)
    return {"params": p, "momentum": m}


# -------------------------------------------------------------------------------------------- work

def _iteration_flops(rows, cols):
    """One step on the matrix's short side n and long side m: A (one triangle of it), A² (the same), and (bA + cA²)X."""
    n, m = min(rows, cols), max(rows, cols)
    return n * (n + 1) * m + n * (n + 1) * n + 2 * n * n * m


def work(case):
    kind = case["kind"]
    if kind in ("loss", "train"):
        rows, hidden, vocab = case["rows"], case["hidden"], case["vocab"]
        labels = max(1, round(rows * case["labelled"]))
        product = 2.0 * labels * hidden * vocab
        table, each = (2 if case["bf16"] else 4) * vocab * hidden, 4 * labels * hidden
        nbytes = table + each + (4 * vocab if case["bias"] else 0) + 4 * rows * (4 if case["weighted"] else 3)
        if kind == "loss":
            return {"bytes": nbytes, "flops": product}
        nbytes += 4 * rows * hidden + 8 * vocab * hidden + (8 * vocab if case["bias"] else 0)
        return {"bytes": nbytes, "flops": 3 * product}
    if kind == "orthogonalize":
        n = case["count"] * case["rows"] * case["cols"]
        return {"bytes": 8 * n, "flops": STEPS * case["count"] * _iteration_flops(case["rows"], case["cols"])}
    shapes = _matrix_shapes(case)
    n = case["layers"] * sum(r * c for r, c in shapes)
    return {"bytes": 20 * n, "flops": STEPS * case["layers"] * sum(_iteration_flops(r, c) for r, c in shapes)}
