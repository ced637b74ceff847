"""More operators of a training pass, as cases that can be timed and checked: its first, the token embedding, with its
gradient, and its last, the update of the weight matrices.

A case is a dict of plain values.  Its ``kind`` names the operator:

* ``lookup``      ``ops.embedding``: scaled rows of the table;
* ``gradient``    ``ops.embedding_grad``: the table's gradient, new or added to the one of the tied head;
* ``embed``       ``ops.embedding`` and torch's backward over it;
* ``orthogonal``  ``ops.newton_schulz``: a batch of matrices orthogonalised by Newton-Schulz products;
* ``update``      ``ops.muon_step``: momentum, Newton-Schulz products and the weights' update, in place, over a list of
                  matrices.

``listed`` holds the named cases, ``draw`` more of the same ranges, ``prepare`` makes what a program holds before the call,
``run`` is one pass -- through the framework where ``own`` is true, else in elementary torch operations -- and ``exact`` the
same outputs in float64.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
VOCAB = 20480  # the benchmark's vocabulary
STEPS = 5
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01

# The largest listed cases; a drawn one costs no more.
ROWS_MOST = 32 * 8192 * 1024
TABLE_MOST = 65536 * 640
MATRIX_MOST = 24 * (3 * 1024 * 1024 * 4096 + 1024**3)


def listed() -> list:
    token = dict(type="f32", scale=1.0, padding=False, skew=3.0)
    return [
        # The smallest call: the embedding of one short phrase of the tiny model, where the launch counts.
        dict(token, kind="lookup", name="lookup_16", rows=16, vocab=512, cols=128),
        # A training step's batch of the default model, rows scaled by the root of their width.
        dict(token, kind="lookup", name="lookup_8x2048", rows=16384, vocab=VOCAB, cols=640, scale=25.298221281347036),
        # Its gradient, added to the one that the tied head left; few tokens make up most of the music.
        dict(token, kind="gradient", name="gradient_8x2048", rows=16384, vocab=VOCAB, cols=640, add=True),
        # A ragged batch over the default vocabulary (odd sizes), its padded tail without a gradient.
        dict(token, kind="gradient", name="gradient_bf16_673", type="bf16", rows=4111, vocab=673, cols=333, padding=True, add=False),
        # The wide model's batch: the longest runs of one token.
        dict(token, kind="gradient", name="gradient_32x8192", type="bf16", rows=262144, vocab=VOCAB, cols=1024, add=False),
        # The operator inside a program of torch's: ragged pieces of the wide model's sequences, lookup and backward.
        dict(token, kind="embed", name="embed_autograd", rows=2331, vocab=VOCAB, cols=1024),
        # One low-rank matrix of the default model: the smallest update, launches and latency.
        dict(kind="orthogonal", name="orthogonal_640x64", type="f32", count=1, rows=640, cols=64),
        # A square projection of all layers of the default model.
        dict(kind="orthogonal", name="orthogonal_14x640", type="f32", count=14, rows=640, cols=640),
        # One odd matrix in the gradients' type.
        dict(kind="orthogonal", name="orthogonal_bf16_odd", type="bf16", count=1, rows=333, cols=1111),
        # The widening half of the default model's feed-forward parts.
        dict(kind="orthogonal", name="orthogonal_ffn", type="bf16", count=14, rows=2560, cols=640),
        # The update of the default model's square projections, four to a layer: a list of weights.
        dict(kind="update", name="update_56x640", type="f32", count=56, rows=640, cols=640),
        # The narrowing half of the wide model's feed-forward parts, bf16 weights and gradients: the largest.
        dict(kind="update", name="update_wide_ffn", type="bf16", count=24, rows=1024, cols=4096),
    ]


def _log_int(rng: random.Random, low: int, high: int) -> int:
    high = max(low, high)
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["lookup", "gradient", "gradient", "embed", "orthogonal", "orthogonal", "update", "update"])
    if kind in ("lookup", "gradient", "embed"):
        cols = rng.choice([128, 640, 1024, _log_int(rng, 1, 2048)])
        vocab = rng.choice([673, VOCAB, _log_int(rng, 1, 65536)])
        case = dict(kind=kind, type=rng.choice(["f32", "bf16"]), scale=rng.choice([1.0, math.sqrt(cols)]), padding=rng.random() < 0.4,
                    skew=rng.choice([1.0, 3.0, 8.0]), rows=_log_int(rng, 1, min(262144, ROWS_MOST // cols)),
                    vocab=min(vocab, TABLE_MOST // cols), cols=cols)
        if kind == "gradient":
            case["add"] = rng.random() < 0.5
        return case
    rows, cols = (rng.choice([640, 1024, _log_int(rng, 1, 2560), _log_int(rng, 1, 2560)]) for _ in range(2))
    p, q = min(rows, cols), max(rows, cols)
    count = _log_int(rng, 1, min(64, MATRIX_MOST // (3 * p * p * q + p**3)))
    return dict(kind=kind, type=rng.choice(["f32", "bf16"]), count=count, rows=rows, cols=cols)


# ------------------------------------------------------------------------------------------------------------------ inputs
def _inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind = torch.bfloat16 if case["type"] == "bf16" else torch.float32

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    if case["kind"] in ("lookup", "gradient", "embed"):
        M, V, D = (case[k] for k in ("rows", "vocab", "cols"))
        # Token frequencies fall with the id as a power: skew 1 is uniform, from 3 on few ids take most places.
        u = torch.rand(M, generator=gen, device=DEVICE, dtype=torch.float64)
        tokens = (u**case["skew"] * V).long().clamp_(max=V - 1)
        if case["padding"]:
            tokens[M - M // 5 :] = 0
        s = dict(tokens=tokens, scale=case["scale"], padding=0 if case["padding"] else None, vocab=V)
        if case["kind"] != "gradient":
            s["weight"] = (0.02 * normal(V, D)).to(kind)
        if case["kind"] != "lookup":
            s["dout"] = normal(M, D).to(kind)
        if case["kind"] == "gradient":
            s["out"] = normal(V, D).to(kind) if case["add"] else None
        return s
    B, R, C = (case[k] for k in ("count", "rows", "cols"))

    def gradient():  # a few strong directions over noise, as a batch's gradients are
        few = max(1, min(R, C) // 16)
        strong = torch.matmul(normal(B, R, few) * torch.logspace(0.0, -2.0, few, device=DEVICE), normal(B, few, C))
        return (1e-3 * (strong + 0.1 * normal(B, R, C))).to(kind)

    if case["kind"] == "orthogonal":
        return dict(x=gradient())
    return dict(params=(normal(B, R, C) / math.sqrt(C)).to(kind), grads=gradient(), momenta=gradient().float())


def prepare(case: dict, seed: int) -> dict:
    state = _inputs(case, seed)
    if case["kind"] == "embed":
        state["weight"].requires_grad_()
    if case["kind"] == "update":  # the program's weights, gradients and momenta: views into one buffer each
        state["lists"] = [list(state[k].unbind(0)) for k in ("params", "grads", "momenta")]
    return dict(state, case=case)


# -------------------------------------------------------------------------------------------------------------------- pass
def run(state: dict):
    kind = state["case"]["kind"]
    if kind == "lookup":
        return _lookup(state)
    if kind == "gradient":
        return _gradient(state)
    if kind == "embed":
        return _embed(state)
    if kind == "orthogonal":
        return _orthogonal(state)
    return _update(state)


def _lookup(s: dict):
    if own:
        from yufmusicgen_amd import ops

        return ops.embedding(s["tokens"], s["weight"], scale=s["scale"], padding_idx=s["padding"])
    return (s["weight"][s["tokens"]].float() * s["scale"]).to(s["weight"].dtype)


def _gradient(s: dict):
    if own:
        from yufmusicgen_amd import ops

        return ops.embedding_grad(s["tokens"], s["dout"], s["vocab"], scale=s["scale"], padding_idx=s["padding"], out=s["out"])
    grad = _gradient_plain(s)
    if s["out"] is None:
        return grad.to(s["dout"].dtype)
    return s["out"].copy_(s["out"].float() + grad)


def _gradient_plain(s: dict):
    """The rows of dout summed by their tokens in float32."""
    dout = s["dout"].float()
    if s["padding"] is not None:
        dout = torch.where((s["tokens"] != s["padding"])[:, None], dout, 0.0)
    total = torch.zeros(s["vocab"], dout.shape[1], device=dout.device)
    return total.index_add_(0, s["tokens"], dout) * s["scale"]


def _embed(s: dict) -> dict:
    if own:
        from yufmusicgen_amd import ops

        out = ops.embedding(s["tokens"], s["weight"], scale=s["scale"], padding_idx=s["padding"])
        (grad,) = torch.autograd.grad(out, s["weight"], s["dout"])
        return dict(out=out.detach(), grad=grad)
    with torch.no_grad():
        return dict(out=_lookup(s), grad=_gradient_plain(s).to(s["dout"].dtype))


def _newton_schulz_plain(x):
    """X <- a X + (b A + c A A) X with A = X X^T, from x over its Frobenius norm, in float32; of the transpose where there are
    more rows than columns."""
    a, b, c = COEFFICIENTS
    wide = x.shape[-2] <= x.shape[-1]
    X = x.float() if wide else x.float().transpose(-1, -2).contiguous()
    norm = X.double().square().sum((-1, -2), keepdim=True).sqrt()
    X = (X / (norm + EPS)).float()
    for _ in range(STEPS):
        A = torch.matmul(X, X.transpose(-1, -2).contiguous())
        X = a * X + torch.matmul(b * A + c * torch.matmul(A, A), X)
    return X if wide else X.transpose(-1, -2)


def _orthogonal(s: dict):
    if own:
        from yufmusicgen_amd import ops

        return ops.newton_schulz(s["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    return _newton_schulz_plain(s["x"]).to(s["x"].dtype).contiguous()


def _update(s: dict) -> dict:
    params, grads, momenta = s["params"], s["grads"], s["momenta"]
    if own:
        from yufmusicgen_amd import ops

        ops.muon_step(*s["lists"], LR, momentum=MOMENTUM, nesterov=True, weight_decay=DECAY, steps=STEPS,
                      coefficients=COEFFICIENTS, eps=EPS)
    else:
        rows, cols = params.shape[-2:]
        g = grads.float()
        momenta.copy_(MOMENTUM * momenta + (1.0 - MOMENTUM) * g)
        step = _newton_schulz_plain((1.0 - MOMENTUM) * g + MOMENTUM * momenta)
        params.copy_(params.float() * (1.0 - LR * DECAY) - LR * math.sqrt(max(1.0, rows / cols)) * step)
    return dict(params=params, momenta=momenta)


# -------------------------------------------------------------------------------------------------------------------- work
def work(case: dict) -> dict:
    """Every input read once and every output written once; the operations of the definition, a symmetric product's half."""
    size = 2 if case["type"] == "bf16" else 4
    if case["kind"] in ("lookup", "gradient", "embed"):
        M, V, D = (case[k] for k in ("rows", "vocab", "cols"))
        look = size * D * (min(M, V) + M) + 8 * M
        grad = size * D * (M + V * (2 if case.get("add") else 1)) + 8 * M
        if case["kind"] == "lookup":
            return dict(bytes=look, flops=M * D)
        return dict(bytes=grad + (look if case["kind"] == "embed" else 0), flops=M * D)
    B, R, C = (case[k] for k in ("count", "rows", "cols"))
    p, q = min(R, C), max(R, C)
    flops = B * STEPS * (3 * p * p * q + p**3)
    if case["kind"] == "orthogonal":
        return dict(bytes=2 * size * B * R * C, flops=flops)
    return dict(bytes=B * R * C * (3 * size + 8), flops=flops)


# ------------------------------------------------------------------------------------------------------------------- exact
def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    if case["kind"] in ("lookup", "gradient", "embed"):
        grad = None
        if case["kind"] != "lookup":
            V, D = case["vocab"], case["cols"]
            grad = torch.zeros(V, D, dtype=torch.float64, device=DEVICE)
            for t, g in zip(s["tokens"].split(32768), s["dout"].split(32768)):
                keep = t >= 0 if s["padding"] is None else t != s["padding"]
                grad.index_put_((t[keep],), g[keep].double(), accumulate=True)
            grad = grad * case["scale"]
            if case.get("add"):
                grad = grad + s["out"].double()
        if case["kind"] == "gradient":
            return grad
        out = torch.nn.functional.embedding(s["tokens"], s["weight"].double()) * case["scale"]
        return out if case["kind"] == "lookup" else dict(out=out, grad=grad)
    if case["kind"] == "orthogonal":
        return _newton_schulz_exact(s["x"].double())
    params, grads, momenta = (s[k].double() for k in ("params", "grads", "momenta"))
    momenta = torch.lerp(grads, momenta, MOMENTUM)
    step = _newton_schulz_exact(torch.lerp(grads, momenta, MOMENTUM))
    step = step * max(1.0, case["rows"] / case["cols"]) ** 0.5
    return dict(params=params - LR * (DECAY * params + step), momenta=momenta)


def _newton_schulz_exact(x):
    """The polynomial on the smaller side's Gram matrix, in float64."""
    a, b, c = COEFFICIENTS
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + EPS)
    eye = torch.eye(min(x.shape[-2:]), dtype=x.dtype, device=x.device)
    left = x.shape[-2] <= x.shape[-1]
    for _ in range(STEPS):
        gram = x @ x.mT if left else x.mT @ x
        poly = a * eye + (b * eye + c * gram) @ gram
        x = poly @ x if left else x @ poly
    return x
