"""The operators of a training pass, as cases that can be timed and checked.

A case is a dict of plain values.  Its ``kind`` names the operator:

* ``wkv``      the gradients of the WKV-7 scan: ``ops.rwkv7_scan_backward``, or, with ``through`` "autograd",
               ``ops.rwkv7_scan`` and torch's backward over it;
* ``rosa``     the gradients of the ROSA Householder scan: ``ops.rosa_householder_scan_backward``, or
               ``ops.rosa_householder_scan`` and torch's backward;
* ``dropout``  ``ops.dropout`` with its mask from a counter-based generator, alone (as the gradient takes it) or added to
               the residual stream (as the forward pass takes it);
* ``loss``     the cross-entropy of logits and token ids: ``ops.cross_entropy`` (the loss alone) or
               ``ops.cross_entropy_grad`` (the loss and the logits' gradient).

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
HEAD_SIZES = (8, 16, 32, 40, 48, 64, 128)  # the WKV-7 scan's
IGNORE = -100
DECAY_RATE = math.exp(-0.5)  # d = exp(-e^{-1/2} sigmoid(w))

# The largest listed cases; a drawn one costs no more.
WKV_MOST = 8 * 2048 * 16 * 40 * 40  # state elements over all tokens
ROSA_MOST = 8 * 2048 * 128
DROPOUT_MOST = 16384 * 640
LOSS_MOST = 16384 * VOCAB
STEPS_MOST = 2048  # a training context


def listed() -> list:
    wkv = dict(kind="wkv", heads=16, state=False, through="call")
    rosa = dict(kind="rosa", gated=True, state=False, through="call")
    drop = dict(kind="dropout", type="f32", p=0.1, residual=True)
    loss = dict(kind="loss", type="f32", ignored=0.05, grad=True, reduction="mean")
    return [
        # The smallest call: one short phrase of the tiny model, where launches and latency count.
        dict(wkv, name="wkv_16_tokens", batch=1, tokens=16, heads=4, size=32),
        # A training step's batch of the default model at its full context.
        dict(wkv, name="wkv_8x2048", batch=8, tokens=2048, size=40),
        # Ragged pieces of the wide model's sequences, trained through a carried state.
        dict(wkv, name="wkv_ragged_state", batch=3, tokens=777, size=64, state=True),
        # One long piece alone: few heads, so the work has to be split along the sequence.
        dict(wkv, name="wkv_one_sequence", batch=1, tokens=2048, size=64),
        # The operator inside a program of torch's: two sequences (what the reference trains on 8 GB), scan and backward.
        dict(wkv, name="wkv_autograd", batch=2, tokens=1024, size=40, through="autograd"),
        # ROSA beside the above: the default model's batch with the read gate in the scan,
        dict(rosa, name="rosa_8x2048", batch=8, tokens=2048, dim=128),
        # and the wide model's memory, ungated and from a carried memory, ragged.
        dict(rosa, name="rosa_ragged_state", batch=3, tokens=777, dim=256, gated=False, state=True),
        # The residual stream of that batch: dropout and sum in the forward pass,
        dict(drop, name="dropout_residual", rows=16384, cols=640),
        # and the gradient of an odd-sized bf16 activation: the same mask again, without the residual.
        dict(drop, name="dropout_bf16_odd", type="bf16", rows=1111, cols=333, p=0.25, residual=False),
        # The loss of that batch over the benchmark's vocabulary, with the logits' gradient.
        dict(loss, name="loss_16384", rows=16384, vocab=VOCAB),
        # bf16 logits of a ragged batch over the default vocabulary (an odd one: rows lie on odd addresses).
        dict(loss, name="loss_bf16_673", type="bf16", rows=4111, vocab=673, reduction="sum"),
        # A validation step of few positions: their losses alone.
        dict(loss, name="loss_only_64", rows=64, vocab=VOCAB, grad=False, ignored=0.0, reduction="none"),
    ]


def _log_int(rng: random.Random, low: int, high: int) -> int:
    high = max(low, high)
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["wkv", "wkv", "rosa", "rosa", "dropout", "loss", "loss"])
    through = rng.choice(["call", "call", "autograd"])
    if kind == "wkv":
        size = rng.choice(HEAD_SIZES)
        tokens = _log_int(rng, 1, STEPS_MOST)
        heads = _log_int(rng, 1, min(32, WKV_MOST // (tokens * size * size)))
        batch = _log_int(rng, 1, min(32, WKV_MOST // (tokens * size * size * heads)))
        return dict(kind="wkv", batch=batch, tokens=tokens, heads=heads, size=size, state=rng.random() < 0.5, through=through)
    if kind == "rosa":
        dim = rng.choice([64, 128, 256, _log_int(rng, 1, 1024)])
        tokens = _log_int(rng, 1, STEPS_MOST)
        batch = _log_int(rng, 1, min(64, ROSA_MOST // (tokens * dim)))
        return dict(kind="rosa", batch=batch, tokens=tokens, dim=dim, gated=rng.random() < 0.5, state=rng.random() < 0.5,
                    through=through)
    if kind == "dropout":
        cols = rng.choice([640, 1024, _log_int(rng, 1, 4096)])
        return dict(kind="dropout", type=rng.choice(["f32", "bf16"]), rows=_log_int(rng, 1, DROPOUT_MOST // cols), cols=cols,
                    p=rng.choice([0.0, 0.05, 0.1, 0.25, 0.5, 0.9]), residual=rng.random() < 0.5)
    vocab = rng.choice([673, VOCAB, _log_int(rng, 2, 65536)])
    return dict(kind="loss", type=rng.choice(["f32", "bf16"]), rows=_log_int(rng, 1, min(16384, LOSS_MOST // vocab)), vocab=vocab,
                ignored=rng.choice([0.0, 0.05, 0.5]), grad=rng.random() < 0.75, reduction=rng.choice(["mean", "sum", "none"]))


# ------------------------------------------------------------------------------------------------------------------ inputs
def _inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    if case["kind"] == "wkv":
        B, T, H, N = (case[k] for k in ("batch", "tokens", "heads", "size"))
        kappa = normal(B, T, H, N)
        kappa /= kappa.norm(dim=-1, keepdim=True)
        # As the block makes them: a = -kappa, b = kappa sigmoid(z), decays over the whole of (0.545, 1).
        s = dict(r=normal(B, T, H, N), w=normal(B, T, H, N) * 1.5 - 1.0, k=normal(B, T, H, N), v=normal(B, T, H, N), a=-kappa,
                 b=kappa * torch.sigmoid(normal(B, T, H, N)), dy=normal(B, T, H, N))
        s["state"] = normal(B, H, N, N) if case["state"] else None
        s["dstate"] = normal(B, H, N, N) if case["state"] or case["through"] == "autograd" else None
        return s
    if case["kind"] == "rosa":
        B, T, D = (case[k] for k in ("batch", "tokens", "dim"))
        u = normal(D)
        return dict(cand=normal(B, T, D), write=normal(B, T, D), read_raw=normal(B, T, D),
                    decay=torch.sigmoid(2.0 + 0.5 * normal(D)), direction=u / u.norm(),
                    memory=normal(B, D) if case["state"] else torch.zeros(B, D, device=DEVICE), dread=normal(B, T, D),
                    dmemory=normal(B, D))
    kind = torch.bfloat16 if case["type"] == "bf16" else torch.float32
    if case["kind"] == "dropout":
        shape = (case["rows"], case["cols"])
        return dict(x=normal(*shape).to(kind), residual=normal(*shape).to(kind) if case["residual"] else None, p=case["p"],
                    seed=random.Random(seed).getrandbits(63), counter=7 * seed + 3)
    M, V = case["rows"], case["vocab"]
    targets = torch.randint(0, V, (M,), generator=gen, device=DEVICE)
    ignored = torch.rand(M, generator=gen, device=DEVICE) < case["ignored"]
    ignored[0] = False  # a mean has something to average
    return dict(logits=(3.0 * normal(M, V)).to(kind), targets=torch.where(ignored, IGNORE, targets))


def prepare(case: dict, seed: int) -> dict:
    state = _inputs(case, seed)
    if case.get("through") == "autograd":
        for name in _leaves(case):
            state[name].requires_grad_()
    return dict(state, case=case)


def _leaves(case: dict) -> list:
    """What a pass through autograd takes gradients of."""
    if case["kind"] == "wkv":
        return ["r", "w", "k", "v", "a", "b"] + (["state"] if case["state"] else [])
    return ["cand", "write"] + (["read_raw"] if case["gated"] else []) + ["decay", "direction", "memory"]


# -------------------------------------------------------------------------------------------------------------------- pass
def run(state: dict):
    case = state["case"]
    if case["kind"] == "wkv":
        return _wkv(state, case)
    if case["kind"] == "rosa":
        return _rosa(state, case)
    if case["kind"] == "dropout":
        return _dropout(state)
    return _loss(state, case)


def _wkv(s: dict, case: dict) -> dict:
    x = [s[k] for k in ("r", "w", "k", "v", "a", "b")]
    if own:
        from yufmusicgen_amd import ops

        if case["through"] == "autograd":
            y, final = ops.rwkv7_scan(*x, state=s["state"])
            grads = torch.autograd.grad((y, final), [s[k] for k in _leaves(case)], (s["dy"], s["dstate"]))
            return dict(y=y.detach(), final=final.detach(), grads=list(grads))
        grads = ops.rwkv7_scan_backward(*x, s["dy"], state=s["state"], dstate=s["dstate"])
        return dict(grads=list(grads[: 7 if case["state"] else 6]))
    with torch.no_grad():
        y, final, grads = _wkv_plain(x, s["dy"], s["state"], s["dstate"])
    if case["through"] == "autograd":
        return dict(y=y, final=final, grads=grads)
    return dict(grads=grads)


def _wkv_plain(x, dy, state, dstate):
    """S_t = S_{t-1} diag(d_t) + (S_{t-1} a_t) b_t^T + v_t k_t^T, y_t = S_t r_t, and the adjoint recurrence
    G_{t-1} = G_t diag(d_t) + (G_t b_t) a_t^T with G_t += dy_t r_t^T.  Only the two recurrences go token by token."""
    r, w, k, v, a, b = x
    B, T, H, N = r.shape
    sig = 1.0 / (1.0 + torch.exp(-w))
    d = torch.exp(-DECAY_RATE * sig)
    S = torch.zeros(B, H, N, N, device=r.device) if state is None else state
    right = torch.stack([b, k], dim=3)  # [B, T, H, 2, N]
    before, sa = [], []
    for t in range(T):
        before.append(S)
        u = torch.matmul(S, a[:, t].unsqueeze(-1))
        sa.append(u)
        S = S * d[:, t].unsqueeze(-2) + torch.matmul(torch.cat([u, v[:, t].unsqueeze(-1)], dim=-1), right[:, t])
    final = S
    G = torch.zeros_like(S) if dstate is None else dstate
    after, gb = [None] * T, [None] * T
    for t in reversed(range(T)):
        G = G + dy[:, t].unsqueeze(-1) * r[:, t].unsqueeze(-2)
        after[t] = G
        gb[t] = torch.matmul(G, b[:, t].unsqueeze(-1))
        G = G * d[:, t].unsqueeze(-2) + gb[t] * a[:, t].unsqueeze(-2)
    states = torch.stack(before + [final], dim=1)  # [B, T + 1, H, N, N]
    after, sa, gb = torch.stack(after, dim=1), torch.stack(sa, dim=1), torch.stack(gb, dim=1)
    del before

    def rows(vec, mat):  # vec^T mat
        return torch.matmul(vec.unsqueeze(-2), mat).squeeze(-2)

    y = torch.matmul(states[:, 1:], r.unsqueeze(-1)).squeeze(-1)
    dr = rows(dy, states[:, 1:])
    dw = (after * states[:, :-1]).sum(-2) * d * (-DECAY_RATE) * sig * (1.0 - sig)
    dk = rows(v, after)
    dv = torch.matmul(after, k.unsqueeze(-1)).squeeze(-1)
    da = rows(gb.squeeze(-1), states[:, :-1])
    db = rows(sa.squeeze(-1), after)
    return y, final, [dr, dw, dk, dv, da, db] + ([G] if state is not None else [])


def _rosa(s: dict, case: dict) -> dict:
    x = [s[k] for k in ("cand", "write", "read_raw", "decay", "direction", "memory")]
    if own:
        from yufmusicgen_amd import ops

        if case["through"] == "autograd":
            read, final = ops.rosa_householder_scan(*x, gated=case["gated"])
            grads = torch.autograd.grad((read, final), [s[k] for k in _leaves(case)], (s["dread"], s["dmemory"]))
            return dict(read=read.detach(), final=final.detach(), grads=list(grads))
        grads = ops.rosa_householder_scan_backward(*x, s["dread"], dmemory=s["dmemory"], gated=case["gated"])
        return dict(grads=[g for g in grads if g is not None])
    with torch.no_grad():
        read, final, grads = _rosa_plain(x, s["dread"], s["dmemory"], case["gated"])
    if case["through"] == "autograd":
        return dict(read=read, final=final, grads=grads)
    return dict(grads=grads)


def _rosa_plain(x, dread, dmemory, gated):
    """m_t = lambda H(m_{t-1}) + sigmoid(write_t) tanh(cand_t), H(x) = x - 2 (x.u) u, read_t = H(m_t) [sigmoid(read_raw_t)], and
    the adjoint n_t = H(dq_t + lambda n_{t+1}) of m_t (dq_t: the gradient of H(m_t))."""
    cand, write, read_raw, lam, u, memory = x
    T = cand.shape[1]
    one = torch.ones((), device=cand.device)
    g, c = one / (one + torch.exp(-write)), torch.tanh(cand)
    gate = one / (one + torch.exp(-read_raw)) if gated else one
    e, dq = g * c, dread * gate

    def H(z):
        return z - 2.0 * (z * u).sum(-1, keepdim=True) * u

    m, q = [memory], [H(memory)]
    for t in range(T):
        m.append(torch.addcmul(e[:, t], lam, q[-1]))
        q.append(H(m[-1]))
    p, n = [None] * (T + 1), [None] * (T + 1)
    p[T] = dq[:, T - 1] if T else torch.zeros_like(memory)
    n[T] = H(p[T]) + dmemory
    for t in reversed(range(T)):
        p[t] = lam * n[t + 1] if t == 0 else torch.addcmul(dq[:, t - 1], lam, n[t + 1])
        n[t] = H(p[t])
    m, q, p, n = (torch.stack(z, dim=1) for z in (m, q, p, n))
    after = n[:, 1:]
    read = q[:, 1:] * gate
    grads = [after * g * (1.0 - c * c), after * c * g * (1.0 - g)]
    if gated:
        grads.append(dread * q[:, 1:] * gate * (1.0 - gate))
    long = (after.double() * q[:, :-1]).sum((0, 1)).float()  # sums over every token: in 64 bits
    pu, mu = (p.double() * u).sum(-1, keepdim=True), (m.double() * u).sum(-1, keepdim=True)
    du = (-2.0 * (pu * m + mu * p)).sum((0, 1)).float()
    return read, m[:, -1].contiguous(), grads + [long, du, n[:, 0].contiguous()]


_MASK32 = 0xFFFFFFFF


def _philox(index, counter: int, seed: int):
    """Philox 4x32 with 10 rounds (Salmon et al., SC 2011): four 32-bit words of the 128-bit counter (index, counter) under the
    64-bit key ``seed``, in int64 tensors."""
    c = [index & _MASK32, index >> 32, torch.full_like(index, counter & _MASK32), torch.full_like(index, counter >> 32 & _MASK32)]
    k0, k1 = seed & _MASK32, seed >> 32 & _MASK32
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [b >> 32 & _MASK32 ^ c[1] ^ k0, b & _MASK32, a >> 32 & _MASK32 ^ c[3] ^ k1, a & _MASK32]
        k0, k1 = k0 + 0x9E3779B9 & _MASK32, k1 + 0xBB67AE85 & _MASK32
    return c


def _kept(n: int, p: float, seed: int, counter: int, device):
    """Which of n elements dropout keeps: element i takes word i % 4 of block i / 4, and drops where it is below p 2^32."""
    words = torch.stack(_philox(torch.arange((n + 3) // 4, device=device), counter, seed), dim=-1).reshape(-1)[:n]
    return words >= int(p * 2.0**32)


def _dropout(s: dict):
    if own:
        from yufmusicgen_amd import ops

        return ops.dropout(s["x"], s["p"], s["seed"], counter=s["counter"], residual=s["residual"])
    x = s["x"]
    kept = _kept(x.numel(), s["p"], s["seed"], s["counter"], x.device).reshape(x.shape)
    out = torch.where(kept, x.float() * (1.0 / (1.0 - s["p"])), 0.0)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return out.to(x.dtype)


def _loss(s: dict, case: dict):
    logits, targets = s["logits"], s["targets"]
    if own:
        from yufmusicgen_amd import ops

        if not case["grad"]:
            return ops.cross_entropy(logits, targets, ignore_index=IGNORE, reduction=case["reduction"])
        return ops.cross_entropy_grad(logits, targets, ignore_index=IGNORE, reduction=case["reduction"])
    x = logits.float()
    valid = targets != IGNORE
    at = torch.where(valid, targets, 0).unsqueeze(-1)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    rows = torch.where(valid, (torch.log(total) - (x.gather(-1, at) - top)).squeeze(-1), 0.0)
    scale = valid.float()
    loss = rows
    if case["reduction"] == "mean":
        scale = scale / valid.sum()
        loss = (rows.double().sum() / valid.sum()).float()
    elif case["reduction"] == "sum":
        loss = rows.double().sum().float()
    if not case["grad"]:
        return loss
    grad = e / total
    grad.scatter_add_(-1, at, torch.full_like(at, -1.0, dtype=grad.dtype))
    return loss, (grad * scale.unsqueeze(-1)).to(logits.dtype)


# -------------------------------------------------------------------------------------------------------------------- work
def work(case: dict) -> dict:
    """Every input read once and every output written once; the operations of the definition."""
    if case["kind"] == "wkv":
        B, T, H, N = (case[k] for k in ("batch", "tokens", "heads", "size"))
        through = case["through"] == "autograd"
        vectors = 13 + through  # r, w, k, v, a, b, dy and six gradients (and y)
        states = (2 if case["state"] else 0) + (1 if case["state"] or through else 0) + through
        # Per token, in products of N x N: the state again (S a, its update by two rank-1 terms and the decay: 7 N^2),
        # the adjoint likewise (9 N^2), and dr, dw, dk, dv, da, db (12 N^2); y 2 N^2.
        return dict(bytes=4 * (vectors * B * T * H * N + states * B * H * N * N), flops=(28 + 2 * through) * B * T * H * N * N)
    if case["kind"] == "rosa":
        B, T, D = (case[k] for k in ("batch", "tokens", "dim"))
        vectors = (7 if case["gated"] else 5) + (case["through"] == "autograd")
        return dict(bytes=4 * (vectors * B * T * D + (3 + (case["through"] == "autograd")) * B * D + 4 * D), flops=40 * B * T * D)
    size = 2 if case["type"] == "bf16" else 4
    if case["kind"] == "dropout":
        n = case["rows"] * case["cols"]
        return dict(bytes=size * n * (3 if case["residual"] else 2), flops=2 * n)
    n = case["rows"] * case["vocab"]
    rows = case["rows"] if case["reduction"] == "none" else 1
    return dict(bytes=size * n * (2 if case["grad"] else 1) + 8 * case["rows"] + 4 * rows, flops=(6 if case["grad"] else 4) * n)


# ------------------------------------------------------------------------------------------------------------------- exact
def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    if case["kind"] == "wkv":
        return _wkv_exact(case, s)
    if case["kind"] == "rosa":
        return _rosa_exact(case, s)
    if case["kind"] == "dropout":
        x = s["x"].double()
        kept = _kept(x.numel(), s["p"], s["seed"], s["counter"], x.device).reshape(x.shape)
        out = torch.where(kept, x / (1.0 - s["p"]), 0.0)
        return out if s["residual"] is None else out + s["residual"].double()
    return _loss_exact(case, s)


def _wkv_exact(case: dict, s: dict) -> dict:
    """The definition's step in float64, differentiated by torch."""
    leaf = {k: s[k].double().requires_grad_() for k in _leaves(case)}
    B, T, H, N = leaf["r"].shape
    d = torch.exp(-DECAY_RATE * torch.sigmoid(leaf["w"]))
    per_token = [z.unbind(1) for z in (leaf["r"], d, leaf["k"], leaf["v"], leaf["a"], leaf["b"])]
    S = leaf["state"] if case["state"] else torch.zeros(B, H, N, N, dtype=torch.float64, device=DEVICE)
    ys = []
    for r, dt, k, v, a, b in zip(*per_token):
        S = S * dt[..., None, :] + torch.cat([S @ a[..., None], v[..., None]], -1) @ torch.stack([b, k], -2)
        ys.append((S @ r[..., None])[..., 0])
    y = torch.stack(ys, 1)
    aims = [(y * s["dy"].double()).sum()]
    if s["dstate"] is not None:
        aims.append((S * s["dstate"].double()).sum())
    grads = list(torch.autograd.grad(sum(aims), list(leaf.values())))
    if case["through"] == "autograd":
        return dict(y=y.detach(), final=S.detach(), grads=grads)
    return dict(grads=grads)


def _rosa_exact(case: dict, s: dict) -> dict:
    leaf = {k: s[k].double().requires_grad_() for k in _leaves(case)}
    lam, u, m = leaf["decay"], leaf["direction"], leaf["memory"]
    writes = (torch.sigmoid(leaf["write"]) * torch.tanh(leaf["cand"])).unbind(1)
    q, reads = m - 2.0 * (m @ u)[:, None] * u, []
    for e in writes:
        m = lam * q + e
        q = m - 2.0 * (m @ u)[:, None] * u
        reads.append(q)
    read = torch.stack(reads, 1)
    if case["gated"]:
        read = read * torch.sigmoid(leaf["read_raw"])
    aim = (read * s["dread"].double()).sum() + (m * s["dmemory"].double()).sum()
    grads = list(torch.autograd.grad(aim, list(leaf.values())))
    if case["through"] == "autograd":
        return dict(read=read.detach(), final=m.detach(), grads=grads)
    return dict(grads=grads)


def _loss_exact(case: dict, s: dict):
    losses, grads = [], []
    count = int((s["targets"] != IGNORE).sum())
    for x, t in zip(s["logits"].split(2048), s["targets"].split(2048)):  # float64 rows, some at a time
        logp = torch.log_softmax(x.double(), -1)
        valid = (t != IGNORE).double()
        at = t.clamp(min=0)[:, None]
        losses.append(-logp.gather(-1, at)[:, 0] * valid)
        if case["grad"]:
            g = logp.exp_().scatter_add_(-1, at, torch.full(at.shape, -1.0, dtype=torch.float64, device=x.device))
            grads.append(g.mul_(valid[:, None] / (count if case["reduction"] == "mean" else 1)))
    loss = torch.cat(losses)
    if case["reduction"] != "none":
        loss = loss.sum() / (count if case["reduction"] == "mean" else 1)
    return (loss, torch.cat(grads)) if case["grad"] else loss
