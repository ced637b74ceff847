"""GPU parity of the training pass's operators with float64 on the CPU: the gradients of the
two scans, dropout and the cross-entropy.

Tolerances.  A gradient of the scans is a chain of fp32 sums over at most N + 32 terms (N
columns of a state, twice 16 tokens of a chunk), and a sum of n fp32 terms is off by at most
n 2^-24 of its terms' magnitude; the terms of different signs cancel to about their root mean
square.  So the error's 2-norm is held to (N + 32) 2^-24 of the gradient's 2-norm and a single
element's to 40 times that of the larger of itself and the root mean square -- forty, for the
largest of some 10^5 normally distributed elements' cancellations.  dropout and the
cross-entropy have short sums: their bounds stand at their tests.
"""

import numpy as np
import pytest
import torch

from oracle import rosa as orosa
from oracle import wkv7 as owkv
from yufmusicgen_amd.synth import rosa_inputs, wkv_inputs

pytestmark = pytest.mark.gpu

EPS32 = 2.0**-24


def close(got, expect, terms, what=""):
    got, expect = got.detach().double().cpu(), expect.detach().double().cpu()
    assert got.shape == expect.shape, what
    assert torch.isfinite(got).all(), what
    rms = expect.pow(2).mean().sqrt().item() if expect.numel() else 0.0
    err = got - expect
    assert err.norm() <= terms * EPS32 * expect.norm() + 1e-30, (what, (err.norm() / expect.norm()).item(), terms * EPS32)
    worst = (err.abs() / expect.abs().clamp(min=max(rms, 1e-30))).max().item() if expect.numel() else 0.0
    assert worst <= 40 * terms * EPS32, (what, worst, 40 * terms * EPS32)


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).cuda()


def leaf64(x):
    return torch.from_numpy(np.asarray(x, np.float64)).requires_grad_()


# ------------------------------------------------------------------------------- WKV-7
WKV_NAMES = ("r", "w", "k", "v", "a", "b", "state")


def wkv_case(seed, batch, steps, heads, size, state=True):
    arrs = list(wkv_inputs(seed, batch, steps, heads, size))
    rng = np.random.default_rng(seed + 1)
    s0 = rng.standard_normal((batch, heads, size, size)).astype(np.float32) if state else None
    dy = rng.standard_normal((batch, steps, heads, size)).astype(np.float32)
    ds = rng.standard_normal((batch, heads, size, size)).astype(np.float32) if state else None
    return arrs, s0, dy, ds


def wkv_exact(arrs, s0, dy, ds):
    leaves = [leaf64(x) for x in arrs]
    start = leaf64(np.zeros((arrs[0].shape[0], arrs[0].shape[2]) + (arrs[0].shape[3],) * 2) if s0 is None else s0)
    y, final = owkv.wkv7_scan(*leaves, start)
    aim = (y * torch.from_numpy(dy).double()).sum()
    if ds is not None:
        aim = aim + (final * torch.from_numpy(ds).double()).sum()
    return torch.autograd.grad(aim, leaves + [start], allow_unused=True)


def wkv_grads(arrs, s0, dy, ds):
    from yufmusicgen_amd.ops import rwkv7_scan_backward

    return rwkv7_scan_backward(*(cuda(x) for x in arrs), cuda(dy), state=None if s0 is None else cuda(s0),
                               dstate=None if ds is None else cuda(ds))


def wkv_compare(got, expect, size):
    for name, g, e in zip(WKV_NAMES, got, expect):
        close(g, torch.zeros_like(g) if e is None else e, size + 32, name)


@pytest.mark.parametrize("state", [True, False])
@pytest.mark.parametrize("steps", [1, 15, 16, 17, 50, 130])
@pytest.mark.parametrize("size", [8, 16, 32, 40, 48, 64, 128])
def test_wkv7_gradients(size, steps, state):
    print(f"wkv7 gradients N={size} T={steps} state={state}", flush=True)
    case = wkv_case(size + steps, 2, steps, 3, size, state)
    wkv_compare(wkv_grads(*case), wkv_exact(*case), size)


@pytest.mark.parametrize("batch,steps,heads,size", [(1, 1000, 1, 40), (1, 777, 2, 64), (1, 333, 1, 128), (9, 70, 16, 40),
                                                     (1, 2048, 1, 16)])
def test_wkv7_gradients_of_long_and_many_sequences(batch, steps, heads, size):
    print(f"wkv7 gradients {batch} x {steps} x {heads} x {size}", flush=True)
    case = wkv_case(7, batch, steps, heads, size)
    wkv_compare(wkv_grads(*case), wkv_exact(*case), size)


@pytest.mark.parametrize("steps", [90, 200, 333])
@pytest.mark.parametrize("size", [8, 16, 32, 40, 48, 64, 128])
def test_wkv7_gradients_of_many_heads_are_those_of_each(size, steps):
    """However many heads a call brings -- they choose how long its segments are and which kernels make
    the local pass -- a sequence's gradients are those of that sequence alone, up to both calls' rounding."""
    print(f"wkv7 gradients many heads N={size} T={steps}", flush=True)
    arrs, s0, dy, ds = wkv_case(size + steps, 10, steps, 16, size)
    many = wkv_grads(arrs, s0, dy, ds)
    last = slice(9, 10)
    alone = wkv_grads([a[last] for a in arrs], s0[last], dy[last], ds[last])
    for name, m, a in zip(WKV_NAMES, many, alone):
        close(m[last], a, 2 * (size + 32), name)


@pytest.mark.parametrize("steps,heads", [(512, 32), (512, 33), (512, 96), (512, 128), (512, 129)])
@pytest.mark.parametrize("size", [16, 40, 64, 128])
def test_wkv7_gradients_at_the_limits_of_the_split(size, steps, heads):
    """256, 768 and 1024 segments of a call and the next heads after: the last head as alone."""
    print(f"wkv7 gradients limits {steps} x {heads} x {size}", flush=True)
    arrs, s0, dy, ds = wkv_case(size + heads, 1, steps, heads, size)
    many = wkv_grads(arrs, s0, dy, ds)
    alone = wkv_grads([x[:, :, -1:] for x in arrs], s0[:, -1:], dy[:, :, -1:], ds[:, -1:])
    for name, m, x in zip(WKV_NAMES, many, alone):
        close(m[:, -1:] if name == "state" else m[:, :, -1:], x, 2 * (size + 32), name)


def test_wkv7_gradients_of_no_token():
    from yufmusicgen_amd.ops import rwkv7_scan_backward

    empty = [torch.empty(2, 0, 3, 40, device="cuda") for _ in range(7)]
    ds = torch.randn(2, 3, 40, 40, device="cuda")
    *grads, dstate = rwkv7_scan_backward(*empty, state=torch.randn_like(ds), dstate=ds)
    assert all(g.shape == (2, 0, 3, 40) for g in grads) and torch.equal(dstate, ds)
    none = [torch.empty(0, 5, 3, 40, device="cuda") for _ in range(7)]
    assert rwkv7_scan_backward(*none)[0].shape == (0, 5, 3, 40)


@pytest.mark.parametrize("size", [8, 40, 64])
@pytest.mark.parametrize("steps", [21, 200])
def test_wkv7_gradients_stay_inside_their_outputs(size, steps):
    """Ragged last chunk and padded columns: what lies behind each output, and behind the
    workspace, stays as it was; an output may start at any element."""
    from yufmusicgen_amd._lib import check, lib

    arrs, s0, dy, ds = wkv_case(size, 2, steps, 3, size)
    expect = wkv_grads(arrs, s0, dy, ds)
    held = [torch.full((e.numel() + 133,), 7.0, device="cuda") for e in expect]
    space = torch.full((lib().yuf_wkv7_scan_backward_workspace(2, steps, 3, size) + 4096,), 7, dtype=torch.uint8, device="cuda")
    inputs = [cuda(x) for x in (*arrs, s0, dy, ds)]
    check(lib().yuf_wkv7_scan_backward_f32(2, steps, 3, size, *(x.data_ptr() for x in inputs),
                                           *(h[3:].data_ptr() for h in held), space.data_ptr(),
                                           torch.cuda.current_stream().cuda_stream))
    for h, e in zip(held, expect):
        assert torch.equal(h[3 : 3 + e.numel()], e.reshape(-1)) and (h[:3] == 7).all() and (h[3 + e.numel() :] == 7).all()
    assert (space[-4096:] == 7).all()


def test_wkv7_gradients_at_extreme_decays():
    """w at both ends of the decay's range (0.545 and 1) and beyond: the gradients stay
    finite, and dw vanishes where the sigmoid is flat."""
    arrs, s0, dy, ds = wkv_case(3, 1, 64, 2, 40)
    arrs[1][:, :, 0] = 100.0  # the fastest decay in every step
    arrs[1][:, ::2, 1] = -200.0  # no decay at all: exp(200) is no float32
    case = (arrs, s0, dy, ds)
    got, expect = wkv_grads(*case), wkv_exact(*case)
    for name, g, e in zip(WKV_NAMES, got, expect):
        if name == "w":
            assert torch.isfinite(g).all() and g[:, :, 0].abs().max() < 1e-30 and g[:, ::2, 1].abs().max() < 1e-30
        else:
            close(g, e, 72, name)


def test_wkv7_gradients_match_differences():
    """Along a random direction the gradients predict the float64 forward pass's difference
    (h^2 of a central difference with h = 1e-4, and the gradients' own fp32 error)."""
    arrs, s0, dy, ds = wkv_case(11, 2, 37, 2, 40)
    grads = [g.double().cpu() for g in wkv_grads(arrs, s0, dy, ds)]
    rng = np.random.default_rng(5)

    def value(xs):
        y, final = owkv.wkv7_scan(*(torch.from_numpy(x) for x in xs[:6]), torch.from_numpy(xs[6]))
        return float((y * torch.from_numpy(dy).double()).sum() + (final * torch.from_numpy(ds).double()).sum())

    at = [np.asarray(x, np.float64) for x in [*arrs, s0]]
    for i, name in enumerate(WKV_NAMES):
        d = rng.standard_normal(at[i].shape)
        h = 1e-4
        ends = [value([x + sign * h * d if j == i else x for j, x in enumerate(at)]) for sign in (1, -1)]
        slope = float((grads[i] * torch.from_numpy(d)).sum())
        assert abs((ends[0] - ends[1]) / (2 * h) - slope) <= 1e-5 * float(grads[i].norm()) * np.sqrt(1.0), name


def test_wkv7_autograd_is_the_operator():
    """rwkv7_scan under autograd: the outputs it gives without, and the gradients of
    rwkv7_scan_backward; an output that nothing uses, a strided dy, a shared input."""
    from yufmusicgen_amd.ops import rwkv7_cuda, rwkv7_scan, rwkv7_scan_backward

    arrs, s0, dy, ds = wkv_case(13, 2, 45, 3, 40)
    plain = [cuda(x) for x in arrs]
    state, dy, ds = cuda(s0), cuda(dy), cuda(ds)
    leaves = [x.clone().requires_grad_() for x in plain]
    start = state.clone().requires_grad_()
    y, final = rwkv7_scan(*leaves, state=start)
    y0, final0 = rwkv7_scan(*plain, state=state)
    assert torch.equal(y, y0) and torch.equal(final, final0) and not y0.requires_grad
    grads = torch.autograd.grad((y, final), leaves + [start], (dy, ds))
    for g, e in zip(grads, rwkv7_scan_backward(*plain, dy, state=state, dstate=ds)):
        assert torch.equal(g, e)
    # Only the outputs (a dy that is expanded, not stored), then only the state.
    y, _ = rwkv7_cuda(*leaves)
    g = torch.autograd.grad(y.sum(), leaves[0])[0]
    assert torch.equal(g, rwkv7_scan_backward(*plain, torch.ones_like(y0))[0])
    _, final = rwkv7_scan(*leaves)
    g = torch.autograd.grad(final, leaves[3], ds)[0]
    assert torch.equal(g, rwkv7_scan_backward(*plain, torch.zeros_like(y0), dstate=ds)[3])
    # One tensor as two inputs: its gradients add up.
    x = plain[0].clone().requires_grad_()
    y, _ = rwkv7_scan(x, plain[1], x, *plain[3:])
    g = torch.autograd.grad(y, x, dy)[0]
    dr, _, dk, *_ = rwkv7_scan_backward(plain[0], plain[1], plain[0], *plain[3:], dy)
    assert torch.equal(g, dr + dk)


# -------------------------------------------------------------------------------- ROSA
ROSA_NAMES = ("cand", "write", "read_raw", "decay", "direction", "memory")


def rosa_case(seed, batch, steps, dim):
    arrs = list(rosa_inputs(seed, batch, steps, dim))
    rng = np.random.default_rng(seed + 1)
    return arrs + [rng.standard_normal((batch, dim)).astype(np.float32)], \
        rng.standard_normal((batch, steps, dim)).astype(np.float32), rng.standard_normal((batch, dim)).astype(np.float32)


def rosa_exact(arrs, dread, dmem, gated):
    leaves = [leaf64(x) for x in arrs]
    read, final = orosa.rosa_scan(*leaves, gated=gated)
    aim = (read * torch.from_numpy(dread).double()).sum()
    if dmem is not None:
        aim = aim + (final * torch.from_numpy(dmem).double()).sum()
    return torch.autograd.grad(aim, leaves, allow_unused=True)


def rosa_compare(got, expect, steps, dim):
    for name, g, e in zip(ROSA_NAMES, got, expect):
        if g is None:
            assert name == "read_raw"
            continue
        if e is None:
            assert not g.any(), name
            continue
        # Every token adds the roundings of its step; a tenth of them survives the decay
        # (lambda ~ 0.9).  decay's and direction's gradients are those values' sums.
        close(g, e, dim + 32, name)


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("dim", [1, 17, 64, 100, 128, 256, 300, 512, 1000, 1024])
@pytest.mark.parametrize("steps", [1, 7, 64, 127, 129, 200])
def test_rosa_gradients(steps, dim, gated):
    from yufmusicgen_amd.ops import rosa_householder_scan_backward

    print(f"rosa gradients T={steps} D={dim} gated={gated}", flush=True)
    arrs, dread, dmem = rosa_case(steps + dim, 2, steps, dim)
    got = rosa_householder_scan_backward(*(cuda(x) for x in arrs), cuda(dread), cuda(dmem), gated=gated)
    assert (got[2] is None) == (not gated)
    rosa_compare(got, rosa_exact(arrs, dread, dmem, gated), steps, dim)


@pytest.mark.parametrize("batch,steps,dim", [(1, 2048, 128), (5, 1000, 64), (1, 9000, 40), (3, 777, 256)])
def test_rosa_gradients_of_long_sequences(batch, steps, dim):
    from yufmusicgen_amd.ops import rosa_householder_scan_backward

    print(f"rosa gradients {batch} x {steps} x {dim}", flush=True)
    arrs, dread, _ = rosa_case(3, batch, steps, dim)
    got = rosa_householder_scan_backward(*(cuda(x) for x in arrs), cuda(dread), gated=True)
    rosa_compare(got, rosa_exact(arrs, dread, None, True), steps, dim)


def test_rosa_gradients_of_no_token():
    from yufmusicgen_amd.ops import rosa_householder_scan_backward

    empty = torch.empty(2, 0, 64, device="cuda")
    vec, dmem = torch.ones(64, device="cuda") / 8, torch.randn(2, 64, device="cuda")
    got = rosa_householder_scan_backward(empty, empty, empty, vec, vec, torch.randn_like(dmem), empty, dmem)
    assert torch.equal(got[5], dmem) and not got[3].any() and not got[4].any()
    got = rosa_householder_scan_backward(*[torch.empty(0, 5, 64, device="cuda")] * 3, vec, vec,
                                         torch.empty(0, 64, device="cuda"), torch.empty(0, 5, 64, device="cuda"))
    assert not got[3].any() and not got[4].any()


def test_rosa_gradients_match_differences():
    from yufmusicgen_amd.ops import rosa_householder_scan_backward

    arrs, dread, dmem = rosa_case(21, 2, 40, 64)
    grads = rosa_householder_scan_backward(*(cuda(x) for x in arrs), cuda(dread), cuda(dmem), gated=True)
    rng = np.random.default_rng(6)

    def value(xs):
        read, final = orosa.rosa_scan(*(torch.from_numpy(x) for x in xs))
        return float((read * torch.from_numpy(dread).double()).sum() + (final * torch.from_numpy(dmem).double()).sum())

    at = [np.asarray(x, np.float64) for x in arrs]
    for i, name in enumerate(ROSA_NAMES):
        d, h = rng.standard_normal(at[i].shape), 1e-4
        ends = [value([x + sign * h * d if j == i else x for j, x in enumerate(at)]) for sign in (1, -1)]
        g = grads[i].double().cpu()
        slope = float((g * torch.from_numpy(d)).sum())
        assert abs((ends[0] - ends[1]) / (2 * h) - slope) <= 1e-5 * float(g.norm()), name


def test_rosa_autograd_is_the_operator():
    from yufmusicgen_amd.ops import rosa_householder_scan, rosa_householder_scan_backward

    arrs, dread, dmem = rosa_case(31, 2, 150, 128)
    plain, dread, dmem = [cuda(x) for x in arrs], cuda(dread), cuda(dmem)
    for gated in (True, False):
        leaves = [x.clone().requires_grad_() for x in plain]
        read, final = rosa_householder_scan(*leaves, gated=gated)
        read0, final0 = rosa_householder_scan(*plain, gated=gated)
        assert torch.equal(read, read0) and torch.equal(final, final0)
        grads = torch.autograd.grad((read, final), leaves, (dread, dmem), allow_unused=True)
        for g, e in zip(grads, rosa_householder_scan_backward(*plain, dread, dmem, gated=gated)):
            assert g is e is None or torch.equal(g, e)
    # bf16 and strided inputs are converted by torch, whose gradients come back in their type.
    cand = plain[0].transpose(0, 1).contiguous().transpose(0, 1).bfloat16().requires_grad_()
    read, _ = rosa_householder_scan(cand, *plain[1:])
    g = torch.autograd.grad(read, cand, dread)[0]
    e = rosa_householder_scan_backward(cand.detach(), *plain[1:], dread)[0]
    assert g.dtype == torch.bfloat16 and torch.equal(g, e.bfloat16())


# ----------------------------------------------------------------------------- dropout
def philox_block(block, counter, seed):
    """Four words of Philox 4x32-10 with Python's integers."""
    c = [block & 0xFFFFFFFF, block >> 32, counter & 0xFFFFFFFF, counter >> 32]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def philox_words(n, counter, seed):
    """The first n words, block by block."""
    words = []
    for block in range((n + 3) // 4):
        words += philox_block(block, counter, seed)
    return torch.tensor(words[:n], dtype=torch.int64)


def test_philox_words_are_the_published_ones():
    """The generator's published known answers (counter and key all zero; all ones)."""
    assert [f"{w:08x}" for w in philox_words(4, 0, 0).tolist()] == ["6627e8d5", "e169c58d", "bc57ac4c", "9b00dbd8"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("n", [1, 3, 4, 7, 8, 1023, 4099, 9000])
def test_dropout(n, residual, dtype):
    """Equal to the formula with one rounding at the end: the product x / (1 - p) and the sum
    each round once in fp32 (2^-24 of their size), bf16 once more (2^-8)."""
    from yufmusicgen_amd.ops import dropout

    print(f"dropout n={n} residual={residual} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(n)
    x, res = (torch.randn(n, generator=gen).to(dtype) for _ in range(2))
    seed, counter, p = 0xFEDCBA9876543210, 0x123456789ABC, 0.3
    keep = philox_words(n, counter, seed) >= int(p * 2**32)
    got = dropout(x.cuda(), p, seed, counter=counter, residual=res.cuda() if residual else None).cpu()
    scaled = torch.where(keep, x.double() / (1 - p), 0.0)
    expect = scaled + (res.double() if residual else 0.0)
    bound = 3 * EPS32 * (scaled.abs() + expect.abs()) + (2.0**-8 * expect.abs() if dtype == torch.bfloat16 else 0.0)
    assert got.dtype == dtype and ((got.double() - expect).abs() <= bound).all()
    if not residual:
        assert (got[~keep] == 0).all()


def test_dropout_ends_of_p_and_dropped_infinities():
    from yufmusicgen_amd.ops import dropout

    x = torch.randn(1000, device="cuda")
    assert torch.equal(dropout(x, 0.0, 1), x)
    assert not dropout(x, 1.0, 1).any() and torch.equal(dropout(x, 1.0, 1, residual=x), x)
    x[::2] = float("inf")
    x[1::2] = float("nan")
    keep = philox_words(1000, 0, 1) >= 2**31
    out = dropout(x, 0.5, 1).cpu()
    assert (out[~keep] == 0).all() and not torch.isfinite(out[keep]).any()
    assert dropout(x[:0], 0.5, 1).shape == (0,)
    # Values next to bf16's largest: rounded, not wrapped; a NaN stays one.
    big = torch.tensor([3.38e38, -3.38e38, float("nan"), float("inf")], device="cuda").bfloat16()
    out = dropout(big, 0.0, 1, residual=big)
    assert out[0] == float("inf") and out[1] == -float("inf") and out[2].isnan() and out[3] == float("inf")


def test_dropout_of_unaligned_and_strided_tensors():
    """Views that start at any element, and layouts that are copied: the mask goes by the
    element's place in the tensor, and nothing beyond its ends is touched."""
    from yufmusicgen_amd._lib import check, lib
    from yufmusicgen_amd.ops import dropout

    for dtype, entry in ((torch.float32, "yuf_dropout_f32"), (torch.bfloat16, "yuf_dropout_bf16")):
        x = torch.randn(5001, device="cuda").to(dtype)
        whole = dropout(x[1:4098].clone(), 0.25, 9)
        assert torch.equal(dropout(x[1:4098], 0.25, 9), whole)
        out = torch.full((5001,), 7.0, device="cuda", dtype=dtype)
        check(getattr(lib(), entry)(4097, x[1:].data_ptr(), None, 0.25, 9, 0, None, out[3:].data_ptr(),
                                    torch.cuda.current_stream().cuda_stream))
        assert torch.equal(out[3:4100], whole) and (out[:3] == 7).all() and (out[4100:] == 7).all()
        t = torch.randn(30, 50, device="cuda").to(dtype)
        assert torch.equal(dropout(t.t(), 0.25, 9), dropout(t.t().contiguous(), 0.25, 9))


def test_dropout_rate_and_independence():
    """About p of a million elements are dropped (5 sigma), other seeds and counters share no
    mask: agreement of two masks is p^2 + (1 - p)^2 of the elements (5 sigma)."""
    from yufmusicgen_amd.ops import dropout

    n, p = 1 << 20, 0.1
    one = torch.ones(n, device="cuda")
    masks = [dropout(one, p, s, counter=c) != 0 for s, c in ((1, 0), (2, 0), (1, 1), (1 << 40, 0), (1, 1 << 40))]
    for m in masks:
        assert abs(m.double().mean().item() - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5
    agree = p * p + (1 - p) ** 2
    for i, a in enumerate(masks):
        for b in masks[:i]:
            assert abs((a == b).double().mean().item() - agree) < 5 * (agree * (1 - agree) / n) ** 0.5


def test_dropout_gradient():
    from yufmusicgen_amd.ops import dropout

    x = torch.randn(33, 65, device="cuda", requires_grad=True)
    res = torch.randn(33, 65, device="cuda", requires_grad=True)
    dout = torch.randn(33, 65, device="cuda")
    out = dropout(x, 0.4, 77, counter=5, residual=res)
    dx, dres = torch.autograd.grad(out, (x, res), dout)
    assert torch.equal(dx, dropout(dout, 0.4, 77, counter=5)) and torch.equal(dres, dout)
    # A counter on the device is read as the kernel runs, and may not change before the backward pass.
    counter = torch.tensor([5], device="cuda")
    again = dropout(x, 0.4, 77, counter=counter, residual=res)
    assert torch.equal(again, out)
    assert torch.equal(torch.autograd.grad(again, x, dout)[0], dx)
    again = dropout(x, 0.4, 77, counter=counter)
    counter += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        again.sum().backward()


# -------------------------------------------------------------------------------- loss
def loss_exact(logits, targets, ignore, reduction, dloss=1.0):
    x = logits.double().requires_grad_()
    loss = torch.nn.functional.cross_entropy(x, targets.long(), ignore_index=ignore, reduction=reduction)
    grad = torch.autograd.grad(loss, x, torch.as_tensor(dloss, dtype=torch.float64).expand_as(loss))[0]
    return loss.detach(), grad


def loss_case(rows, vocab, dtype=torch.float32, ignored=0.2, seed=0):
    gen = torch.Generator().manual_seed(seed + vocab)
    logits = (3 * torch.randn(rows, vocab, generator=gen)).to(dtype)
    targets = torch.randint(0, vocab, (rows,), generator=gen)
    targets[torch.rand(rows, generator=gen) < ignored] = -100
    targets[-1] = vocab - 1
    return logits, targets


def loss_close(got, expect, dtype, vocab):
    """The sum of V exponentials is off by log2(V) + 20 roundings (a lane sums a part, lanes
    and waves pairwise) plus the exponential's own, of at most 2 units and |x - max| 2^-24 of
    its argument (x within 40 of the maximum): 60 of 2^-24 in all; a bf16 gradient rounds once."""
    (loss, grad), (loss_e, grad_e) = got, expect
    loss, grad = loss.cpu().double(), grad.cpu()
    assert ((loss - loss_e).abs() <= 60 * EPS32 * (1 + loss_e.abs())).all()
    step = 2.0**-8 if dtype == torch.bfloat16 else 0.0
    # The target's p - 1 is off by p's own error.
    bound = (60 * EPS32 + step) * grad_e.abs() + 60 * EPS32 * grad_e.abs().amax(-1, keepdim=True) * 1e-3 + 1e-38
    at_target = grad_e < 0
    bound = torch.where(at_target, bound + 60 * EPS32 * grad_e.abs().amax(), bound)
    assert grad.dtype == dtype and ((grad.double() - grad_e).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (7, 63), (5, 257), (9, 673), (4, 1000), (5, 2049), (3, 8191),
                                        (3, 20480), (2, 20481), (2, 40000), (2, 66001), (1, 140000)])
def test_cross_entropy(rows, vocab, dtype):
    from yufmusicgen_amd.ops import cross_entropy, cross_entropy_grad

    logits, targets = loss_case(rows, vocab, dtype)
    for reduction in ("none", "mean", "sum"):
        print(f"cross entropy {rows} x {vocab} {dtype} {reduction}", flush=True)
        expect = loss_exact(logits, targets, -100, reduction)
        for t in (targets.cuda(), targets.int().cuda()):
            got = cross_entropy_grad(logits.cuda(), t, reduction=reduction)
            loss_close(got, expect, dtype, vocab)
            assert torch.equal(cross_entropy(logits.cuda(), t, reduction=reduction), got[0])
        x = logits.cuda().requires_grad_()
        g = torch.autograd.grad(cross_entropy(x, targets.cuda(), reduction=reduction).sum(), x)[0]
        assert torch.equal(g, got[1])
        same = logits.cuda()
        loss, g = cross_entropy_grad(same, targets.cuda(), reduction=reduction, inplace=True)
        assert g is same and torch.equal(g, got[1]) and torch.equal(loss, got[0])


@pytest.mark.parametrize("vocab", [673, 20480])
def test_cross_entropy_of_many_rows_counts_them_once(vocab):
    """More rows than a workgroup counts by itself; the loss is the same on every run."""
    from yufmusicgen_amd.ops import cross_entropy_grad

    logits, targets = loss_case(5003 if vocab == 673 else 4100, vocab, ignored=0.5)
    x, t = logits.cuda(), targets.cuda()
    got = cross_entropy_grad(x, t)
    loss_close(got, loss_exact(logits, targets, -100, "mean"), torch.float32, vocab)
    for _ in range(2):
        again = cross_entropy_grad(x, t)
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@pytest.mark.parametrize("vocab", [300, 20480, 140000])
def test_cross_entropy_of_masked_and_broken_rows(vocab):
    """-inf logits (a generation mask) are no candidates; a row of nothing else, a NaN, a
    +inf and a target outside the vocabulary give NaN in their row alone, and an ignored row
    is 0 whatever it holds."""
    from yufmusicgen_amd.ops import cross_entropy_grad

    logits, targets = loss_case(8, vocab, ignored=0.0)
    targets %= 8
    logits[0, 8:] = -float("inf")
    logits[1, :] = -float("inf")
    logits[2, vocab // 2] = float("nan")
    logits[3, vocab - 1] = float("inf")
    targets[4] = vocab
    targets[5] = -100
    logits[5, :] = float("nan")
    logits[6] = -1000.0 + logits[6]  # every exponential below the range but for the maximum's
    logits[7, targets[7]] = -float("inf")
    loss, grad = (z.cpu() for z in cross_entropy_grad(logits.cuda(), targets.cuda(), reduction="none"))
    for row in (1, 2, 3, 4):
        assert loss[row].isnan(), row
    assert grad[1].isnan().all() and grad[2].isnan().all() and grad[4].isnan().all()
    assert loss[5] == 0 and not grad[5].any()
    assert loss[7] == float("inf") and grad[7, targets[7]] == -1
    good = [0, 6]
    expect = loss_exact(logits[good], targets[good], -100, "none")
    loss_close((loss[good], grad[good]), expect, torch.float32, vocab)


def test_cross_entropy_of_nothing():
    from yufmusicgen_amd.ops import cross_entropy, cross_entropy_grad

    x = torch.randn(3, 50, device="cuda")
    ignored = torch.full((3,), -100, device="cuda")
    loss, grad = cross_entropy_grad(x, ignored)
    assert loss.isnan() and not grad.any()
    assert cross_entropy(x, ignored, reduction="sum") == 0
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert cross_entropy(x[:0], none).isnan() and cross_entropy(x[:0], none, reduction="none").shape == (0,)
    assert cross_entropy_grad(x[:0], none, reduction="sum")[0] == 0


def test_cross_entropy_layouts():
    """Rows a stride apart are read in place, others copied; upstream gradients; [B, T, V]."""
    from yufmusicgen_amd.ops import cross_entropy, cross_entropy_grad

    logits, targets = loss_case(24, 100)
    padded = torch.full((24, 131), float("nan"))
    padded[:, 3:103] = logits
    view, t = padded.cuda()[:, 3:103], targets.cuda()
    plain = cross_entropy_grad(logits.cuda(), t, reduction="none")
    got = cross_entropy_grad(view, t, reduction="none")
    assert all(torch.equal(a, b) for a, b in zip(got, plain))
    cross_entropy_grad(view, t, reduction="none", inplace=True)
    assert torch.equal(view, plain[1]) and view._base.isnan().sum() == 24 * 31
    three = logits.cuda().reshape(4, 6, 100)
    loss, grad = cross_entropy_grad(three, t.reshape(4, 6), reduction="none")
    assert torch.equal(loss.reshape(-1), plain[0]) and torch.equal(grad.reshape(24, 100), plain[1])
    shifted = cross_entropy(three[:, :-1], t.reshape(4, 6)[:, 1:])
    expect = cross_entropy(three[:, :-1].reshape(-1, 100), t.reshape(4, 6)[:, 1:].reshape(-1))
    assert torch.equal(shifted, expect)
    columns = logits.cuda().t().contiguous().t()
    assert torch.equal(cross_entropy(columns, t, reduction="none"), plain[0])
    scale = torch.rand(24)
    expect = loss_exact(logits, targets, -100, "none", scale)
    loss_close(cross_entropy_grad(logits.cuda(), t, reduction="none", dloss=scale.cuda()), expect, torch.float32, 100)
    expect = loss_exact(logits, targets, -100, "mean", 1024.0)
    loss_close(cross_entropy_grad(logits.cuda(), t, dloss=torch.tensor(1024.0, device="cuda")), expect, torch.float32, 100)


# ----------------------------------------------------------------------------- together
def training_step(leaves, tokens, ops, p, seed):
    """One block-like step: the WKV-7 scan, dropout into the residual, the ROSA scan, the loss."""
    r, w, k, v, a, b, cand, write, rr, decay, direction, memory, head = leaves
    B, T, H, N = r.shape
    y, _ = ops["scan"](r, w, k, v, a, b)
    x = ops["dropout"](y.reshape(B, T, H * N), p, seed, cand)
    read, _ = ops["rosa"](x, write, rr, decay, direction, memory)
    return ops["loss"](read.reshape(B * T, H * N) @ head, tokens.reshape(-1))


def test_a_training_step_together():
    """The operators as a model uses them, each the next one's input, through autograd:
    float64 on the CPU within the operators' tolerances (the longest chain of sums: 3 x (N + 32)
    of the scans, the head's product, the loss)."""
    from yufmusicgen_amd import ops

    B, T, H, N, V = 2, 70, 2, 40, 101
    arrs = list(wkv_inputs(1, B, T, H, N)) + list(rosa_inputs(2, B, T, H * N))
    rng = np.random.default_rng(3)
    arrs += [rng.standard_normal((B, H * N)), rng.standard_normal((H * N, V)) * 0.1]
    tokens = torch.from_numpy(rng.integers(0, V, (B, T)))
    tokens[0, :5] = -100
    keep = (philox_words(B * T * H * N, 4, 99) >= int(0.2 * 2**32)).reshape(B, T, H * N)
    mine = dict(scan=ops.rwkv7_scan, dropout=lambda x, p, s, res: ops.dropout(x, p, s, counter=4, residual=res),
                rosa=lambda *z: ops.rosa_householder_scan(*z, gated=True), loss=ops.cross_entropy)
    plain = dict(scan=owkv.wkv7_scan, dropout=lambda x, p, s, res: torch.where(keep, x / (1 - p), 0.0) + res,
                 rosa=orosa.rosa_scan, loss=torch.nn.functional.cross_entropy)
    leaves = [cuda(x).requires_grad_() for x in arrs]
    exact = [x.detach().double().cpu().requires_grad_() for x in leaves]
    loss = training_step(leaves, tokens.cuda(), mine, 0.2, 99)
    loss_e = training_step(exact, tokens, plain, 0.2, 99)
    assert abs(loss.item() - loss_e.item()) <= 1e-6 * abs(loss_e.item())
    for i, (g, e) in enumerate(zip(torch.autograd.grad(loss, leaves), torch.autograd.grad(loss_e, exact))):
        close(g, e, 3 * (N + 32) + H * N + 60, f"leaf {i}")


# ------------------------------------------------------------------- streams and graphs
def all_operators():
    """Every gradient operator once on fixed buffers: (inputs to refresh, call)."""
    from yufmusicgen_amd import ops

    arrs, s0, dy, ds = wkv_case(41, 2, 150, 2, 40)
    wkv = [cuda(x) for x in (*arrs, dy)]
    rarrs, dread, dmem = rosa_case(42, 2, 200, 64)
    rosa = [cuda(x) for x in (*rarrs, dread, dmem)]
    state, dstate = cuda(s0), cuda(ds)
    x, counter = torch.randn(3001, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    logits, targets = loss_case(70, 673)
    logits, targets = logits.cuda(), targets.cuda()

    def call():
        return [*ops.rwkv7_scan_backward(*wkv, state=state, dstate=dstate),
                *ops.rosa_householder_scan_backward(*rosa, gated=True), ops.dropout(x, 0.3, 8, counter=counter),
                *ops.cross_entropy_grad(logits, targets)]

    def refresh(step):
        wkv[6].mul_(1.0 + step)
        rosa[6].add_(step)
        counter.add_(1)
        logits.mul_(0.9)

    return refresh, call


def test_operators_on_a_side_stream():
    refresh, call = all_operators()
    expect = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert all(torch.equal(g, e) for g, e in zip(got, expect))


def test_two_streams_at_once_have_their_own_scratch():
    refresh, call = all_operators()
    expect = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([call() for _ in range(3)])
    torch.cuda.synchronize()
    for results in got:
        for r in results:
            assert all(torch.equal(g, e) for g, e in zip(r, expect))


def test_operators_captured_and_replayed():
    """Two graphs of the same calls, replayed in turn with new inputs and eager calls between."""
    refresh, call = all_operators()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for step in range(4):
        refresh(step)
        expect = call()
        torch.cuda.synchronize()
        graph, out = graphs[step % 2]
        graph.replay()
        torch.cuda.synchronize()
        for i, (g, e) in enumerate(zip(out, expect)):
            assert torch.equal(g, e), (step, i)


def test_a_captured_backward_pass_is_refused():
    """backward() under capture raises (and the process lives), also beside an eager graph of the
    same leaves; a captured forward pass of leaves that want gradients works as without them."""
    from yufmusicgen_amd import ops

    leaves = [cuda(x).requires_grad_() for x in wkv_inputs(3, 1, 40, 2, 16)]
    eager, _ = ops.rwkv7_scan(*leaves)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.rwkv7_scan(*leaves)
    torch.cuda.current_stream().wait_stream(side)
    for take in (lambda y: y.sum().backward(), lambda y: torch.autograd.grad(y.sum(), leaves)):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                take(ops.rwkv7_scan(*leaves)[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = ops.rwkv7_scan(*leaves)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, eager)
    torch.autograd.grad(eager.sum(), leaves)


# ------------------------------------------------------------------ a sequence in pieces
@pytest.mark.parametrize("steps,dim", [(3000, 128), (40000, 8), (1500, 300)])
def test_rosa_gradients_of_a_sequence_in_two_pieces(steps, dim):
    """The whole sequence's gradients are those of its pieces, joined by the memory and its
    gradient: other cuts into blocks and ranges, the same sums."""
    from yufmusicgen_amd.ops import rosa_householder_scan, rosa_householder_scan_backward

    arrs, dread, dmem = rosa_case(5, 1, steps, dim)
    cand, write, rr, decay, u, memory = (cuda(x) for x in arrs)
    dread, dmem, cut = cuda(dread), cuda(dmem), steps * 5 // 8 + 3
    whole = rosa_householder_scan_backward(cand, write, rr, decay, u, memory, dread, dmem, gated=True)
    head, tail = slice(None, cut), slice(cut, None)
    _, middle = rosa_householder_scan(cand[:, head], write[:, head], rr[:, head], decay, u, memory, gated=True)
    late = rosa_householder_scan_backward(cand[:, tail], write[:, tail], rr[:, tail], decay, u, middle, dread[:, tail], dmem, gated=True)
    early = rosa_householder_scan_backward(cand[:, head], write[:, head], rr[:, head], decay, u, memory, dread[:, head], late[5], gated=True)
    for i, name in enumerate(ROSA_NAMES):
        joined = torch.cat([early[i], late[i]], 1) if i < 3 else early[i].double() + late[i].double() if i < 5 else early[i]
        close(whole[i], joined, 2 * (dim + 32), name)  # the errors of both


@pytest.mark.parametrize("steps,size", [(2000, 40), (700, 64), (500, 128)])
def test_wkv7_gradients_of_a_sequence_in_two_pieces(steps, size):
    from yufmusicgen_amd.ops import rwkv7_scan, rwkv7_scan_backward

    arrs, s0, dy, ds = wkv_case(9, 1, steps, 2, size)
    x, state, dy, ds, cut = [cuda(a) for a in arrs], cuda(s0), cuda(dy), cuda(ds), steps * 5 // 8 + 3
    whole = rwkv7_scan_backward(*x, dy, state=state, dstate=ds)
    head, tail = [a[:, :cut].contiguous() for a in (*x, dy)], [a[:, cut:].contiguous() for a in (*x, dy)]
    _, middle = rwkv7_scan(*head[:6], state=state)
    late = rwkv7_scan_backward(*tail, state=middle, dstate=ds)
    early = rwkv7_scan_backward(*head, state=state, dstate=late[6])
    for i, name in enumerate(WKV_NAMES):
        close(whole[i], torch.cat([early[i], late[i]], 1) if i < 6 else early[i], 2 * (size + 32), name)


def test_cross_entropy_of_more_rows_than_a_launch_takes():
    """2^21 rows are one launch; the rows behind them get theirs too."""
    from yufmusicgen_amd.ops import cross_entropy_grad

    rows = (1 << 21) + 5
    x, t = torch.randn(rows, 3, device="cuda"), torch.randint(0, 3, (rows,), device="cuda")
    loss, grad = cross_entropy_grad(x, t, reduction="none")
    logp = torch.log_softmax(x.double(), -1)
    expect = -logp.gather(-1, t[:, None])[:, 0]
    assert (loss.double() - expect).abs().max() <= 60 * EPS32 * (1 + expect.abs().max())
    one = torch.zeros_like(logp).scatter_(-1, t[:, None], 1.0)
    assert (grad.double() - (logp.exp() - one)).abs().max() <= 60 * EPS32


def test_offsets_beyond_32_bits():
    """Over 2^31 bf16 elements (4.5 GB, all in one buffer): the last rows' loss and gradient and the
    last elements' dropout are those of the same rows alone."""
    from yufmusicgen_amd._lib import check, lib
    from yufmusicgen_amd.ops import cross_entropy_grad, dropout

    rows, vocab = 110000, 20480
    x = torch.zeros(rows, vocab, device="cuda", dtype=torch.bfloat16)
    tail = torch.randn(7, vocab, device="cuda").bfloat16()
    x[-7:] = tail
    t = torch.arange(rows, device="cuda") % vocab
    loss, grad = cross_entropy_grad(x, t, reduction="none", inplace=True)
    alone = cross_entropy_grad(tail, t[-7:], reduction="none")
    assert torch.equal(loss[-7:], alone[0]) and torch.equal(grad[-7:], alone[1])
    assert (loss[:-7] - np.log(vocab)).abs().max() <= 60 * EPS32 * 10
    x.fill_(1.0)
    n, check_from = x.numel(), x.numel() - 4096
    check(lib().yuf_dropout_bf16(n, x.data_ptr(), None, 0.5, 3, 0, None, x.data_ptr(), torch.cuda.current_stream().cuda_stream))
    words = []
    for block in range(check_from // 4, n // 4):  # the mask goes by the element's 64-bit place
        words += philox_block(block, 0, 3)
    assert torch.equal(x.reshape(-1)[check_from:].cpu() != 0, torch.tensor(words) >= 2**31)
    assert dropout(x[:1, :8], 0.5, 3).shape == (1, 8)


def test_rosa_autograd_takes_the_scans_layouts():
    """decay, direction and memory in other shapes of the same elements, as the forward call takes them."""
    from yufmusicgen_amd.ops import rosa_householder_scan

    arrs, dread, _ = rosa_case(3, 1, 70, 64)
    x = [cuda(a) for a in arrs]
    odd = [x[0], x[1], x[2], x[3].reshape(1, 64), x[4].reshape(64, 1), x[5].reshape(64)]
    leaves = [z.clone().requires_grad_() for z in odd]
    plain = [z.clone().requires_grad_() for z in x]
    got = torch.autograd.grad(rosa_householder_scan(*leaves, gated=True)[0], leaves, cuda(dread))
    expect = torch.autograd.grad(rosa_householder_scan(*plain, gated=True)[0], plain, cuda(dread))
    for g, e, z in zip(got, expect, leaves):
        assert g.shape == z.shape and torch.equal(g.reshape(-1), e.reshape(-1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cross_entropy_backward_over_no_rows(reduction, dtype):
    """As torch's loss: an empty gradient, also through [0, T, V] logits and a head's product."""
    from yufmusicgen_amd.ops import cross_entropy

    for shape in ((0, 50), (0, 7, 50), (3, 0, 50)):
        x = torch.empty(*shape, device="cuda", dtype=dtype, requires_grad=True)
        loss = cross_entropy(x, torch.empty(*shape[:-1], dtype=torch.int64, device="cuda"), reduction=reduction)
        loss.sum().backward()
        assert x.grad.shape == x.shape and x.grad.dtype == dtype
    h = torch.empty(0, 8, device="cuda")
    head = torch.randn(8, 50, device="cuda", requires_grad=True)
    cross_entropy(h @ head, torch.empty(0, dtype=torch.int64, device="cuda"), reduction=reduction).sum().backward()
    assert head.grad.shape == (8, 50) and not head.grad.any()


# ---------------------------------------------------------- the decays' gradient, token by token
def wkv_decay_gradient(arrs, s0, dy, ds):
    """float64: dw and, per element, the sum of its terms' magnitudes, sum_i |G_ij S_ij| d_j |slope_j|."""
    r, w, k, v, a, b, dy = (torch.from_numpy(np.asarray(x, np.float64)) for x in (*arrs, dy))
    batch, steps, heads, size = r.shape
    sig = torch.sigmoid(w)
    d, slope = torch.exp(-np.exp(-0.5) * sig), -np.exp(-0.5) * sig * torch.sigmoid(-w)
    zero = torch.zeros(batch, heads, size, size, dtype=torch.float64)
    S = zero if s0 is None else torch.from_numpy(np.asarray(s0, np.float64))
    G = zero if ds is None else torch.from_numpy(np.asarray(ds, np.float64))
    states = []
    for t in range(steps):
        states.append(S)
        u = S @ a[:, t, :, :, None]
        S = S * d[:, t, :, None, :] + u @ b[:, t, :, None, :] + v[:, t, :, :, None] @ k[:, t, :, None, :]
    dw, size_of = torch.empty_like(w), torch.empty_like(w)
    for t in reversed(range(steps)):
        G = G + dy[:, t, :, :, None] @ r[:, t, :, None, :]
        terms = G * states[t] * (d[:, t] * slope[:, t])[:, :, None, :]
        dw[:, t], size_of[:, t] = terms.sum(-2), terms.abs().sum(-2)
        G = G * d[:, t, :, None, :] + (G @ b[:, t, :, :, None]) @ a[:, t, :, None, :]
    return dw, size_of


def decay_gradient_close(got, arrs, s0, dy, ds, floor=0.0):
    """Every token's dw by itself: its error's 2-norm over the columns is at most N + 32 roundings (the terms
    of the sums that make a state, its gradient and their product) of its own terms' magnitudes -- not of other
    tokens' -- and so exactly 0 where no term is left.  floor: an absolute error that a test derives."""
    dw, size_of = wkv_decay_gradient(arrs, s0, dy, ds)
    err = (got.double().cpu() - dw).norm(dim=-1)
    terms, size_of = dw.shape[-1] + 32, size_of.norm(dim=-1)
    bound = terms * EPS32 * size_of + torch.where(size_of > 0, terms * 2.0**-114 + floor, 0.0)
    worst = ((err - bound) / bound.clamp(min=1e-30)).argmax().item()
    assert (err <= bound).all(), (worst, err.reshape(-1)[worst].item(), bound.reshape(-1)[worst].item())


def decay_inputs(kind, seed, batch, steps, heads, size):
    """Inputs whose tokens' decay gradients differ by orders of magnitude."""
    arrs, s0, dy, ds = wkv_case(seed, batch, steps, heads, size)
    half = np.arange(steps) % 16 < 8
    if kind.startswith("fast"):  # a state that dies out within a chunk, but for the chunk's last token
        arrs[1][:] = 30.0
        arrs[1][:, 15::16] = -1.0
        arrs[2] *= float(kind[4:])  # writes
    elif kind == "padded":  # right padding: nothing follows the last token that counts
        dy[:, steps - steps // 3 :] = 0.0
        s0 *= 30.0
        ds = None
    elif kind == "left":  # nothing before the first token that counts
        s0 = None
        arrs[2][:, : steps // 3] = 0.0
    elif kind == "early":
        arrs[3][:, half] *= 100.0
        dy[:, half] *= 100.0
        arrs[1][:, ~half] = 30.0
    elif kind == "late":
        arrs[3][:, ~half] *= 100.0
        dy[:, ~half] *= 100.0
    elif kind == "state":
        s0 *= 30.0
    return arrs, s0, dy, ds


@pytest.mark.parametrize("kind", ["fast0.01", "fast0.001", "fast0", "padded", "left", "early", "late", "state", "plain"])
@pytest.mark.parametrize("size", [8, 40, 64, 128])
@pytest.mark.parametrize("steps", [16, 27, 50, 333])
def test_wkv7_decay_gradient_of_every_token(steps, size, kind):
    print(f"wkv7 decay gradient {kind} N={size} T={steps}", flush=True)
    case = decay_inputs(kind, size + steps, 1, steps, 2, size)
    got = wkv_grads(*case)
    decay_gradient_close(got[1], *case)
    expect = wkv_exact(*case)
    close(got[1], expect[1], size + 32, "w")
    if kind == "padded":
        assert not got[1][:, steps - steps // 3 :].any()


def test_wkv7_decay_gradient_of_a_zero_states_first_token():
    arrs, _, dy, ds = wkv_case(4, 2, 40, 3, 40)
    assert not wkv_grads(arrs, None, dy, ds)[1][:, 0].any()


def test_wkv7_decay_gradient_at_extreme_decays():
    """The values, where the sigmoid is flat too: exp(-80) is the smallest exponential the kernel takes, 1.8e-35,
    and a gradient below it is the state's and its gradient's product (some 10^3 here) with that."""
    arrs, s0, dy, ds = wkv_case(3, 1, 64, 2, 40)
    arrs[1][:, :, 0] = 100.0
    arrs[1][:, ::2, 1] = -200.0
    decay_gradient_close(wkv_grads(arrs, s0, dy, ds)[1], arrs, s0, dy, ds, floor=1e-30)


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("dim", [64, 100, 300])
def test_rosa_gradients_through_open_gates_and_small_candidates(dim, gated):
    """Every element by itself.  One token, no memory and the first unit vector as direction: H only changes the first
    element's sign, so each gradient is a product of its own element's factors.  exp of x is off by |x| + 2 roundings
    (its argument's and its own), a sigmoid, 1 - sigmoid, tanh and 1 - tanh^2 by their exponential's (|x|, 2 |x| for
    tanh) and at most 8 more (tanh beyond 1/4 divides E - 1 by E + 1, of which the first magnifies E's 2 by up to 3);
    six factors and their products are within 64 beside the exponentials'.  Below float32's smallest normal number
    2^-126 a factor is off by that, times factors below 2^4."""
    from yufmusicgen_amd.ops import rosa_householder_scan_backward

    batch, rng = 40, np.random.default_rng(dim)

    def spread(most):
        """Either sign, from 1e-6 to `most` evenly in the logarithm."""
        x = np.exp(rng.uniform(np.log(1e-6), np.log(most), (batch, 1, dim))) * rng.choice([-1.0, 1.0], (batch, 1, dim))
        return x.astype(np.float32)

    cand, write, rr, dread = spread(30.0), spread(40.0), spread(40.0), rng.uniform(0.5, 2.0, (batch, 1, dim)).astype(np.float32)
    u, lam = np.zeros(dim, np.float32), np.full(dim, 0.5, np.float32)
    u[0] = 1.0
    got = rosa_householder_scan_backward(*(cuda(x) for x in (cand, write, rr, lam, u, np.zeros((batch, dim)), dread)),
                                         gated=gated)
    c, w, r, n = (torch.from_numpy(x).double() for x in (cand, write, rr, dread))
    sign = 1.0 - 2.0 * torch.from_numpy(u).double()
    g, th, slope = torch.sigmoid(w), torch.tanh(c), 1.0 / torch.cosh(c) ** 2
    dq = n * torch.sigmoid(r) if gated else n
    expect = [sign * dq * g * slope, sign * dq * th * g * torch.sigmoid(-w)]
    if gated:
        expect.append(n * sign * g * th * torch.sigmoid(r) * torch.sigmoid(-r))
    roundings = 64 + 2 * w.abs() + 2 * c.abs() + (2 * r.abs() if gated else 0)
    for name, x, e in zip(("cand", "write", "read_raw"), got, expect):
        err, bound = (x.double().cpu() - e).abs(), roundings * EPS32 * e.abs() + 2.0**-122
        at = (err / bound).argmax()
        assert (err <= bound).all(), (name, *(z.reshape(-1)[at].item() for z in (c, w, r, x.double().cpu(), e)))


def test_rosa_gradients_of_saturated_inputs_are_finite():
    """Infinities and the largest numbers as gates and candidates: no 0 times infinity."""
    from yufmusicgen_amd.ops import rosa_householder_scan_backward

    ends = torch.tensor([float("inf"), -float("inf"), 3e38, -3e38, 100.0, -100.0, 88.8, -88.8], device="cuda")
    cand = ends.repeat(8)[None, None]
    write, rr = ends.repeat_interleave(8)[None, None], ends.roll(3).repeat(8)[None, None]
    vec, one = torch.full((64,), 0.125, device="cuda"), torch.ones(1, 1, 64, device="cuda")
    for gated in (True, False):
        for g in rosa_householder_scan_backward(cand, write, rr, vec, vec, torch.zeros(1, 64, device="cuda"), one, gated=gated):
            assert g is None or torch.isfinite(g).all()


@pytest.mark.parametrize("side", [1, -1])
def test_gradients_beside_their_logits(side):
    """Logits and gradient in the two halves of one buffer's rows: of one stride, each between the other's."""
    from yufmusicgen_amd._lib import check, lib
    from yufmusicgen_amd.ops import cross_entropy_grad

    logits, targets = loss_case(9, 67)
    both = torch.full((9, 134), 7.0, device="cuda")
    x, g = (both[:, :67], both[:, 67:]) if side > 0 else (both[:, 67:], both[:, :67])
    x.copy_(logits)
    loss, t = torch.empty(9, device="cuda"), targets.cuda()
    check(lib().yuf_cross_entropy_f32(9, 67, x.data_ptr(), 134, t.data_ptr(), 64, -100, 0, loss.data_ptr(), None, g.data_ptr(), 134,
                                      None, torch.cuda.current_stream().cuda_stream))
    expect = cross_entropy_grad(logits.cuda(), t, reduction="none")
    assert torch.equal(loss, expect[0]) and torch.equal(g, expect[1]) and torch.equal(x.cpu(), logits)


@pytest.mark.parametrize("rows", [(1 << 31) - 1, (1 << 31) - 8193])
def test_cross_entropy_of_the_most_rows(rows):
    """Up to 2^31 - 1 rows (26 GB with their scratch): where the rows are counted and summed, steps end beyond the
    last one.  All but the first three and the last five are ignored, and each of those is one of two equal logits."""
    from yufmusicgen_amd.ops import cross_entropy_grad

    x = torch.zeros(rows, 2, device="cuda", dtype=torch.bfloat16)
    t = torch.full((rows,), -100, device="cuda", dtype=torch.int32)
    t[:3], t[-5:] = 0, 1
    for reduction, scale in (("mean", 8), ("sum", 1)):
        loss, grad = cross_entropy_grad(x, t, reduction=reduction, inplace=True)
        assert abs(loss.item() - np.log(2) * 8 / scale) <= 60 * EPS32 * 8 / scale
        assert (grad[:3] == torch.tensor([-0.5, 0.5], device="cuda") / scale).all()
        assert (grad[-5:] == torch.tensor([0.5, -0.5], device="cuda") / scale).all()
        assert not grad[3:4096].any() and not grad[-(1 << 20) : -5].any()
        x.zero_()


def test_philox_words_of_published_counters_and_keys():
    """The generator's other two published known answers: every bit of counter and key set, and words that all
    differ (digits of pi), which pin the order of the counter's and the key's words."""
    for (block, counter, seed), words in (
        ((2**64 - 1, 2**64 - 1, 2**64 - 1), "408f276d 41c83b0e a20bc7c6 6d5451fd"),
        ((0x85A308D3243F6A88, 0x0370734413198A2E, 0x299F31D0A4093822), "d16cfe09 94fdcceb 5001e420 24126ea1"),
    ):
        assert " ".join(f"{w:08x}" for w in philox_block(block, counter, seed)) == words


def test_autograd_over_no_tokens_and_no_sequences():
    """The scans, dropout and their backward passes over empty tensors: the carried state's gradient passes through."""
    from yufmusicgen_amd import ops

    for batch, steps in ((2, 0), (0, 5)):
        x = [torch.empty(batch, steps, 3, 40, device="cuda", requires_grad=True) for _ in range(6)]
        state = torch.randn(batch, 3, 40, 40, device="cuda", requires_grad=True)
        y, final = ops.rwkv7_scan(*x, state=state)
        dfinal = torch.randn_like(final)
        grads = torch.autograd.grad((y, final), [*x, state], (torch.ones_like(y), dfinal))
        assert torch.equal(final, state) and torch.equal(grads[6], dfinal) and all(g.shape == z.shape for g, z in zip(grads, x))
        seq = [torch.empty(batch, steps, 64, device="cuda", requires_grad=True) for _ in range(3)]
        vec = [torch.full((64,), 0.125, device="cuda", requires_grad=True) for _ in range(2)]
        memory = torch.randn(batch, 64, device="cuda", requires_grad=True)
        read, last = ops.rosa_householder_scan(*seq, *vec, memory, gated=True)
        dlast = torch.randn_like(last)
        grads = torch.autograd.grad((read, last), [*seq, *vec, memory], (torch.ones_like(read), dlast))
        assert torch.equal(last, memory) and torch.equal(grads[5], dlast) and not grads[3].any() and not grads[4].any()
    h = torch.empty(0, 7, device="cuda", requires_grad=True)
    ops.dropout(h, 0.5, 1, residual=h).sum().backward()
    assert h.grad.shape == (0, 7)


@pytest.mark.parametrize("batch,steps,heads,size", [(700, 3, 8, 32), (40, 17, 33, 128), (1, 9, 2000, 8)])
def test_wkv7_gradients_of_more_heads_than_segments(batch, steps, heads, size):
    """More than 1024 heads, one segment each: the last ones' gradients are those of the last ones alone."""
    print(f"wkv7 gradients {batch} x {steps} x {heads} x {size}", flush=True)
    arrs, s0, dy, ds = wkv_case(size, batch, steps, heads, size)
    many = wkv_grads(arrs, s0, dy, ds)
    alone = wkv_grads([x[-1:, :, -2:] for x in arrs], s0[-1:, -2:], dy[-1:, :, -2:], ds[-1:, -2:])
    for name, m, x in zip(WKV_NAMES, many, alone):
        close(m[-1:, -2:] if name == "state" else m[-1:, :, -2:], x, 2 * (size + 32), name)


@pytest.mark.parametrize("dim", [64, 300, 700])
def test_rosa_gradients_of_many_sequences(dim):
    from yufmusicgen_amd.ops import rosa_householder_scan_backward

    batch, steps = 1500, 40
    arrs, dread, dmem = rosa_case(dim, batch, steps, dim)
    cand, write, rr, decay, u, memory = (cuda(x) for x in arrs)
    many = rosa_householder_scan_backward(cand, write, rr, decay, u, memory, cuda(dread), cuda(dmem), gated=True)
    cut = slice(batch - 3, None)
    alone = rosa_householder_scan_backward(cand[cut], write[cut], rr[cut], decay, u, memory[cut], cuda(dread)[cut],
                                           cuda(dmem)[cut], gated=True)
    for i in (0, 1, 2, 5):
        assert torch.equal(many[i][cut], alone[i]), ROSA_NAMES[i]


def test_gradient_over_logits_in_inference_mode():
    from yufmusicgen_amd.ops import cross_entropy_grad

    logits, targets = loss_case(6, 100)
    expect = cross_entropy_grad(logits.cuda(), targets.cuda())
    with torch.inference_mode():
        x = logits.cuda()
        loss, grad = cross_entropy_grad(x, targets.cuda(), inplace=True)
        assert grad is x and torch.equal(grad, expect[1]) and torch.equal(loss, expect[0])


@pytest.mark.parametrize("rows,vocab", [(8192, 33), (8193, 33), (2048, 1100), (2049, 1100), (1024, 5000), (1025, 5000),
                                        (512, 10300), (513, 10300)])
def test_cross_entropy_where_rows_are_counted_apart(rows, vocab):
    """As many rows as the workgroups count by themselves, and one more, for each number of a row's waves."""
    from yufmusicgen_amd.ops import cross_entropy, cross_entropy_grad

    print(f"cross entropy count {rows} x {vocab}", flush=True)
    logits, targets = loss_case(rows, vocab, ignored=0.4)
    got = cross_entropy_grad(logits.cuda(), targets.cuda())
    loss_close(got, loss_exact(logits, targets, -100, "mean"), torch.float32, vocab)
    x = logits.cuda().requires_grad_()
    loss = cross_entropy(x, targets.cuda())
    assert torch.equal(loss, got[0]) and torch.equal(torch.autograd.grad(loss, x)[0], got[1])


@pytest.mark.parametrize("blocks", [128, 129, 768, 769, 4096, 4097, 12288, 12289])
def test_rosa_gradients_at_the_limits_of_the_ranges(blocks):
    """The longest sequences of each range length and the next ones, by pieces of other cuts joined by the memory and
    its gradient (decay's and direction's sums over all tokens in fp64)."""
    from yufmusicgen_amd.ops import rosa_householder_scan, rosa_householder_scan_backward

    steps, dim = 32 * blocks - 5, 24
    print(f"rosa gradients of {blocks} blocks", flush=True)
    arrs, dread, dmem = rosa_case(7, 1, steps, dim)
    *seq, decay, u, memory = (cuda(x) for x in arrs)
    dread, dmem = cuda(dread), cuda(dmem)
    whole = rosa_householder_scan_backward(*seq, decay, u, memory, dread, dmem, gated=True)
    cuts = [0, steps // 3 + 1, steps * 3 // 4, steps]
    pieces = [slice(a, b) for a, b in zip(cuts, cuts[1:])]
    starts = [memory]
    for piece in pieces[:-1]:
        starts.append(rosa_householder_scan(*(x[:, piece] for x in seq), decay, u, starts[-1], gated=True)[1])
    parts, end = [], dmem
    for piece, start in zip(pieces[::-1], starts[::-1]):
        parts.append(rosa_householder_scan_backward(*(x[:, piece] for x in seq), decay, u, start, dread[:, piece], end, gated=True))
        end = parts[-1][5]
    parts = parts[::-1]
    for i, name in enumerate(ROSA_NAMES):
        joined = torch.cat([p[i] for p in parts], 1) if i < 3 else sum(p[i].double() for p in parts) if i < 5 else end
        close(whole[i], joined, 2 * (dim + 32), name)  # the errors of both
