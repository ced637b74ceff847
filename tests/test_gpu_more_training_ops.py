"""GPU parity of the embedding's and the weight update's operators with float64.

Tolerances.  A lookup is one product, rounded once: the same bits as the same product of torch's.
A gradient row is an fp32 sum of n terms in some order, times the scale, plus what is there:
off by at most (n + 2) 2^-24 of the terms' magnitudes, and by half a step of the output's type.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS32 = 2.0**-24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def table(seed, vocab, cols, kind):
    return torch.randn(vocab, cols, generator=gen(seed), device="cuda").to(kind)


def ids(seed, shape, vocab, skew=1.0):
    return (torch.rand(shape, generator=gen(seed), device="cuda", dtype=torch.float64) ** skew * vocab).long()


# --------------------------------------------------------------------------- embedding
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,cols", [(1, 1, 1), (1, 5, 3), (16, 512, 128), (7, 673, 4), (70, 673, 5), (300, 20480, 640),
                                              (33, 100, 333), (5, 9, 7), (5, 9, 8), (5, 9, 9), (2000, 100, 1023), (3, 4, 5000)])
def test_embedding(rows, vocab, cols, kind):
    from yufmusicgen_amd import ops

    print(f"embedding {rows} of {vocab} x {cols} {kind}", flush=True)
    weight, tokens = table(1, vocab, cols, TYPES[kind]), ids(2, (rows,), vocab)
    for scale in (1.0, cols**0.5):
        for t in (tokens, tokens.int()):
            expect = (weight[tokens].float() * scale).to(weight.dtype)
            assert torch.equal(ops.embedding(t, weight, scale=scale), expect)


def test_embedding_of_other_shapes_and_layouts():
    from yufmusicgen_amd import ops

    weight, tokens = table(1, 50, 24, torch.float32), ids(2, (6, 4), 50)
    assert torch.equal(ops.embedding(tokens.t(), weight), weight[tokens.t()])  # strided ids
    assert ops.embedding(tokens[0, 0], weight).shape == (24,)
    assert ops.embedding(tokens[:, :0], weight).shape == (6, 0, 24)
    assert ops.embedding(tokens, weight[:, :0].contiguous()).shape == (6, 4, 0)
    held = table(3, 51, 24, torch.bfloat16).reshape(-1)
    for start in range(1, 9):  # a table at any element
        w = held[start : start + 50 * 24].view(50, 24)
        assert torch.equal(ops.embedding(tokens, w), w[tokens])
    wild = torch.tensor([0, -1, 49, 50, 1 << 40, -(1 << 40), 7], device="cuda")
    got = ops.embedding(wild, weight)
    assert torch.equal(got[[0, 2, 6]], weight[[0, 49, 7]]) and got[[1, 3, 4, 5]].isnan().all()
    assert ops.embedding(tokens, weight[:0].contiguous()).isnan().all()


def grad_reference(tokens, dout, vocab, scale, padding=None, out=None):
    """The sums in float64, and how far a float32 sum of each may be off."""
    tokens, rows = tokens.reshape(-1).long(), dout.reshape(tokens.numel(), dout.shape[-1]).double() * scale
    keep = (tokens >= 0) & (tokens < vocab)
    if padding is not None:
        keep &= tokens != padding
    tokens, rows = tokens[keep], rows[keep]
    total = torch.zeros(vocab, rows.shape[1], dtype=torch.float64, device=rows.device)
    size = total.index_put((tokens,), rows.abs(), accumulate=True)
    total = total.index_put((tokens,), rows, accumulate=True)
    if out is not None:
        total, size = total + out.double(), size + out.double().abs()
    return total, (torch.bincount(tokens, minlength=vocab)[:, None] + 2) * EPS32 * size


def check_grad(got, tokens, dout, vocab, scale, padding=None, out=None):
    expect, off = grad_reference(tokens, dout, vocab, scale, padding, out)
    off = off + torch.finfo(got.dtype).eps / 2 * (expect.abs() + off)
    assert got.shape == expect.shape and got.dtype == dout.dtype
    assert ((got.double() - expect).abs() <= off).all(), ((got.double() - expect).abs() - off).max()


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,cols,skew", [(1, 1, 1, 1), (1, 20480, 640, 1), (16, 512, 128, 1), (15, 7, 3, 1), (17, 7, 5, 1),
                                                   (300, 1, 640, 1), (2331, 673, 333, 3), (4111, 673, 1024, 8), (5000, 4, 9, 8),
                                                   (1000, 65536, 8, 1), (777, 20480, 2047, 3), (40000, 300, 40, 3),
                                                   (8192, 255, 12, 1), (8193, 255, 12, 1), (9001, 256, 12, 3), (9000, 130560, 4, 1),
                                                   (9000, 130561, 4, 1), (70000, 65536, 4, 3), (300000, 20480, 4, 8), (270000, 1, 3, 1),
                                                   (65536, 2, 3, 1), (65537, 2, 3, 1), (100000, 3, 5, 1), (90000, 256, 4, 8),
                                                   (200000, 673, 33, 8), (530000, 600, 2, 8)])
def test_embedding_gradient(rows, vocab, cols, skew, kind, add):
    from yufmusicgen_amd import ops

    print(f"embedding gradient {rows} of {vocab} x {cols} skew {skew} {kind} add {add}", flush=True)
    tokens, dout = ids(3, (rows,), vocab, skew), table(4, rows, cols, TYPES[kind])
    out = table(5, vocab, cols, TYPES[kind]) if add else None
    for t, scale in ((tokens, 1.0), (tokens.int(), cols**0.5)):
        there = None if out is None else out.clone()
        got = ops.embedding_grad(t, dout, vocab, scale=scale, out=there)
        assert there is None or got is there
        check_grad(got, tokens, dout, vocab, scale, out=out)
        again = ops.embedding_grad(t, dout, vocab, scale=scale, out=None if out is None else out.clone())
        assert torch.equal(got, again)  # one order of summation


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [16, 31, 32, 33, 64, 128, 4096, 9000, 40000])
def test_embedding_gradient_of_runs_at_the_chunks_ends(rows, kind):
    """Runs of one token that begin, end and pass at every place of a chunk, up to one run of everything."""
    from yufmusicgen_amd import ops

    print(f"embedding gradient runs of {rows} {kind}", flush=True)
    dout = table(6, rows, 72, TYPES[kind])
    for length in (1, 15, 16, 17, 48, 63, 64, 65, 256, 1000, rows):
        tokens = torch.arange(rows, device="cuda") // length
        tokens = tokens[torch.randperm(rows, generator=gen(7), device="cuda")]
        check_grad(ops.embedding_grad(tokens, dout, rows + 3), tokens, dout, rows + 3, 1.0)


@pytest.mark.parametrize("tokens,vocab", [(lambda n: n // 20000, 300), (lambda n: n // 20000 * 255, 2000), (lambda n: n % 3 * 255 + 254, 1000),
                                          (lambda n: (n % 70000 == 0) * 5, 700)], ids=["runs", "runs of a range", "last range", "one id"])
def test_embedding_gradient_of_many_positions_in_few_ranges(tokens, vocab):
    """Ranges that several workgroups share, their positions in one place and all over, some shares empty."""
    from yufmusicgen_amd import ops

    rows = 140001
    print(f"embedding gradient of {rows} positions in few ranges, {vocab} tokens", flush=True)
    tokens, dout = tokens(torch.arange(rows, device="cuda")), table(8, rows, 6, torch.float32)
    got = ops.embedding_grad(tokens, dout, vocab)
    check_grad(got, tokens, dout, vocab, 1.0)
    assert torch.equal(got, ops.embedding_grad(tokens, dout, vocab))


def test_embedding_gradient_of_paddings_and_wild_ids():
    from yufmusicgen_amd import ops

    tokens, dout = ids(8, (5, 200), 90), table(9, 1000, 40, torch.float32).view(5, 200, 40)
    tokens[:, 150:] = 3
    tokens[0, :50] = torch.tensor([-1, 90, 1 << 40, -(1 << 33), 1 << 32], device="cuda").repeat(10)
    check_grad(ops.embedding_grad(tokens, dout, 90), tokens, dout, 90, 1.0)
    got = ops.embedding_grad(tokens, dout, 90, padding_idx=3)
    check_grad(got, tokens, dout, 90, 1.0, padding=3)
    assert (got[3] == 0).all()
    old = table(10, 90, 40, torch.float32)
    got = ops.embedding_grad(tokens, dout, 90, padding_idx=3, out=old.clone())
    assert torch.equal(got[3], old[3])
    nothing = torch.full((7,), 90, device="cuda")
    assert (ops.embedding_grad(nothing, dout[0, :7], 90) == 0).all()
    assert (ops.embedding_grad(nothing[:0], dout[0, :0], 90) == 0).all()
    assert torch.equal(ops.embedding_grad(nothing[:0], dout[0, :0], 90, out=old.clone()), old)
    assert ops.embedding_grad(nothing, dout[0, :7], 0).shape == (0, 40)
    wild = dout[0].clone()
    wild[5, 2], wild[6, 3] = float("nan"), float("inf")
    got = ops.embedding_grad(torch.arange(200, device="cuda") // 3, wild, 90)
    assert got[1, 2].isnan() and got[2, 3] == float("inf") and got.isfinite().sum() == got.numel() - 2


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [1, 7, 40, 333])
def test_embedding_writes_stay_inside(cols, kind):
    """What lies around the outputs, and behind the workspace, stays as it was; they may start at any element."""
    from yufmusicgen_amd._lib import check, lib

    dtype, rows, vocab = TYPES[kind], 100, 37
    tokens, dout, weight = ids(11, (rows,), vocab, 3), table(12, rows, cols, dtype), table(13, vocab, cols, dtype)
    stream = torch.cuda.current_stream().cuda_stream
    for start in (0, 1, 3):
        held = torch.full((start + rows * cols + 50,), 7.0, device="cuda", dtype=dtype)
        call = lib().yuf_embedding_f32 if kind == "f32" else lib().yuf_embedding_bf16
        check(call(rows, vocab, cols, weight.data_ptr(), tokens.data_ptr(), 64, 1.0, held[start:].data_ptr(), stream))
        assert torch.equal(held[start : start + rows * cols].view(rows, cols), weight[tokens])
        assert (held[:start] == 7).all() and (held[start + rows * cols :] == 7).all()
        call = lib().yuf_embedding_grad_f32 if kind == "f32" else lib().yuf_embedding_grad_bf16
        size = lib().yuf_embedding_grad_workspace(rows, vocab, cols)
        space = torch.full((size + 512,), 7, device="cuda", dtype=torch.uint8)
        held = torch.full((start + vocab * cols + 50,), 7.0, device="cuda", dtype=dtype)
        check(call(rows, vocab, cols, tokens.data_ptr(), 64, dout.data_ptr(), 1.0, -1, 0, held[start:].data_ptr(),
                   space.data_ptr(), stream))
        check_grad(held[start : start + vocab * cols].view(vocab, cols), tokens, dout, vocab, 1.0)
        assert (held[:start] == 7).all() and (held[start + vocab * cols :] == 7).all() and (space[size:] == 7).all()


def test_embedding_beyond_32_bit_offsets():
    """Tables and outputs of more than 2^31 elements (bf16, 8 GB each)."""
    from yufmusicgen_amd import ops

    vocab, cols = 1 << 21, 2048
    weight = torch.zeros(vocab, cols, device="cuda", dtype=torch.bfloat16)
    tokens = torch.tensor([vocab - 1, 0, vocab // 2 + 1, vocab - 1], device="cuda")
    weight[tokens] = table(14, 3, cols, torch.bfloat16)[[0, 1, 2, 0]]
    assert torch.equal(ops.embedding(tokens, weight, scale=2.0), weight[tokens] * 2)
    grad = ops.embedding_grad(tokens, weight[tokens], vocab, out=weight.clone())
    assert torch.equal(grad[tokens[1]], weight[0] * 2) and torch.equal(grad[vocab - 1], (weight[-1].float() * 3).bfloat16())
    del grad
    many = (torch.arange(vocab, device="cuda") * 7919) % 1000
    out = ops.embedding(many, weight[-1000:])
    assert torch.equal(out[-1], weight[-1000 + many[-1]]) and torch.equal(out[vocab // 2 + 3], weight[-1000 + many[vocab // 2 + 3]])
    grad = ops.embedding_grad(many, out, 1000)
    count = torch.bincount(many, minlength=1000)[:, None]
    assert torch.allclose(grad.float(), count * weight[-1000:].float(), rtol=2.0**-8 + 2200 * EPS32, atol=0)


def test_embedding_through_autograd():
    from yufmusicgen_amd import ops

    weight = table(15, 90, 40, torch.float32).requires_grad_()
    tokens = ids(16, (3, 50), 90)
    out = ops.embedding(tokens, weight, scale=3.0, padding_idx=4)
    dout = table(17, 150, 40, torch.float32).view(3, 50, 40)
    out.backward(dout, retain_graph=True)
    check_grad(weight.grad, tokens, dout, 90, 3.0, padding=4)
    weight.grad = None
    out.sum().backward()  # an expanded gradient
    check_grad(weight.grad, tokens, torch.ones_like(dout), 90, 3.0, padding=4)
    # Against differences: the output is linear in the weight.
    step = table(18, 90, 40, torch.float32)
    step[4] = 0
    value = (ops.embedding(tokens, step, scale=3.0).double() * dout.double()).sum()
    (grad,) = torch.autograd.grad(ops.embedding(tokens, weight, scale=3.0, padding_idx=4), weight, dout)
    terms = (ops.embedding(tokens, step, scale=3.0).double() * dout.double()).abs().sum()
    assert abs((grad.double() * step.double()).sum() - value) <= 60 * EPS32 * terms
    # Once differentiable: a recorded gradient is the same and cannot be differentiated again.
    (recorded,) = torch.autograd.grad(ops.embedding(tokens, weight, scale=3.0, padding_idx=4), weight, dout.requires_grad_(),
                                      create_graph=True)
    assert recorded.requires_grad and torch.equal(recorded, grad)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        recorded.sum().backward()


def test_a_captured_backward_pass_of_the_embedding_is_refused():
    """backward() under capture raises, also beside an eager graph of the same weight; a captured forward
    pass of a weight that wants a gradient works as without."""
    from yufmusicgen_amd import ops

    weight, tokens = table(22, 90, 40, torch.float32).requires_grad_(), ids(23, (200,), 90)
    eager = ops.embedding(tokens, weight)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.embedding(tokens, weight)
    torch.cuda.current_stream().wait_stream(side)
    for take in (lambda y: y.sum().backward(), lambda y: torch.autograd.grad(y.sum(), weight)):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                take(ops.embedding(tokens, weight))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.embedding(tokens, weight)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
    torch.autograd.grad(eager.sum(), weight)


def test_embedding_in_graphs_and_on_streams():
    """Two captured graphs and eager calls between their replays; work on another stream than the tensors'."""
    from yufmusicgen_amd import ops

    weight, tokens = table(19, 400, 130, torch.float32), ids(20, (3000,), 400, 3)
    dout = table(21, 3000, 130, torch.float32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.embedding_grad(tokens, dout, 400), ops.embedding(tokens, weight)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for scale in (1.0, 2.0):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = ops.embedding(tokens, weight, scale=scale), ops.embedding_grad(tokens, dout, 400, scale=scale)
        graphs.append((graph, outs, scale))
    for k in range(4):
        tokens.copy_(ids(30 + k, (3000,), 400, 3))
        weight.mul_(-1.0)
        for graph, outs, scale in graphs if k % 2 else graphs[::-1]:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], ops.embedding(tokens, weight, scale=scale))
            assert torch.equal(outs[1], ops.embedding_grad(tokens, dout, 400, scale=scale))
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            got = ops.embedding_grad(tokens, dout, 400)
        torch.cuda.current_stream().wait_stream(side)
        check_grad(got, tokens, dout, 400, 1.0)


# ----------------------------------------------------------------------- weight update
# The polynomial amplifies what a step's rounding adds, by up to a = 3.4 each step and by how much depends on the
# matrix: the error is compared with that of the same formula in float32 products.  fp32's operands here have
# 22 bits for 24, so each rounding is at most 4 times as large: 4 times that error.  A small matrix has few
# roundings, and float32's may cancel; then the last step's remain: its terms a X, b A X and c A A X are
# together up to (3.4 + 4.8 * 1.2^2 + 2.0 * 1.2^4) = 14.6 times X, each with up to three operands off by 2^-22 of
# themselves, 44 times 2^-22 in all, of which LAST = 16 are allowed.  bf16's products, of 22 bits too, are held to the half
# step of its output, 2^-8 in the 2-norm, whose rounding alone takes up to 0.6 of that.
ABC = (3.4445, -4.7750, 2.0315)
LAST = 16 * 2.0**-22


def polynomial(x, steps=5, abc=ABC, eps=1e-7):
    """In x's type, of products as they stand."""
    a, b, c = abc
    wide = x.shape[-2] <= x.shape[-1]
    X = x if wide else x.mT.contiguous()
    X = (X.double() / (X.double().square().sum((-1, -2), keepdim=True).sqrt() + eps)).to(x.dtype)
    for _ in range(steps):
        A = X @ X.mT.contiguous()
        X = a * X + (b * A + c * (A @ A)) @ X
    return X if wide else X.mT


def gradient(seed, *shape, noise=0.1):
    few = max(1, min(shape[-2:]) // 16)
    g = gen(seed)
    left = torch.randn(*shape[:-1], few, generator=g, device="cuda") * torch.logspace(0, -2, few, device="cuda")
    return 1e-3 * (left @ torch.randn(*shape[:-2], few, shape[-1], generator=g, device="cuda") +
                   noise * torch.randn(*shape, generator=g, device="cuda"))


def norms(x):
    return x.double().square().sum((-1, -2)).sqrt()


def allowed(x, kind, **how):
    """float64's result for x and, for each matrix, how far one may be from it in the 2-norm."""
    expect = polynomial(x.double(), **how)
    if kind == "bf16":
        return expect, 2.0**-8 * norms(expect)
    return expect, 4 * norms(polynomial(x.float(), **how).double() - expect) + LAST * norms(expect)


def check_ns(got, x, kind, floor=0.0, **how):
    expect, off = allowed(x, kind, **how)
    off = off + floor
    assert got.shape == x.shape and got.dtype == x.dtype
    err = norms(got.double() - expect)
    assert (err <= off + 1e-30).all(), (err / norms(expect), off / norms(expect))


NS_SHAPES = [(1, 1, 1), (2, 1, 7), (2, 7, 1), (3, 3, 5), (3, 16, 16), (2, 31, 33), (1, 64, 64), (2, 65, 64), (1, 640, 64),
             (2, 64, 640), (1, 127, 129), (2, 256, 257), (2, 257, 256), (1, 300, 700), (3, 640, 640), (1, 1000, 129),
             (1, 129, 1000), (1, 333, 1111), (2, 1111, 333), (1, 2560, 640), (33, 20, 30), (70, 9, 5), (1, 64, 256), (1, 64, 257), (2, 64, 513),
             (1, 64, 768), (1, 64, 769), (1, 769, 33), (65, 65, 65), (12, 640, 640), (18, 640, 640), (26, 640, 640), (11, 640, 1200)]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("count,rows,cols", NS_SHAPES)
def test_newton_schulz(count, rows, cols, kind):
    from yufmusicgen_amd import ops

    print(f"newton schulz {count} x {rows} x {cols} {kind}", flush=True)
    x = gradient(count + rows, count, rows, cols).to(TYPES[kind])
    kept = x.clone()
    got = ops.newton_schulz(x)
    check_ns(got, x, kind)
    assert torch.equal(x, kept)
    check_ns(ops.newton_schulz(x.mT), x.mT, kind)  # the other orientation, and a strided input
    assert torch.equal(got, ops.newton_schulz(x))
    # A matrix alone: other tiles, and with them the order in which the low parts of A's lower half are summed.
    check_ns(ops.newton_schulz(x[-1]), x[-1], kind)
    for a, b in zip(ops.newton_schulz(list(x)), got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("steps,abc", [(1, ABC), (3, ABC), (10, ABC), (20, (1.5, -0.5, 0.0)), (12, (15 / 8, -10 / 8, 3 / 8)),
                                       (5, (0.5, 0.0, 0.0)), (2, (0.0, 1.0, -1.0)), (3, (-2.0, 1.0, 0.25))])
def test_newton_schulz_of_other_coefficients(steps, abc, kind):
    from yufmusicgen_amd import ops

    print(f"newton schulz {steps} steps of {abc} {kind}", flush=True)
    x = torch.randn(2, 96, 200, generator=gen(1), device="cuda").to(TYPES[kind])
    check_ns(ops.newton_schulz(x, steps=steps, coefficients=abc), x, kind, steps=steps, abc=abc)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_newton_schulz_of_extreme_matrices(kind):
    """Scales over the type's range, zeros, ranks of one, and non-finite matrices among finite ones."""
    from yufmusicgen_amd import ops

    x = gradient(5, 9, 70, 90).to(TYPES[kind])
    x[1] *= 1e30
    x[2] *= 1e-30  # eps leaves nothing of it
    x[3] = 0
    x[4] = x[4, :, :1] @ x[4, :1, :]
    x[5, 3, 4] = float("nan")
    x[6, 69, 89] = float("inf")
    x[7] = 0
    x[7, 69, 89] = -3.0
    got = ops.newton_schulz(x)
    assert got[5].isnan().all() and got[6].isnan().all()
    rest = [0, 1, 2, 3, 4, 7, 8]
    # X is held in steps of fp16's subnormals, 2^-24, times 2^-14: an element is off by at most 2^-39, a matrix by
    # the root of its size times that, and a step makes at most 4 times as much of it, after adding its own.
    check_ns(got[rest], x[rest], kind, floor=(70 * 90) ** 0.5 * 2.0**-39 * 4**5 * 4 / 3)
    assert (got[3] == 0).all()
    got = ops.newton_schulz(x[2], eps=0.0)  # without eps the scale does not matter
    check_ns(got, x[2], kind, eps=0.0)
    assert ops.newton_schulz(x[3], eps=0.0).isnan().all()
    assert ops.newton_schulz(x[:0]).shape == (0, 70, 90) and ops.newton_schulz(x[:, :0]).shape == (9, 0, 90)
    assert ops.newton_schulz(x.view(3, 3, 70, 90)).shape == (3, 3, 70, 90)


def muon_reference(p, g, m, lr, momentum=0.95, nesterov=True, weight_decay=0.0):
    m = momentum * m.double() + (1 - momentum) * g.double()
    u = momentum * m + (1 - momentum) * g.double() if nesterov else m
    rate = lr * max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5
    step = polynomial(u)
    loose = polynomial(u.float()).double() - step
    return p.double() * (1 - lr * weight_decay) - rate * step, m, rate * norms(step), rate * norms(loose)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("nesterov,weight_decay", [(True, 0.1), (False, 0.0)])
@pytest.mark.parametrize("count,rows,cols", [(1, 1, 1), (3, 40, 64), (2, 200, 77), (33, 12, 9), (2, 640, 640), (1, 300, 2000)])
def test_muon_step(count, rows, cols, nesterov, weight_decay, kind):
    from yufmusicgen_amd import ops

    print(f"muon step {count} x {rows} x {cols} {kind}", flush=True)
    dtype = TYPES[kind]
    p, g, m = table(1, count * rows, cols, dtype).view(count, rows, cols), gradient(2, count, rows, cols).to(dtype), gradient(3, count, rows, cols)
    new_p, new_m, step, loose = muon_reference(p, g, m, 0.3, nesterov=nesterov, weight_decay=weight_decay)
    ps, gs, ms = list(p.clone().unbind()), list(g.unbind()), [t.clone() for t in m]
    ops.muon_step(ps, gs, ms, 0.3, nesterov=nesterov, weight_decay=weight_decay)
    ps, ms = torch.stack(ps), torch.stack(ms)
    # Two products and a sum, and a rounded coefficient in each product.
    assert ((ms.double() - new_m).abs() <= 4 * EPS32 * (0.95 * m.double().abs() + 0.05 * g.double().abs())).all()
    off = (2.0**-8 if kind == "bf16" else 0) * (step + norms(new_p)) + 4 * loose + LAST * (step + norms(p))
    assert (norms(ps.double() - new_p) <= off).all(), (norms(ps.double() - new_p), off)


def test_muon_step_over_a_models_matrices():
    """Matrices of several shapes and types in one call, parameters that require gradients, an odd layout of a gradient."""
    from yufmusicgen_amd import ops

    shapes = [(40, 64), (64, 40), (40, 64), (7, 7), (64, 40)]
    params = [torch.nn.Parameter(table(i, *s, torch.bfloat16 if i == 4 else torch.float32)) for i, s in enumerate(shapes)]
    for i, p in enumerate(params):
        p.grad = gradient(10 + i, *p.shape).to(p.dtype)
    params[1].grad = params[1].grad.t().contiguous().t()
    momenta = [torch.zeros(p.shape, device="cuda") for p in params]
    expect = [muon_reference(p.detach(), p.grad, m, 0.1) for p, m in zip(params, momenta)]
    versions = [p._version for p in params]
    ops.muon_step(params, [p.grad for p in params], momenta, 0.1)
    for p, m, v, (new_p, new_m, step, loose) in zip(params, momenta, versions, expect):
        assert p._version > v and p.requires_grad and p.is_leaf
        off = (2.0**-8 if p.dtype == torch.bfloat16 else 0) * (step + norms(new_p)) + 4 * loose + LAST * (step + norms(p.detach()))
        assert norms(p.detach().double() - new_p) <= off
        assert ((m.double() - new_m).abs() <= 4 * EPS32 * new_m.abs()).all()


def test_muon_step_refuses_before_it_updates():
    """Matrices that share memory, in one shape or in two: nothing is updated."""
    from yufmusicgen_amd import ops
    from yufmusicgen_amd._lib import YufError

    p, g, m = table(50, 12, 8, torch.float32), gradient(51, 12, 8), torch.zeros(12, 8, device="cuda")
    q, h, n = table(52, 6, 8, torch.float32), gradient(53, 6, 8), torch.zeros(6, 8, device="cuda")
    before = [t.clone() for t in (p, m, q, n)]
    for params, grads, momenta in (([q, p, p], [h, g, g], [n, m, m.clone()]), ([q, p, p.view(8, 12)], [h, g, g.view(8, 12)], [n, m, m.clone().view(8, 12)]),
                                   ([q, p], [h, g], [n, p]), ([q, p], [q, g], [n, m]), ([p, p[:6]], [g, h], [m, n])):
        with pytest.raises((ValueError, YufError), match="overlap"):
            ops.muon_step(params, grads, momenta, 0.1)
    for refused in (dict(steps=0), dict(eps=-1.0), dict(coefficients=(30.0, 0.0, 0.0)), dict(lr=float("nan"))):
        with pytest.raises(YufError):
            ops.muon_step([q, p], [h, g], [n, m], **{"lr": 0.1, **refused})
    assert all(torch.equal(a, b) for a, b in zip(before, (p, m, q, n)))
    ops.muon_step([q, p], [h, g], [n, m], 0.1)
    assert not torch.equal(p, before[0]) and not torch.equal(q, before[2])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("count,rows,cols", [(2, 33, 70), (1, 300, 257)])
def test_newton_schulz_writes_stay_inside(count, rows, cols, kind):
    """What lies around the outputs and behind the workspace stays as it was; matrices may start at any element."""
    import ctypes

    from yufmusicgen_amd._lib import check, lib

    dtype, n = TYPES[kind], rows * cols
    x = gradient(6, count, rows, cols).to(dtype)
    from yufmusicgen_amd import ops

    expect = ops.newton_schulz(x)
    size = lib().yuf_newton_schulz_workspace(count, rows, cols)
    call = lib().yuf_newton_schulz_f32 if kind == "f32" else lib().yuf_newton_schulz_bf16
    for start in (0, 1, 3):
        space = torch.full((size + 4096,), 7, device="cuda", dtype=torch.uint8)
        gap = n + 5
        held, given = (torch.full((start + count * gap + 50,), 7.0, device="cuda", dtype=dtype) for _ in range(2))
        at = [start + i * gap for i in range(count)]
        for i, a in enumerate(at):
            given[a : a + n] = x[i].reshape(-1)
        lists = [(ctypes.c_void_p * count)(*[t[a:].data_ptr() for a in at]) for t in (given, held)]
        check(call(count, rows, cols, *lists, 5, *ABC, 1e-7, space.data_ptr(), torch.cuda.current_stream().cuda_stream))
        untouched = torch.ones_like(held, dtype=torch.bool)
        for i, a in enumerate(at):
            assert torch.equal(held[a : a + n], expect[i].reshape(-1))
            untouched[a : a + n] = False
        assert (held[untouched] == 7).all() and (space[size:] == 7).all()
        check(call(count, rows, cols, lists[0], lists[0], 5, *ABC, 1e-7, space.data_ptr(), torch.cuda.current_stream().cuda_stream))
        assert all(torch.equal(given[a : a + n], expect[i].reshape(-1)) for i, a in enumerate(at))  # in place


def test_weight_updates_in_graphs_and_on_streams():
    """Two captured graphs with eager calls between their replays, and a side stream."""
    from yufmusicgen_amd import ops

    x, p, m = gradient(7, 3, 70, 130), table(8, 64, 200, torch.float32), torch.zeros(64, 200, device="cuda")
    g = gradient(9, 64, 200)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.newton_schulz(x), ops.muon_step([p.clone()], [g], [m.clone()], 0.1)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for k in range(2):
        weights, momenta = p.clone(), m.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.newton_schulz(x)
            ops.muon_step([weights], [g], [momenta], 0.1 * (k + 1))
        weights.copy_(p), momenta.copy_(m)
        graphs.append((graph, out, weights, momenta, p.clone(), m.clone(), 0.1 * (k + 1)))
    for k in range(4):
        x.copy_(gradient(20 + k, 3, 70, 130)), g.copy_(gradient(30 + k, 64, 200))
        for graph, out, weights, momenta, wp, wm, lr in graphs if k % 2 else graphs[::-1]:
            graph.replay()
            torch.cuda.synchronize()
            ops.muon_step([wp], [g], [wm], lr)
            assert torch.equal(out, ops.newton_schulz(x)) and torch.equal(weights, wp) and torch.equal(momenta, wm)
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            got = ops.newton_schulz(x)
        torch.cuda.current_stream().wait_stream(side)
        check_ns(got, x, "f32")


def test_a_training_step_of_these_operators():
    """Embedding, a projection, the loss over the tied table, and the updates: the gradients are those of float64."""
    from yufmusicgen_amd import ops

    vocab, dim = 300, 64
    weight = (0.1 * table(40, vocab, dim, torch.float32)).requires_grad_()
    square = (table(41, dim, dim, torch.float32) / 8).requires_grad_()
    tokens, targets = ids(42, (4, 50), vocab, 3), ids(43, (4, 50), vocab, 3)
    targets[:, 45:] = -100
    tokens[:, 45:] = 0

    def loss_of(e, w, s, cross):
        return cross((torch.tanh(e @ s) @ w.t()).reshape(-1, vocab), targets.reshape(-1))

    loss = loss_of(ops.embedding(tokens, weight, scale=dim**0.5, padding_idx=0), weight, square, ops.cross_entropy)
    loss.backward()
    w64, s64 = (t.detach().double().requires_grad_() for t in (weight, square))
    e64 = torch.nn.functional.embedding(tokens, w64, padding_idx=0) * dim**0.5
    loss64 = loss_of(e64, w64, s64, torch.nn.functional.cross_entropy)
    loss64.backward()
    # Sums of up to vocab + 200 terms, twice.
    assert abs(loss.item() - loss64.item()) <= 1000 * EPS32 * loss64.item()
    for t, e in ((weight, w64), (square, s64)):
        assert (t.grad.double() - e.grad).norm() <= 1000 * EPS32 * e.grad.norm()
    momenta = [torch.zeros_like(square)]
    new_p, _, step, loose = muon_reference(square.detach(), square.grad, momenta[0], 0.02)
    ops.muon_step([square], [square.grad], momenta, 0.02)
    assert norms(square.detach().double() - new_p) <= 4 * loose + LAST * (step + norms(new_p))


# ------------------------------------------------------- weight updates: spectra, coefficients, launches
STEEP = (4.0848, -6.8946, 2.9270)  # slopes of up to 4 near the values that the steps settle at


def normal(seed, *shape):
    return torch.randn(*shape, generator=gen(seed), device="cuda")


def of_singular_values(seed, values, rows, cols):
    """A [rows, cols] matrix of these singular values."""
    few = min(rows, cols)
    left, right = (torch.linalg.qr(normal(seed + i, n, few).double())[0] for i, n in enumerate((rows, cols)))
    return (left * values.to(left)) @ right.mT.contiguous()


def one_row(seed, rows, cols, few=None):
    x = torch.zeros(rows, cols, device="cuda")
    x[rows // 2, :few] = normal(seed, cols if few is None else few)
    return x


SPECTRA = {
    "normal": lambda r, c: normal(60, r, c),
    "equal": lambda r, c: of_singular_values(61, torch.ones(min(r, c)), r, c),
    "near": lambda r, c: of_singular_values(63, torch.logspace(0, -0.3, min(r, c)), r, c),
    "one row": lambda r, c: one_row(65, r, c),
    "seven elements": lambda r, c: one_row(66, r, c, 7),
    "ones": lambda r, c: torch.ones(r, c, device="cuda"),
}


@pytest.mark.parametrize("steps,abc", [(5, ABC), (6, ABC), (5, STEEP)], ids=["5", "6", "steep"])
@pytest.mark.parametrize("rows,cols", [(129, 200), (160, 160), (333, 1111), (640, 2560), (1024, 1024)])
@pytest.mark.parametrize("spectrum", SPECTRA)
def test_newton_schulz_bf16_of_any_spectrum(spectrum, rows, cols, steps, abc):
    """Before its rounding a bf16 result is as near as a float32 one, whatever the matrix: the rounding's half step, 2^-8 of each
    element, is all that is seen.  (Operands of 11 bits are not enough: amplified in few directions near 1 their errors reached 1.2e-2
    with seven elements, 2^-8 = 3.9e-3, and 8.5e-2 with equal singular values and steep coefficients.)"""
    from yufmusicgen_amd import ops

    print(f"newton schulz bf16 {spectrum} {rows} x {cols}, {steps} steps of {abc}", flush=True)
    x = SPECTRA[spectrum](rows, cols).bfloat16()
    expect = polynomial(x.double(), steps, abc)
    off = 2.0**-8 * norms(expect) + 4 * norms(polynomial(x.float(), steps, abc).double() - expect) + LAST * norms(expect)
    err = norms(ops.newton_schulz(x, steps=steps, coefficients=abc).double() - expect)
    print(f"  {(err / norms(expect)).item():.2e}, allowed {(off / norms(expect)).item():.2e}", flush=True)
    assert err <= off


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("steps,abc", [(1, ABC), (3, ABC), (6, ABC), (7, ABC), (20, (1.5, -0.5, 0.0)), (5, (0.5, 0.0, 0.0)),
                                       (2, (0.0, 1.0, -1.0)), (3, (-2.0, 1.0, 0.25))])
def test_newton_schulz_of_other_coefficients_in_tiles(steps, abc, kind):
    from yufmusicgen_amd import ops

    print(f"newton schulz in tiles, {steps} steps of {abc} {kind}", flush=True)
    x = normal(67, 2, 200, 300).to(TYPES[kind])
    check_ns(ops.newton_schulz(x, steps=steps, coefficients=abc), x, kind, steps=steps, abc=abc)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_newton_schulz_of_extreme_matrices_in_tiles(kind):
    """As of small ones: scales over the type's range, zeros, a rank of one, non-finite matrices among finite ones."""
    from yufmusicgen_amd import ops

    x = gradient(68, 7, 200, 300).to(TYPES[kind])
    x[1] *= 1e30
    x[2] *= 1e-20
    x[3] = 0
    x[4] = x[4, :, :1] @ x[4, :1, :]
    x[5, 3, 4] = float("nan")
    x[6, 199, 299] = float("inf")
    got = ops.newton_schulz(x, eps=0.0)
    assert got[[3, 5, 6]].isnan().all()
    check_ns(got[[0, 1, 2, 4]], x[[0, 1, 2, 4]], kind, eps=0.0)
    assert (ops.newton_schulz(x)[3] == 0).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("count,rows,cols", [(60, 256, 256), (64, 640, 640), (49, 256, 256)])
def test_newton_schulz_of_many_matrices(count, rows, cols, kind):
    """Launches whose symmetric products take other tiles than their last product, and full groups of 64."""
    from yufmusicgen_amd import ops

    print(f"newton schulz {count} x {rows} x {cols} {kind}", flush=True)
    x = gradient(69, count, rows, cols).to(TYPES[kind])
    check_ns(ops.newton_schulz(x), x, kind)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_newton_schulz_of_more_matrices_than_a_workspace_holds(kind):
    """2 GB of operands are 8 matrices of this size: the ninth is taken alone, in the same memory."""
    from yufmusicgen_amd import ops
    from yufmusicgen_amd._lib import lib

    count, rows, cols = 9, 4000, 4090
    assert lib().yuf_newton_schulz_workspace(count, rows, cols) == lib().yuf_newton_schulz_workspace(count - 1, rows, cols)
    print(f"newton schulz {count} x {rows} x {cols} {kind}", flush=True)
    x = gradient(70, count, rows, cols).to(TYPES[kind])
    got = ops.newton_schulz(list(x))
    for i in (0, 7, 8):
        check_ns(got[i], x[i], kind)


# ------------------------------------------------- embedding gradients of large vocabularies
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,cols,skew", [(70000, 130561, 5, 3), (100001, 151936, 12, 8), (140000, 151936, 3, 1), (9000, 1 << 24, 1, 3),
                                                  (8192, 151936, 7, 3), (8193, 151936, 7, 8)])
def test_embedding_gradient_of_large_vocabularies(rows, vocab, cols, skew, kind):
    """Beyond 130560 ids, where each range's workgroup reads all positions: long batches with frequent neighbours."""
    from yufmusicgen_amd import ops

    print(f"embedding gradient {rows} of {vocab} x {cols} skew {skew} {kind}", flush=True)
    tokens, dout, out = ids(71, (rows,), vocab, skew), table(72, rows, cols, TYPES[kind]), table(73, vocab, cols, TYPES[kind])
    got = ops.embedding_grad(tokens, dout, vocab, scale=2.0, padding_idx=1)
    check_grad(got, tokens, dout, vocab, 2.0, padding=1)
    assert torch.equal(got, ops.embedding_grad(tokens.int(), dout, vocab, scale=2.0, padding_idx=1))
    check_grad(ops.embedding_grad(tokens, dout, vocab, out=out.clone()), tokens, dout, vocab, 1.0, out=out)
