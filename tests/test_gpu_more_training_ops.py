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
                                                   (1000, 65536, 8, 1), (777, 20480, 2047, 3), (40000, 300, 40, 3)])
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
@pytest.mark.parametrize("rows", [16, 31, 32, 33, 64, 128, 4096, 40000])
def test_embedding_gradient_of_runs_at_the_chunks_ends(rows, kind):
    """Runs of one token that begin, end and pass at every place of a chunk, up to one run of everything."""
    from yufmusicgen_amd import ops

    print(f"embedding gradient runs of {rows} {kind}", flush=True)
    dout = table(6, rows, 72, TYPES[kind])
    for length in (1, 15, 16, 17, 48, 63, 64, 65, 256, 1000, rows):
        tokens = torch.arange(rows, device="cuda") // length
        tokens = tokens[torch.randperm(rows, generator=gen(7), device="cuda")]
        check_grad(ops.embedding_grad(tokens, dout, rows + 3), tokens, dout, rows + 3, 1.0)


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
