"""The embedding's and the weight update's operators without a GPU: what they refuse, before any device call."""

import pytest
import torch

from yufmusicgen_amd import ops
from yufmusicgen_amd._lib import lib

FAR = [1 << 20 << i for i in range(8)]  # never dereferenced: each call returns before any device work


def refused(status, *words):
    message = lib().yuf_last_error().decode()
    assert status == -1, (status, message)
    assert all(w in message for w in words), message


@pytest.mark.parametrize("name", ["yuf_embedding_f32", "yuf_embedding_bf16"])
def test_embedding_refusals(name):
    call = getattr(lib(), name)

    def bad(*words, M=4, V=10, D=8, table=FAR[0], tokens=FAR[1], bits=64, out=FAR[2]):
        refused(call(M, V, D, table, tokens, bits, 1.0, out, None), *words)

    bad("negative", M=-1)
    bad("negative", V=-1)
    bad("negative", D=-1)
    bad("token_bits", bits=16)
    bad("2^24", V=(1 << 24) + 1)
    bad("2^24", D=(1 << 24) + 1)
    bad("2^31", M=1 << 31)
    bad("too many", M=1 << 30, D=1 << 20)
    bad("null", table=None)
    bad("null", tokens=None)
    bad("null", out=None)
    for out in (FAR[0], FAR[1], FAR[0] + 2, FAR[1] + 8 * 4 - 2, FAR[0] - 2):
        bad("may not be", out=out)
    assert call(0, 10, 8, None, None, 64, 1.0, None, None) == 0 and call(4, 10, 0, None, None, 64, 1.0, None, None) == 0


@pytest.mark.parametrize("name", ["yuf_embedding_grad_f32", "yuf_embedding_grad_bf16"])
def test_embedding_gradient_refusals(name):
    call = getattr(lib(), name)

    def bad(*words, M=4, V=10, D=8, tokens=FAR[0], bits=64, dout=FAR[1], add=0, out=FAR[2], space=FAR[3]):
        refused(call(M, V, D, tokens, bits, dout, 1.0, -1, add, out, space, None), *words)

    bad("negative", M=-1)
    bad("negative", V=-1)
    bad("negative", D=-1)
    bad("token_bits", bits=8)
    bad("2^24", V=(1 << 24) + 1)
    bad("2^24", D=(1 << 24) + 1)
    bad("2^30", M=(1 << 30) + 1)
    bad("accumulate", add=2)
    bad("too many", M=1 << 30, D=1 << 20)
    bad("null", tokens=None)
    bad("null", dout=None)
    bad("null", out=None)
    bad("workspace", space=None)
    bad("aligned", space=FAR[3] + 64)
    size = 4 if name.endswith("f32") else 2
    for out in (FAR[0], FAR[1], FAR[3], FAR[0] + 8 * 4 - size, FAR[1] + size, FAR[3] + 256, FAR[1] - 10 * 8 * size + size):
        bad("may not be", out=out)
    for space in (FAR[0], FAR[1], FAR[2], FAR[2] - 256):
        bad("may not be", space=space)
    # Nothing to add to, nothing to add: no pointer is looked at.
    assert call(4, 0, 8, None, 64, None, 1.0, -1, 0, None, None, None) == 0
    assert call(4, 10, 0, None, 64, None, 1.0, -1, 0, None, None, None) == 0
    assert call(0, 10, 8, None, 64, None, 1.0, -1, 1, None, None, None) == 0


def test_embedding_gradient_scratch():
    space = lib().yuf_embedding_grad_workspace
    for sizes in ((-1, 10, 8), (4, -1, 8), (4, 10, -1), (4, (1 << 24) + 1, 8), (4, 10, (1 << 24) + 1), ((1 << 30) + 1, 10, 8),
                  (4, 0, 8), (4, 10, 0)):
        assert space(*sizes) == 0, sizes
    assert space(0, 10, 8) > 0
    # Positions with their tokens, a start for each token, and two rows of parts for each chunk of at least 16 positions.
    assert 16384 * 8 + 20481 * 4 < space(16384, 20480, 640) < 16384 * 8 + 20481 * 4 + 1024 * 2 * 640 * 4 + 1024


def test_python_refusals():
    tokens, weight = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4)
    with pytest.raises(ValueError, match="GPU"):
        ops.embedding(tokens, weight)
    with pytest.raises(ValueError, match="shape"):
        ops.embedding(tokens, weight[0])
    with pytest.raises(ValueError, match="GPU"):
        ops.embedding_grad(tokens, torch.zeros(3, 4), 5)
    with pytest.raises(ValueError, match="shape"):
        ops.embedding_grad(tokens, torch.zeros(4, 4), 5)


def test_embedding_refuses_what_the_kernels_do_not_take():
    """Stand-ins for GPU tensors: types, layouts, devices and padding ids."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        tokens = torch.empty(3, dtype=torch.int64, device="cuda:0")
        weight, dout = torch.empty(5, 4, device="cuda:0"), torch.empty(3, 4, device="cuda:0")
        for match, args, kind in (("same GPU", (tokens.to("cuda:1"), weight), ValueError), ("int32", (tokens.float(), weight), TypeError),
                                  ("float32", (tokens, weight.half()), TypeError), ("contiguous", (tokens, weight.t()), ValueError),
                                  ("padding_idx", (tokens, weight, 1.0, 5), ValueError), ("padding_idx", (tokens, weight, 1.0, -1), ValueError)):
            with pytest.raises(kind, match=match):
                ops.embedding(*args)
        for match, args, kw, kind in (("same GPU", (tokens.to("cuda:1"), dout, 5), {}, ValueError), ("int32", (tokens.short(), dout, 5), {}, TypeError),
                                      ("float32", (tokens, dout.half(), 5), {}, TypeError), ("negative", (tokens, dout, -1), {}, ValueError),
                                      ("padding_idx", (tokens, dout, 5), dict(padding_idx=5), ValueError),
                                      ("shape", (tokens, dout, 5), dict(out=torch.empty(6, 4, device="cuda:0")), ValueError),
                                      ("out must be", (tokens, dout, 5), dict(out=weight.bfloat16()), TypeError),
                                      ("inputs' GPU", (tokens, dout, 5), dict(out=weight.to("cuda:1")), ValueError),
                                      ("contiguous", (tokens, dout, 5), dict(out=torch.empty(4, 5, device="cuda:0").t()), ValueError),
                                      ("require", (tokens, dout, 5), dict(out=torch.empty(5, 4, device="cuda:0", requires_grad=True)), ValueError)):
            with pytest.raises(kind, match=match):
                ops.embedding_grad(*args, **kw)
