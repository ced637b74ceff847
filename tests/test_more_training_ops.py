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
    # Positions with their tokens, a start for each token, two rows of parts (whole vectors of 64 lanes) for each chunk
    # of at least 8 positions; for many positions also nine bytes for each, 1 KB for each block of at least 1024, and
    # starts for up to 254 ids that do not occur.
    most = 16384 * 8 + 20735 * 4 + 2048 * 2 * 1024 * 4 + 16384 * 9 + 16 * 1024
    assert 16384 * 17 + 20481 * 4 < space(16384, 20480, 640) < most + 2048


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


# ------------------------------------------------------------------- weight update
import ctypes  # noqa: E402


def pointers(*at):
    return (ctypes.c_void_p * len(at))(*at)


GOOD = (5, 3.4445, -4.7750, 2.0315, 1e-7)


@pytest.mark.parametrize("name", ["yuf_newton_schulz_f32", "yuf_newton_schulz_bf16"])
def test_newton_schulz_refusals(name):
    call = getattr(lib(), name)
    size = 64 * 40 * (4 if name.endswith("f32") else 2)
    space = lib().yuf_newton_schulz_workspace(2, 64, 40)
    assert space > 0 and space % 8 == 0

    def bad(*words, count=2, rows=64, cols=40, x=pointers(FAR[0], FAR[1]), out=pointers(FAR[2], FAR[3]), how=GOOD, at=FAR[7]):
        refused(call(count, rows, cols, x, out, *how, at, None), *words)

    bad("negative", count=-1)
    bad("negative", rows=-1)
    bad("negative", cols=-1)
    bad("2^28", rows=1 << 14, cols=(1 << 14) + 1)
    bad("2^22", rows=1, cols=(1 << 22) + 1)
    for steps in (0, -1, 65):
        bad("steps", how=(steps, *GOOD[1:]))
    for eps in (-1.0, float("nan"), float("inf")):
        bad("eps", how=(*GOOD[:4], eps))
    for abc in ((30.0, 0.0, 0.0), (3.4445, -4.7750, 4.0), (float("nan"), 0.0, 0.0), (float("inf"), 0.0, 0.0), (0.0, 1e300, 1e300)):
        bad("grow", how=(5, *abc, 1e-7))
    bad("null", x=None)
    bad("null", out=None)
    bad("null", x=pointers(FAR[0], None))
    bad("null", out=pointers(None, FAR[3]))
    bad("workspace", at=None)
    bad("aligned", at=FAR[7] + 128)
    for out in ((FAR[1], FAR[0]), (FAR[0] + 4, FAR[3]), (FAR[2], FAR[2]), (FAR[2], FAR[2] + size - 4), (FAR[7], FAR[3]),
                (FAR[7] + space - 4, FAR[3]), (FAR[2], FAR[1] - size + 4)):
        bad("overlap", out=pointers(*out))
    bad("overlap", at=FAR[1])
    for sizes in ((0, 64, 40), (2, 0, 40), (2, 64, 0)):
        assert call(*sizes, None, None, *GOOD, None, None) == 0


def test_newton_schulz_scratch():
    space = lib().yuf_newton_schulz_workspace
    for sizes in ((-1, 4, 4), (0, 4, 4), (1, 0, 4), (1, 4, 0), (1, 1 << 14, (1 << 14) + 1), (1, (1 << 22) + 1, 1)):
        assert space(*sizes) == 0, sizes
    assert space(1, 1, 1 << 20) > 0 and space(1, 1 << 14, 1 << 14) > 0
    assert space(1000, 640, 640) == space(100, 640, 640)  # a group's, however many there are


@pytest.mark.parametrize("name", ["yuf_muon_step_f32", "yuf_muon_step_bf16"])
def test_muon_step_refusals(name):
    call = getattr(lib(), name)
    size = 64 * 40 * (4 if name.endswith("f32") else 2)

    def bad(*words, p=(FAR[0], FAR[1]), g=(FAR[2], FAR[3]), m=(FAR[4], FAR[5]), lr=0.02, beta=0.95, nesterov=1, decay=0.0, how=GOOD, at=FAR[7]):
        lists = [None if x is None else pointers(*x) for x in (p, g, m)]
        refused(call(2, 64, 40, *lists, lr, beta, nesterov, decay, *how, at, None), *words)

    for x in (float("nan"), float("inf")):
        bad("finite", lr=x)
        bad("finite", beta=x)
        bad("finite", decay=x)
    bad("nesterov", nesterov=2)
    bad("steps", how=(0, *GOOD[1:]))
    for which in "pgm":
        bad("null", **{which: None})
        bad("null", **{which: (FAR[6], None)})
    bad("workspace", at=None)
    bad("overlap", p=(FAR[0], FAR[0]))  # the same matrix twice
    bad("overlap", m=(FAR[4], FAR[4] + 64 * 40 * 4 - 4))
    bad("overlap", g=(FAR[0], FAR[3]))  # a gradient in its weight's place
    bad("overlap", g=(FAR[4] + 64 * 40 * 4 - 4, FAR[3]))
    bad("overlap", m=(FAR[1] + size - 4, FAR[5]))
    assert call(0, 64, 40, None, None, None, 0.02, 0.95, 1, 0.0, *GOOD, None, None) == 0


def test_weight_update_python_refusals():
    from torch._subclasses.fake_tensor import FakeTensorMode

    x = torch.zeros(4, 4)
    with pytest.raises(ValueError, match="GPU"):
        ops.newton_schulz(x)
    with pytest.raises(ValueError, match="shape"):
        ops.newton_schulz(x[0])
    with pytest.raises(ValueError, match="shape"):
        ops.newton_schulz([x[None], x[None]])
    with pytest.raises(ValueError, match="one shape"):
        ops.newton_schulz([x, x[:2]])
    with pytest.raises(ValueError, match="GPU"):
        ops.muon_step([x], [x], [x], 0.1)
    with pytest.raises(ValueError, match="as many"):
        ops.muon_step([x], [x, x], [x], 0.1)
    assert ops.newton_schulz([]) == [] and ops.muon_step([], [], [], 0.1) is None
    with FakeTensorMode():
        g = torch.empty(4, 6, device="cuda:0")
        for kind, match, arg in ((TypeError, "float32", g.half()), (ValueError, "same GPU", [g, g.to("cuda:1")]), (TypeError, "x must be", [g, g.bfloat16()]),
                                 (ValueError, "differentiable", torch.empty(4, 6, device="cuda:0", requires_grad=True))):
            with pytest.raises(kind, match=match):
                ops.newton_schulz(arg)
        for kind, match, args in ((ValueError, "matrices", (g[0], g[0], g[0])), (TypeError, "float32", (g.half(), g, g)),
                                  (TypeError, "grads", (g, g.bfloat16(), g)), (TypeError, "momenta", (g.bfloat16(), g.bfloat16(), g.bfloat16())),
                                  (ValueError, "grads", (g, g[:2], g)), (ValueError, "momenta", (g, g, g.to("cuda:1"))),
                                  (ValueError, "contiguous", (g.t(), g.t(), g.t())), (ValueError, "contiguous", (g, g, torch.empty(6, 4, device="cuda:0").t()))):
            with pytest.raises(kind, match=match):
                ops.muon_step(*([x] for x in args), 0.1)


# -------------------------------------------------------------- sizes beyond 32 bits
def test_sizes_beyond_32_bits_reach_no_entry_point():
    """A size whose low 32 bits are a valid one is refused where it is converted, not taken for those."""
    big = (1 << 32) + 5
    for call in (lambda: lib().yuf_embedding_grad_workspace(4, big, 8), lambda: lib().yuf_embedding_grad_workspace(4, 8, big),
                 lambda: lib().yuf_newton_schulz_workspace(1, big, 4), lambda: lib().yuf_newton_schulz_workspace(1, 4, -big),
                 lambda: lib().yuf_newton_schulz_workspace(big, 4, 4), lambda: lib().yuf_cross_entropy_workspace(big),
                 lambda: lib().yuf_embedding_grad_workspace(4, 1 << 31, 8), lambda: lib().yuf_embedding_grad_workspace(1 << 64, 8, 8),
                 lambda: lib().yuf_newton_schulz_f32(1, 4, 4, None, None, big, *GOOD[1:], None, None)):
        with pytest.raises(ctypes.ArgumentError, match="bits"):
            call()
    for call in (lambda: lib().yuf_embedding_grad_workspace(4.0, 8, 8), lambda: lib().yuf_newton_schulz_workspace("1", 4, 4)):
        with pytest.raises(ctypes.ArgumentError):
            call()
    assert lib().yuf_embedding_grad_workspace(4, (1 << 31) - 1, 8) == lib().yuf_embedding_grad_workspace(4, -(1 << 31), 8) == 0


def test_python_refuses_sizes_beyond_the_documented_ones():
    from torch._subclasses.fake_tensor import FakeTensorMode

    def empty(*shape):
        return torch.empty(*shape, device="cuda:0", dtype=torch.bfloat16)

    with FakeTensorMode():
        tokens = torch.empty(3, dtype=torch.int64, device="cuda:0")
        for size in ((1 << 24) + 1, 1 << 31, (1 << 32) + 5):
            for weight in (empty(size, 1), empty(5, size)):
                with pytest.raises(ValueError, match="2\\^24"):
                    ops.embedding(tokens, weight)
            for dout, vocab in ((empty(3, 4), size), (empty(3, size), 4)):
                with pytest.raises(ValueError, match="2\\^24"):
                    ops.embedding_grad(tokens, dout, vocab)
        for size in ((1 << 22) + 1, (1 << 32) + 4):
            for x in (empty(size, 1), empty(1, size), empty(2, size, 1)):
                with pytest.raises(ValueError, match="too large"):
                    ops.newton_schulz(x)
            x, m = empty(size, 4), torch.empty(size, 4, device="cuda:0")
            with pytest.raises(ValueError, match="too large"):
                ops.muon_step([x], [x.clone()], [m], 0.1)
        x = empty((1 << 14) + 1, 1 << 14)
        with pytest.raises(ValueError, match="too large"):
            ops.newton_schulz([x, x])
    ops._check_size(0, 1 << 23)  # nothing is not too large
    # The same limit as the library's.
    for rows, cols in ((1 << 14, 1 << 14), ((1 << 14) + 1, 1 << 14), (1, 1 << 20), (1 << 21, 128), ((1 << 21) + 1, 128), (1 << 21, 129), (1 << 22, 1),
                       ((1 << 22) + 1, 1), (1000, 260000), (127, 1 << 21)):
        fits = lib().yuf_newton_schulz_workspace(1, rows, cols) > 0
        try:
            ops._check_size(rows, cols)
        except ValueError:
            assert not fits, (rows, cols)
        else:
            assert fits, (rows, cols)


# ------------------------------------------------------------------- forward mode
def test_tangents_are_refused():
    """A dual tensor's primal alone would be taken, with or without a recorded gradient: every operator raises."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad

    with FakeTensorMode(), forward_ad.dual_level():
        def plain(*shape):
            return torch.empty(shape, device="cuda:0")

        def dual(*shape):
            return forward_ad.make_dual(plain(*shape), plain(*shape))

        tokens = torch.empty(3, dtype=torch.int64, device="cuda:0")
        scan, state, rosa, row = (2, 3, 2, 8), (2, 2, 8, 8), (2, 3, 4), (4,)
        scans, rosas = [plain(*scan) for _ in range(7)], [plain(*rosa), plain(*rosa), plain(*rosa), plain(*row), plain(*row), plain(2, 4), plain(*rosa)]
        calls = [lambda: ops.embedding(tokens, dual(5, 4)), lambda: ops.embedding_grad(tokens, dual(3, 4), 5),
                 lambda: ops.embedding_grad(tokens, plain(3, 4), 5, out=dual(5, 4)), lambda: ops.newton_schulz(dual(4, 4)),
                 lambda: ops.newton_schulz([plain(4, 4), dual(4, 4)]), lambda: ops.dropout(dual(4, 4), 0.5, 1),
                 lambda: ops.dropout(plain(4, 4), 0.5, 1, residual=dual(4, 4)), lambda: ops.cross_entropy(dual(3, 5), tokens),
                 lambda: ops.cross_entropy_grad(dual(3, 5), tokens), lambda: ops.cross_entropy_grad(plain(3, 5), tokens, dloss=dual()),
                 lambda: ops.rwkv7_scan(*scans[:6], dual(*state)), lambda: ops.rwkv7_cuda(*scans[:5], dual(*scan)),
                 lambda: ops.rwkv7_scan_backward(*scans[:6], dual(*scan)), lambda: ops.rwkv7_scan_backward(*scans, dstate=dual(*state)),
                 lambda: ops.rosa_householder_scan(*rosas[:5], dual(2, 4)), lambda: ops.rosa_householder_scan_backward(*rosas[:6], dual(*rosa)),
                 lambda: ops.rosa_householder_scan_backward(*rosas, dmemory=dual(2, 4))]
        for k in range(3):
            lists = [[plain(4, 4)] for _ in range(3)]
            lists[k] = [dual(4, 4)]
            calls.append(lambda lists=lists: ops.muon_step(*lists, 0.1))
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_the_embeddings_gradient_is_not_recorded_in_silence():
    """A dout that wants a gradient would get none: refused, unless nothing is recorded."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        tokens, dout = torch.empty(3, dtype=torch.int64, device="cuda:0"), torch.empty(3, 4, device="cuda:0", requires_grad=True)
        for d in (dout, dout * 2.0):
            for out in (None, torch.empty(5, 4, device="cuda:0")):
                with pytest.raises(ValueError, match="detach"):
                    ops.embedding_grad(tokens, d, 5, out=out)
        with torch.no_grad(), pytest.raises(Exception) as error:  # accepted: what fails is the device that is not there
            ops.embedding_grad(tokens, dout, 5)
        assert "detach" not in str(error.value)


def test_muon_step_names_what_is_no_tensor():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(4, 6, device="cuda:0")
        for name, k in (("params", 0), ("grads", 1), ("momenta", 2)):
            lists = [[x, x] for _ in range(3)]
            lists[k] = [x, None]
            with pytest.raises(TypeError, match=f"{name} must be tensors, got NoneType"):
                ops.muon_step(*lists, 0.1)
