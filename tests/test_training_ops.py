"""The training pass's operators without a GPU: what they refuse, before any device call."""

import ctypes

import pytest
import torch

from yufmusicgen_amd import ops
from yufmusicgen_amd._lib import lib

DUMMY = 256  # never dereferenced: each call returns before any device work


def refused(status, *words):
    message = lib().yuf_last_error().decode()
    assert status == -1, (status, message)
    assert all(w in message for w in words), message


def test_wkv7_backward_refusals():
    call = lib().yuf_wkv7_scan_backward_f32
    full = [DUMMY] * 9 + [2 * DUMMY] * 8 + [None]  # inputs, then outputs and workspace: none aliases
    refused(call(1, 1, 1, 12, *full), "head size")
    refused(call(-1, 1, 1, 40, *full), "negative")
    refused(call(1, 1, 1, 40, *[None] * 18), "null")
    refused(call(1, 0, 1, 40, *[None] * 18), "workspace")
    refused(call(1, 1, 1, 40, *full[:16], None, None), "workspace")
    refused(call(1, 1, 1, 40, *full[:16], DUMMY + 64, None), "aligned")
    apart = [256 * (i + 1) for i in range(17)] + [None]
    for out, inp in ((9, 0), (14, 7), (15, 8), (10, 6), (13, 9)):  # an output as an input, and as another output
        refused(call(1, 1, 1, 40, *apart[:out], apart[inp], *apart[out + 1 :]), "may not be")
    refused(call(1, 1, 1 << 20, 40, *full), "H * N")
    refused(call(1 << 14, 1 << 12, 1 << 10, 40, *full), "chunks")
    for missing in (0, 1, 2, 3, 4, 5, 7, 9, 10, 11, 12, 13, 14):
        args = list(full)
        args[missing] = None
        refused(call(1, 1, 1, 40, *args), "null")
    assert call(0, 5, 3, 40, *[None] * 18) == 0 and call(5, 5, 0, 40, *[None] * 18) == 0
    space = lib().yuf_wkv7_scan_backward_workspace
    assert space(1, 16, 1, 12) == space(0, 16, 1, 40) == space(1, -1, 1, 40) == 0
    assert space(1, 0, 1, 40) > 0 and space(8, 2048, 16, 40) > space(8, 1024, 16, 40)


def test_rosa_backward_refusals():
    call = lib().yuf_rosa_scan_backward_f32
    full = [DUMMY] * 8 + [2 * DUMMY] * 7 + [None]
    refused(call(1, 1, 2048, *full), "D must be")
    refused(call(1, 1, 0, *full), "D must be")
    refused(call(1, -1, 64, *full), "negative")
    for missing in (0, 1, 3, 4, 6, 8, 9, 11, 12):
        args = list(full)
        args[missing] = None
        refused(call(1, 1, 64, *args), "null")
    args = list(full)
    args[10] = None  # dread_raw without its read_raw's gradient
    refused(call(1, 1, 64, *args), "read_raw")
    refused(call(1, 1, 64, *full[:14], None, None), "workspace")
    refused(call(1, 1, 64, *full[:14], DUMMY + 64, None), "aligned")
    apart = [256 * (i + 1) for i in range(15)] + [None]
    for out, inp in ((8, 0), (9, 6), (10, 2), (11, 3), (13, 7), (12, 11)):
        refused(call(1, 1, 64, *apart[:out], apart[inp], *apart[out + 1 :]), "may not be")
    refused(call(1 << 20, 1 << 20, 64, *full), "blocks")
    space = lib().yuf_rosa_scan_backward_workspace
    assert space(1, 16, 1025) == space(0, 16, 64) == space(1, -1, 64) == 0 and space(1, 0, 64) > 0


def test_dropout_refusals():
    for name in ("yuf_dropout_f32", "yuf_dropout_bf16"):
        call = getattr(lib(), name)
        refused(call(-1, DUMMY, None, 0.5, 0, 0, None, DUMMY, None), "negative")
        for p in (-0.1, 1.1, float("nan")):
            refused(call(8, DUMMY, None, p, 0, 0, None, DUMMY, None), "p must be")
        refused(call(8, None, None, 0.5, 0, 0, None, DUMMY, None), "null")
        refused(call(8, DUMMY, None, 0.5, 0, 0, None, None, None), "null")
        refused(call(1 << 62, DUMMY, None, 0.5, 0, 0, None, DUMMY, None), "too many")
        assert call(0, None, None, 0.5, 0, 0, None, None, None) == 0


def test_cross_entropy_refusals():
    for name in ("yuf_cross_entropy_f32", "yuf_cross_entropy_bf16"):
        call = getattr(lib(), name)

        def bad(*words, M=4, V=10, logits=DUMMY, ld=10, targets=DUMMY, bits=32, reduction=1, loss=DUMMY, dlogits=None,
                ld_out=0, space=DUMMY):
            refused(call(M, V, logits, ld, targets, bits, -100, reduction, loss, None, dlogits, ld_out, space, None), *words)

        bad("negative", M=-1)
        bad("negative", V=-1, ld=0)
        bad("without logits", V=0, ld=0)
        bad("stride", ld=9)
        bad("stride", dlogits=DUMMY * 2, ld_out=9)
        bad("in place", dlogits=DUMMY, ld_out=12)
        bad("target_bits", bits=16)
        bad("reduction", reduction=3)
        bad("null", logits=None)
        bad("null", targets=None)
        bad("neither", loss=None)
        bad("workspace", space=None)
    assert lib().yuf_cross_entropy_workspace(-1) == 0 and lib().yuf_cross_entropy_workspace(10) >= 44


def test_python_refusals():
    x = torch.zeros(1, 4, 2, 40)
    with pytest.raises(ValueError, match="GPU"):
        ops.rwkv7_scan_backward(*[x] * 7)
    with pytest.raises(ValueError, match="head size"):
        ops.rwkv7_scan_backward(*[torch.zeros(1, 4, 2, 12)] * 7)
    with pytest.raises(ValueError, match="shape"):
        ops.rwkv7_scan_backward(*[torch.zeros(4, 2, 40)] * 7)
    seq, vec = torch.zeros(1, 4, 64), torch.zeros(64)
    with pytest.raises(ValueError, match="GPU"):
        ops.rosa_householder_scan_backward(seq, seq, seq, vec, vec, torch.zeros(1, 64), seq)
    with pytest.raises(ValueError, match="shape"):
        ops.rosa_householder_scan_backward(vec, vec, vec, vec, vec, vec, vec)
    with pytest.raises(ValueError, match="GPU"):
        ops.dropout(vec, 0.5, 1)
    with pytest.raises(ValueError, match="GPU"):
        ops.cross_entropy(torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="shape"):
        ops.cross_entropy(vec, torch.zeros(64, dtype=torch.int64))


def test_the_abi_takes_ctypes_integers_of_full_width():
    """Seeds and counters are 64-bit: a cut one would repeat masks."""
    from yufmusicgen_amd._lib import SIGNATURES

    for name in ("yuf_dropout_f32", "yuf_dropout_bf16"):
        args = SIGNATURES[name][1]
        assert args[0] is ctypes.c_int64 and args[4] is args[5] is ctypes.c_uint64 and args[3] is ctypes.c_double


@pytest.mark.parametrize("reduction", [0, 1, 2])
def test_cross_entropy_gradient_of_no_rows(reduction):
    """A backward pass over no rows has an empty gradient, whose pointer is null: there is nothing to do."""
    for name in ("yuf_cross_entropy_f32", "yuf_cross_entropy_bf16"):
        call = getattr(lib(), name)
        for bits in (32, 64):
            status = call(0, 10, None, 10, None, bits, -100, reduction, None, DUMMY, None, 10, DUMMY, None)
            assert status == 0, lib().yuf_last_error().decode()


def test_scratch_of_refused_sizes_is_none():
    """A workspace query gives 0 for every size that its operator refuses -- not terabytes that a caller
    would ask the allocator for -- and the operator names the reason, with or without that buffer."""
    call, space = lib().yuf_wkv7_scan_backward_f32, lib().yuf_wkv7_scan_backward_workspace
    full = [256 * (i + 1) for i in range(17)] + [None]
    for sizes, word in (((1, 1, 1 << 20, 40), "H * N"), ((1 << 14, 1 << 12, 1 << 10, 40), "chunks"),
                        ((1 << 15, 17, 1 << 10, 8), "chunks"), ((1 << 15, 0, 1 << 10, 128), "heads"),
                        ((1 << 15, 1, 1 << 10, 32), "heads"), ((1 << 13, 1, 1 << 10, 128), "heads")):
        assert space(*sizes) == 0, sizes
        refused(call(*sizes, *full), word)
        refused(call(*sizes, *full[:16], None, None), word)  # not for want of the buffer
    for sizes in ((1 << 15, 16, 1 << 10, 8), (1 << 12, 1, 1 << 10, 128), (1, 1, 1 << 17, 128)):
        assert space(*sizes) > 0, sizes
    call, space = lib().yuf_rosa_scan_backward_f32, lib().yuf_rosa_scan_backward_workspace
    full = [256 * (i + 1) for i in range(15)] + [None]
    for sizes in ((1 << 20, 1 << 20, 64), (1 << 22, 0, 64), (1 << 17, 1024, 256), (1 << 16, 1024, 257)):
        assert space(*sizes) == 0, sizes
        refused(call(*sizes, *full), "blocks")
        refused(call(*sizes, *full[:14], None, None), "blocks")
    for sizes in (((1 << 22) - 1, 32, 64), ((1 << 17) - 1, 1024, 256), ((1 << 16) - 1, 1024, 512)):
        assert space(*sizes) > 0, sizes


def test_outputs_that_share_memory_are_refused():
    """Not only an output that is an input: one that begins inside of it, or inside of the workspace."""
    batch, steps, heads, size = 2, 16, 3, 40
    token, state = 4 * batch * steps * heads * size, 4 * batch * heads * size * size
    call, space = lib().yuf_wkv7_scan_backward_f32, lib().yuf_wkv7_scan_backward_workspace(batch, steps, heads, size)
    # r, w, k, v, a, b, state, dy, dstate, then dr, dw, dk, dv, da, db, dstate_in, workspace.
    sizes = [token] * 6 + [state, token, state] + [token] * 6 + [state, space]
    at = [1 << 20]
    for n in sizes:
        at.append((at[-1] + n + 255) // 256 * 256)

    def overlapping(out, other, by):
        where = list(at[:17])
        where[out] = at[other] + by
        refused(call(batch, steps, heads, size, *where, None), "may not be")

    for out in range(9, 17):
        for other in (*range(9), *range(9, 17)):
            if other != out:
                overlapping(out, other, 0)
                overlapping(out, other, (sizes[other] - 4) // 256 * 256)  # its last words
                overlapping(out, other, -((sizes[out] - 4) // 256 * 256))  # the output's last words
    batch, steps, dim = 2, 40, 64
    token, memory, vec = 4 * batch * steps * dim, 4 * batch * dim, 4 * dim
    call, space = lib().yuf_rosa_scan_backward_f32, lib().yuf_rosa_scan_backward_workspace(batch, steps, dim)
    sizes = [token, token, token, vec, vec, memory, token, memory, token, token, token, vec, vec, memory, space]
    at = [1 << 20]
    for n in sizes:
        at.append((at[-1] + n + 255) // 256 * 256)
    for out in range(8, 15):
        for other in range(15):
            for by in (0, (sizes[other] - 4) // 256 * 256, -((sizes[out] - 4) // 256 * 256)):
                if other != out:
                    where = list(at[:15])
                    where[out] = at[other] + by
                    refused(call(batch, steps, dim, *where, None), "may not be")
    for name, size in (("yuf_dropout_f32", 4), ("yuf_dropout_bf16", 2)):
        call, n, x, far = getattr(lib(), name), 5000, 1 << 20, 1 << 22
        for by in (size, n * size - size, -size, size - n * size):
            refused(call(n, x, None, 0.5, 0, 0, None, x + by, None), "not a part")
            refused(call(n, far, x, 0.5, 0, 0, None, x + by, None), "not a part")
    for name, size in (("yuf_cross_entropy_f32", 4), ("yuf_cross_entropy_bf16", 2)):
        call, rows, vocab, ld, x, far = getattr(lib(), name), 7, 50, 100, 1 << 20, 1 << 22

        def grad(by, ld_out=ld):
            return call(rows, vocab, x, ld, far, 64, -100, 0, far, None, x + by * size, ld_out, None, None)

        for by in (1, 49, -1, -49, 51, -51, 99, 6 * 100 + 49, -6 * 100 - 49):
            refused(grad(by), "not overlap")
        refused(grad(50, 99), "not overlap")  # strides that differ: some row meets another


def test_scans_refuse_vectors_of_other_sizes():
    """The kernels read D elements of decay and direction and B D of the memory: fewer lie beyond their ends."""
    seq, vec, memory = torch.zeros(2, 4, 64), torch.zeros(64), torch.zeros(2, 64)
    for what, args in (("decay", (vec[:1], vec, memory)), ("decay", (vec[0], vec, memory)),
                       ("direction", (vec, vec[:63], memory)), ("direction", (vec, memory, memory)),
                       ("memory", (vec, vec, memory[:1])), ("memory", (vec, vec, torch.zeros(3, 64)))):
        with pytest.raises(ValueError, match=f"ROSA {what} must have"):
            ops.rosa_householder_scan(seq, seq, seq, *args)
    with pytest.raises(ValueError, match="GPU"):  # their own sizes, in any shape
        ops.rosa_householder_scan(seq, seq, seq, vec.reshape(1, 64), vec.reshape(64, 1), memory.reshape(128))


def test_operators_refuse_tensors_of_two_gpus():
    """Stand-ins for tensors of two GPUs: each input in turn on the other one."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        def on(k, *shapes):
            return [torch.empty(*s, device=f"cuda:{int(i == k)}") for i, s in enumerate(shapes)]

        token, vec, state = (1, 4, 2, 40), (64,), (1, 2, 40, 40)
        for k in range(1, 7):
            *x, s = on(k, *[token] * 6, state)
            with pytest.raises(ValueError, match="same GPU"):
                ops.rwkv7_scan(*x, state=s)
        for k in range(1, 9):
            *x, s, ds = on(k, *[token] * 7, state, state)
            with pytest.raises(ValueError, match="inputs' GPU"):
                ops.rwkv7_scan_backward(*x, state=s, dstate=ds)
        seq, memory = (1, 4, 64), (1, 64)
        for k in range(1, 6):
            with pytest.raises(ValueError, match="same GPU"):
                ops.rosa_householder_scan(*on(k, seq, seq, seq, vec, vec, memory))
        for k in range(1, 8):
            with pytest.raises(ValueError, match="inputs' GPU"):
                ops.rosa_householder_scan_backward(*on(k, seq, seq, seq, vec, vec, memory, seq, memory))
        x, other = on(1, (3, 5), (3, 5))
        with pytest.raises(ValueError, match="inputs' GPU"):
            ops.dropout(x, 0.5, 1, residual=other)
        with pytest.raises(ValueError, match="same GPU"):
            ops.cross_entropy(x, torch.empty(3, dtype=torch.int64, device="cuda:1"))


def test_scans_of_no_sequences():
    """An empty batch's tensors are null: nothing to do, for the scans as for their gradients."""
    assert lib().yuf_wkv7_scan_f32(0, 5, 3, 40, *[None] * 10) == 0 and lib().yuf_wkv7_scan_f32(5, 5, 0, 40, *[None] * 10) == 0
    for name in ("yuf_rosa_scan_f32", "yuf_rosa_scan_f32_noalloc"):
        assert getattr(lib(), name)(0, 5, 64, None, None, None, DUMMY, DUMMY, *[None] * 4) == 0
    refused(lib().yuf_wkv7_scan_f32(1, 5, 3, 40, *[None] * 10), "null")
    refused(lib().yuf_rosa_scan_f32(1, 5, 64, None, None, None, DUMMY, DUMMY, *[None] * 4), "null")


def test_gradients_of_no_sequences_take_any_other_size():
    assert lib().yuf_wkv7_scan_backward_f32(0, 5, 1 << 20, 40, *[None] * 18) == 0
    assert lib().yuf_wkv7_scan_backward_workspace(0, 5, 1 << 20, 40) == 0
