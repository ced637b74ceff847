"""Python mirror of the reference's operator interface for the recurrent scans,
and the operators of a training pass around them.

``rwkv7_cuda`` (yufmusicgen/cuda_ops.py:256-266) and ``rosa_householder_scan``
(yufmusicgen/rosa_cuda.py:157-180) keep their names, argument meaning and
validation errors; they run the gfx950 kernels of ``libyufhip.so`` through the
C ABI on torch's current HIP stream.  Tensors are torch plumbing (device
memory and streams); there is no CPU fallback.

Both scans, ``dropout``, ``cross_entropy`` and ``embedding`` are differentiable once, as the
reference's autograd functions are (cuda_ops.py:189-253, rosa_cuda.py:73-154).
Their gradients are operators too (``rwkv7_scan_backward``,
``rosa_householder_scan_backward``, ``dropout`` itself, ``cross_entropy_grad``,
``embedding_grad``): a HIP graph captures those.  Captured ``backward()`` calls through these
operators raise, because torch ends the process when a capture meets gradient
accumulators that another, still living autograd graph made on a stream outside
of it.  Forward-mode derivatives there are none: an input with a tangent raises.
A capture that holds a backward pass but not its forward pass ends the
process inside torch before an operator is asked.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from ._lib import check, lib

SUPPORTED_HEAD_SIZES = (8, 16, 32, 40, 48, 64, 128)


def _ptr(t):
    return None if t is None else t.data_ptr()


class _on:
    """The device's raw current stream, with the device made current if another is."""

    __slots__ = ("index", "before")

    def __init__(self, device):
        self.index = device.index

    def __enter__(self) -> int:
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc) -> None:
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def _needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _no_tangents(name: str, *tensors) -> None:
    """The kernels see a dual tensor's primal alone: its tangent would be lost."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")


def _scratch(size: int, device):
    """A device buffer of ``size`` bytes, from torch's allocator for the current stream."""
    return torch.empty(size, dtype=torch.uint8, device=device)


def _not_captured(name: str) -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{name}: backward() cannot be captured into a graph; capture the gradient operators")


def _check_one_device(name: str, first, *others) -> None:
    if any(x is not None and x.device != first.device for x in others):
        raise ValueError(f"{name} must be on the same GPU")


def _check_like(name: str, x, shape, device, dtype=torch.float32) -> None:
    if not x.is_cuda or x.device != device:
        raise ValueError(f"{name} must be on the inputs' GPU")
    if x.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}")
    if tuple(x.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {list(shape)}, got {list(x.shape)}")


def rwkv7_scan(r, w, k, v, a, b, state=None):
    """WKV-7 forward scan; returns ``(y [B,T,H,N], final_state [B,H,N,N])``.

    ``state`` (optional, [B,H,N,N], row = value index) is the initial state;
    ``None`` starts from zero like the reference kernel.  Validation follows
    ``cuda_ops.py:200-209``.
    """
    tensors = (r, w, k, v, a, b)
    if r.ndim != 4:
        raise ValueError("RWKV-7 inputs must have shape [B, T, H, N]")
    if not all(x.is_cuda for x in tensors):
        raise ValueError("RWKV-7 inputs must be on the GPU")
    if not all(x.dtype == torch.float32 for x in tensors):
        raise TypeError("the gfx950 scan computes in float32")
    if not all(x.is_contiguous() for x in tensors):
        raise ValueError("RWKV-7 inputs must be contiguous")
    if len({tuple(x.shape) for x in tensors}) != 1:
        raise ValueError("RWKV-7 inputs must have identical shapes")
    batch, steps, heads, size = r.shape
    if size not in SUPPORTED_HEAD_SIZES:
        raise ValueError(f"head size {size} not supported (supported: {SUPPORTED_HEAD_SIZES})")
    if state is not None:
        if state.shape != (batch, heads, size, size) or state.dtype != torch.float32 or not state.is_cuda:
            raise ValueError("state must be a float32 GPU tensor of shape [B, H, N, N]")
        state = state.contiguous()
    _check_one_device("RWKV-7 inputs", *tensors, state)
    _no_tangents("rwkv7_scan", *tensors, state)
    if _needs_grad(*tensors, state):
        return _Rwkv7Scan.apply(*tensors, state)
    return _rwkv7_forward(*tensors, state)


def _rwkv7_forward(r, w, k, v, a, b, state):
    batch, steps, heads, size = r.shape
    y = torch.empty_like(r)
    final = torch.empty(batch, heads, size, size, device=r.device, dtype=torch.float32)
    with _on(r.device) as stream:
        check(lib().yuf_wkv7_scan_f32(batch, steps, heads, size, *(x.data_ptr() for x in (r, w, k, v, a, b)),
                                      _ptr(state), final.data_ptr(), y.data_ptr(), stream))
    return y, final


def rwkv7_cuda(r, w, k, v, a, b):
    """Drop-in for the reference ``rwkv7_cuda`` (zero initial state)."""
    return rwkv7_scan(r, w, k, v, a, b)


def rosa_householder_scan(cand, write, read_raw, decay, direction, memory, gated: bool = False):
    """ROSA scan; returns ``(read [B,T,D], final_memory [B,D])``.

    As the reference operator, ``read`` is H(m_t) and the caller applies the
    sigmoid read gate (model.py:311); ``gated=True`` fuses that gate in.
    ``decay`` is post-sigmoid, ``direction`` a unit vector.
    """
    if cand.ndim != 3:
        raise ValueError("ROSA per-step inputs must have shape [B, T, D]")
    if len({tuple(x.shape) for x in (cand, write, read_raw)}) != 1:
        raise ValueError("ROSA per-step inputs must have identical shapes")
    batch, _, dim = cand.shape
    for name, x, elements in (("decay", decay, dim), ("direction", direction, dim), ("memory", memory, batch * dim)):
        if x.numel() != elements:
            raise ValueError(f"ROSA {name} must have {elements} elements, got shape {list(x.shape)}")
    tensors = [x.float().contiguous() for x in (cand, write, read_raw, decay, direction, memory)]
    if not all(x.is_cuda for x in tensors):
        raise ValueError("ROSA inputs must be on the GPU")
    _check_one_device("ROSA inputs", *tensors)
    _no_tangents("rosa_householder_scan", *tensors)
    if _needs_grad(*tensors):
        cand, write, read_raw, decay, direction, memory = tensors
        return _RosaScan.apply(cand, write, read_raw, decay.reshape(dim), direction.reshape(dim),
                               memory.reshape(batch, dim), gated)
    return _rosa_forward(*tensors, gated)


def _rosa_forward(cand, write, read_raw, decay, direction, memory, gated):
    batch, steps, dim = cand.shape
    read = torch.empty_like(cand)
    final = torch.empty(batch, dim, device=cand.device, dtype=torch.float32)
    with _on(cand.device) as stream:
        check(lib().yuf_rosa_scan_f32(batch, steps, dim, cand.data_ptr(), write.data_ptr(),
                                      read_raw.data_ptr() if gated else None, decay.data_ptr(),
                                      direction.data_ptr(), memory.data_ptr(), final.data_ptr(),
                                      read.data_ptr(), stream))
    return read, final


# ------------------------------------------------------------------ gradients
def rwkv7_scan_backward(r, w, k, v, a, b, dy, state=None, dstate=None):
    """Gradients of ``rwkv7_scan``: ``(dr, dw, dk, dv, da, db, dstate_in)``.

    ``dy`` [B,T,H,N] is the gradient of ``y`` and ``dstate`` [B,H,N,N] that of the
    final state (``None``: zero); the inputs are those of the forward call, under
    its rules.  ``dstate_in`` is the gradient of the initial state (with
    ``state=None``, of the zero state).  Replaces the reference's
    ``_RWKV7CUDAFunction.backward`` (cuda_ops.py:235-253).
    """
    tensors = (r, w, k, v, a, b, dy)
    if r.ndim != 4:
        raise ValueError("RWKV-7 inputs must have shape [B, T, H, N]")
    batch, steps, heads, size = r.shape
    if size not in SUPPORTED_HEAD_SIZES:
        raise ValueError(f"head size {size} not supported (supported: {SUPPORTED_HEAD_SIZES})")
    shape, device = r.shape, r.device
    for x in tensors:
        if x.shape != shape or x.device != device or x.dtype != torch.float32 or not device.type == "cuda":
            for name, t in zip(("r", "w", "k", "v", "a", "b", "dy"), tensors):
                _check_like(name, t, shape, device)
        if not x.is_contiguous():
            raise ValueError("RWKV-7 inputs must be contiguous")
    for name, x in (("state", state), ("dstate", dstate)):
        if x is not None:
            _check_like(name, x, (batch, heads, size, size), r.device)
    _no_tangents("rwkv7_scan_backward", *tensors, state, dstate)
    return _rwkv7_backward(*tensors, state, dstate)


def _rwkv7_backward(r, w, k, v, a, b, dy, state, dstate):
    batch, steps, heads, size = r.shape
    state = None if state is None else state.contiguous()
    dstate = None if dstate is None else dstate.contiguous()
    with _on(r.device) as stream:
        grads = [torch.empty_like(r) for _ in range(6)]
        dstate_in = torch.empty(batch, heads, size, size, device=r.device, dtype=torch.float32)
        space = _scratch(lib().yuf_wkv7_scan_backward_workspace(batch, steps, heads, size), r.device)
        check(lib().yuf_wkv7_scan_backward_f32(
            batch, steps, heads, size, *(x.data_ptr() for x in (r, w, k, v, a, b)), _ptr(state), dy.data_ptr(), _ptr(dstate),
            *(x.data_ptr() for x in grads), dstate_in.data_ptr(), space.data_ptr(), stream))
    return (*grads, dstate_in)


class _Rwkv7Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, r, w, k, v, a, b, state):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(r, w, k, v, a, b, state)
        return _rwkv7_forward(r, w, k, v, a, b, state)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dstate):
        _not_captured("rwkv7_scan")
        *inputs, state = ctx.saved_tensors
        dy = torch.zeros_like(inputs[0]) if dy is None else dy.contiguous()
        *grads, dstate_in = _rwkv7_backward(*inputs, dy, state, dstate)
        grads.append(None if state is None else dstate_in)
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad))


def rosa_householder_scan_backward(cand, write, read_raw, decay, direction, memory, dread, dmemory=None,
                                   gated: bool = False):
    """Gradients of ``rosa_householder_scan``:
    ``(dcand, dwrite, dread_raw, ddecay, ddirection, dmemory_in)``.

    ``dread`` [B,T,D] is the gradient of ``read`` and ``dmemory`` [B,D] that of the
    final memory (``None``: zero).  ``dread_raw`` is ``None`` unless ``gated``.
    ``direction`` is taken as it stands in H(x) = x - 2 (x.u) u: normalise it
    outside and the gradient of the normalisation follows outside too.  Replaces
    ``_RosaHouseholderFunction.backward`` (rosa_cuda.py:117-154).
    """
    if cand.ndim != 3:
        raise ValueError("ROSA per-step inputs must have shape [B, T, D]")
    batch, steps, dim = cand.shape
    names = ("cand", "write", "read_raw", "decay", "direction", "memory", "dread")
    shapes = (cand.shape,) * 3 + ((dim,), (dim,), (batch, dim), cand.shape)
    tensors = [x.float().contiguous() for x in (cand, write, read_raw, decay, direction, memory, dread)]
    for name, x, shape in zip(names, tensors, shapes):
        _check_like(name, x, shape, cand.device)
    if dmemory is not None:
        dmemory = dmemory.float().contiguous()
        _check_like("dmemory", dmemory, (batch, dim), cand.device)
    _no_tangents("rosa_householder_scan_backward", *tensors, dmemory)
    cand, write, read_raw, decay, direction, memory, dread = tensors
    with _on(cand.device) as stream:
        dcand, dwrite, dmemory_in = torch.empty_like(cand), torch.empty_like(cand), torch.empty_like(memory)
        dread_raw = torch.empty_like(cand) if gated else None
        ddecay, ddirection = torch.empty_like(decay), torch.empty_like(decay)
        space = _scratch(lib().yuf_rosa_scan_backward_workspace(batch, steps, dim), cand.device)
        check(lib().yuf_rosa_scan_backward_f32(
            batch, steps, dim, cand.data_ptr(), write.data_ptr(), read_raw.data_ptr() if gated else None,
            decay.data_ptr(), direction.data_ptr(), memory.data_ptr(), dread.data_ptr(), _ptr(dmemory),
            dcand.data_ptr(), dwrite.data_ptr(), _ptr(dread_raw), ddecay.data_ptr(), ddirection.data_ptr(),
            dmemory_in.data_ptr(), space.data_ptr(), stream))
    return dcand, dwrite, dread_raw, ddecay, ddirection, dmemory_in


class _RosaScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cand, write, read_raw, decay, direction, memory, gated):
        ctx.set_materialize_grads(False)
        ctx.gated = gated
        ctx.save_for_backward(cand, write, read_raw, decay, direction, memory)
        return _rosa_forward(cand, write, read_raw, decay, direction, memory, gated)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dread, dmemory):
        _not_captured("rosa_householder_scan")
        inputs = ctx.saved_tensors
        dread = torch.zeros_like(inputs[0]) if dread is None else dread
        grads = rosa_householder_scan_backward(*inputs, dread, dmemory, ctx.gated)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None)


# -------------------------------------------------------------------- dropout
_FLOATS = (torch.float32, torch.bfloat16)


def dropout(x, p: float, seed: int, counter=0, residual=None):
    """``residual + dropout(x)``: each element of ``x`` is dropped with probability
    ``p`` and the rest scaled by 1 / (1 - p) (``residual=None``: without the sum).

    The mask is a function of ``seed``, ``counter`` and the element's index and is
    not stored: the gradient generates it again.  ``counter`` is an int, or an
    int64 GPU tensor of one element that the kernel reads as it runs (advance it
    between the replays of a captured graph, after the backward pass).  float32 or
    bfloat16; other layouts than contiguous are copied.
    """
    if not x.is_cuda:
        raise ValueError("dropout input must be on the GPU")
    if x.dtype not in _FLOATS:
        raise TypeError("dropout takes float32 or bfloat16")
    if residual is not None:
        _check_like("residual", residual, x.shape, x.device, x.dtype)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    counter_dev = None
    if isinstance(counter, torch.Tensor):
        if not counter.is_cuda or counter.device != x.device or counter.dtype != torch.int64 or counter.numel() != 1:
            raise ValueError("counter must be an int or an int64 tensor of one element on the input's GPU")
        counter, counter_dev = 0, counter
    _no_tangents("dropout", x, residual)
    if _needs_grad(x, residual):
        return _Dropout.apply(x, residual, float(p), int(seed), int(counter), counter_dev)
    return _dropout_forward(x, residual, p, seed, counter, counter_dev)


def _dropout_forward(x, residual, p, seed, counter, counter_dev):
    x = x.contiguous()
    residual = None if residual is None else residual.contiguous()
    with _on(x.device) as stream:
        out = torch.empty_like(x)
        entry = lib().yuf_dropout_f32 if x.dtype == torch.float32 else lib().yuf_dropout_bf16
        check(entry(x.numel(), x.data_ptr(), _ptr(residual), float(p), int(seed) & _U64, int(counter) & _U64,
                    _ptr(counter_dev), out.data_ptr(), stream))
    return out


_U64 = 0xFFFFFFFFFFFFFFFF


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, counter, counter_dev):
        ctx.mask = (p, seed, counter)
        ctx.save_for_backward(counter_dev)  # torch refuses the backward pass if it was advanced meanwhile
        return _dropout_forward(x, residual, p, seed, counter, counter_dev)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        _not_captured("dropout")
        (counter_dev,) = ctx.saved_tensors
        dx = _dropout_forward(dout, None, *ctx.mask, counter_dev) if ctx.needs_input_grad[0] else None
        return dx, dout if ctx.needs_input_grad[1] else None, None, None, None, None


# ----------------------------------------------------------------------- loss
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _loss_rows(logits, targets, reduction):
    """The logits as [M, V] rows of unit column stride, and the targets as [M]."""
    if logits.ndim < 2:
        raise ValueError("logits must have shape [..., V]")
    if not logits.is_cuda or targets.device != logits.device:
        raise ValueError("logits and targets must be on the same GPU")
    if logits.dtype not in _FLOATS:
        raise TypeError("cross entropy takes float32 or bfloat16 logits")
    if targets.dtype not in (torch.int32, torch.int64):
        raise TypeError("targets must be int32 or int64")
    if tuple(targets.shape) != tuple(logits.shape[:-1]):
        raise ValueError(f"targets must have shape {list(logits.shape[:-1])}, got {list(targets.shape)}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if logits.shape[-1] == 0:
        raise ValueError("logits must have at least one column")
    if logits.ndim > 2:
        logits, targets = logits.reshape(targets.numel(), logits.shape[-1]), targets.reshape(-1)
    rows = logits
    if rows.stride(-1) != 1 or (rows.shape[0] > 1 and rows.stride(0) < rows.shape[1]):
        rows = rows.contiguous()
    return rows, targets.contiguous()


def _loss_call(rows, targets, ignore_index, reduction, dloss, dlogits, want_loss: bool):
    """Loss of the rows (or None), and their gradient into ``dlogits`` where it is given."""
    count, vocab = rows.shape
    with _on(rows.device) as stream:
        loss = space = None
        if want_loss:
            loss = torch.empty((count,) if reduction == "none" else (), device=rows.device, dtype=torch.float32)
        if reduction != "none":
            space = _scratch(lib().yuf_cross_entropy_workspace(count), rows.device)
        if count == 0 and reduction == "none":
            return loss
        entry = lib().yuf_cross_entropy_f32 if rows.dtype == torch.float32 else lib().yuf_cross_entropy_bf16
        stride = max(rows.stride(0), vocab)  # the stride of a single row says nothing
        stride_out = 0 if dlogits is None else max(dlogits.stride(0), vocab)
        check(entry(count, vocab, rows.data_ptr(), stride, targets.data_ptr(), 8 * targets.element_size(),
                    int(ignore_index), _REDUCTIONS[reduction], _ptr(loss), _ptr(dloss), _ptr(dlogits), stride_out,
                    _ptr(space), stream))
    return loss


def cross_entropy(logits, targets, ignore_index: int = -100, reduction: str = "mean"):
    """Cross-entropy of ``logits`` [..., V] and token ids ``targets`` [...] as float32
    (torch's ``F.cross_entropy`` on [M, V]): a scalar, or [...] for reduction
    "none".  Differentiable by the logits.

    float32 or bfloat16 logits, int32 or int64 targets.  Rows with
    ``ignore_index`` count nowhere; a target outside [0, V) gives NaN, and so does
    a mean over no rows.
    """
    rows, flat = _loss_rows(logits, targets, reduction)
    _no_tangents("cross_entropy", logits)
    if _needs_grad(logits):
        loss = _CrossEntropy.apply(rows, flat, ignore_index, reduction)
    else:
        loss = _loss_call(rows, flat, ignore_index, reduction, None, None, True)
    return loss.reshape(targets.shape) if reduction == "none" else loss


def cross_entropy_grad(logits, targets, ignore_index: int = -100, reduction: str = "mean", dloss=None,
                       inplace: bool = False):
    """``cross_entropy`` and its gradient by the logits in one pass: ``(loss, dlogits)``.

    ``dloss``: gradient of the loss, float32 of its shape (a scaled loss's scale;
    ``None``: ones).  ``inplace`` writes the gradient over the logits.
    """
    rows, flat = _loss_rows(logits, targets, reduction)
    if dloss is not None:
        _check_like("dloss", dloss, targets.shape if reduction == "none" else (), logits.device)
        dloss = dloss.contiguous()
    _no_tangents("cross_entropy_grad", logits, dloss)
    if inplace:
        if rows.data_ptr() != logits.data_ptr():
            raise ValueError("inplace needs logits whose rows are one stride apart")
        dlogits = rows
    else:
        dlogits = torch.empty(rows.shape, device=rows.device, dtype=rows.dtype)
    loss = _loss_call(rows, flat, ignore_index, reduction, dloss, dlogits, True)
    if inplace:
        torch.autograd.graph.increment_version(logits)  # as an in-place operation of torch's does
    loss = loss.reshape(targets.shape) if reduction == "none" else loss
    return loss, logits if inplace else dlogits.reshape(logits.shape)


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, targets, ignore_index, reduction):
        ctx.how = (ignore_index, reduction)
        ctx.save_for_backward(rows, targets)
        return _loss_call(rows, targets, ignore_index, reduction, None, None, True)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        _not_captured("cross_entropy")
        rows, targets = ctx.saved_tensors
        dlogits = torch.empty(rows.shape, device=rows.device, dtype=rows.dtype)
        _loss_call(rows, targets, *ctx.how, dloss.contiguous(), dlogits, False)
        return dlogits, None, None, None


# ------------------------------------------------------------------ embedding
_TABLE_MOST = 1 << 24  # rows, and columns


def _check_tokens(tokens, device) -> None:
    if tokens.device != device:
        raise ValueError("tokens must be on the same GPU")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError("tokens must be int32 or int64")


def _check_padding(padding_idx, vocab: int) -> int:
    if padding_idx is None:
        return -1
    if not 0 <= padding_idx < vocab:
        raise ValueError(f"padding_idx must be in [0, {vocab}), got {padding_idx}")
    return int(padding_idx)


def _check_table(vocab: int, dim: int) -> None:
    if vocab > _TABLE_MOST or dim > _TABLE_MOST:
        raise ValueError(f"a table may have 2^24 rows and columns, got [{vocab}, {dim}]")


def embedding(tokens, weight, scale: float = 1.0, padding_idx=None):
    """``scale * weight[tokens]``: [..., D] for ``tokens`` [...] and ``weight`` [V, D], in
    the weight's type (float32 or bfloat16).  Differentiable by the weight.

    int32 or int64 tokens.  One outside [0, V) gives a row of NaN, and no gradient.
    The row of ``padding_idx`` is looked up like any other and gets no gradient.
    """
    if weight.ndim != 2:
        raise ValueError("weight must have shape [V, D]")
    if not weight.is_cuda:
        raise ValueError("weight must be on the GPU")
    if weight.dtype not in _FLOATS:
        raise TypeError("embedding takes float32 or bfloat16 weights")
    if not weight.is_contiguous():
        raise ValueError("weight must be contiguous")
    _check_table(*weight.shape)
    _no_tangents("embedding", weight)
    _check_tokens(tokens, weight.device)
    padding = _check_padding(padding_idx, weight.shape[0])
    if _needs_grad(weight):
        return _Embedding.apply(tokens, weight, float(scale), padding)
    return _embedding_forward(tokens, weight, scale)


def _embedding_forward(tokens, weight, scale):
    tokens = tokens.contiguous()
    vocab, dim = weight.shape
    with _on(weight.device) as stream:
        out = torch.empty(*tokens.shape, dim, device=weight.device, dtype=weight.dtype)
        entry = lib().yuf_embedding_f32 if weight.dtype == torch.float32 else lib().yuf_embedding_bf16
        check(entry(tokens.numel(), vocab, dim, weight.data_ptr(), tokens.data_ptr(), 8 * tokens.element_size(),
                    float(scale), out.data_ptr(), stream))
    return out


def embedding_grad(tokens, dout, vocab: int, scale: float = 1.0, padding_idx=None, out=None):
    """Gradient of ``embedding`` by its weight: [vocab, D] for ``dout`` [..., D], in dout's type.

    ``out`` (a contiguous [vocab, D] tensor of that type, such as the gradient that a
    tied LM head left): the gradient is added to it, and it is returned.  Each row is
    summed in float32, in an order that the sizes and ids fix.  Not differentiable.
    """
    if dout.ndim < 1 or tuple(dout.shape[:-1]) != tuple(tokens.shape):
        raise ValueError(f"dout must have shape {list(tokens.shape) + ['D']}, got {list(dout.shape)}")
    if not dout.is_cuda:
        raise ValueError("dout must be on the GPU")
    if dout.dtype not in _FLOATS:
        raise TypeError("embedding takes float32 or bfloat16 gradients")
    if vocab < 0:
        raise ValueError(f"vocab must not be negative, got {vocab}")
    _check_table(vocab, dout.shape[-1])
    _check_tokens(tokens, dout.device)
    padding = _check_padding(padding_idx, vocab)
    if out is not None:
        _check_like("out", out, (vocab, dout.shape[-1]), dout.device, dout.dtype)
        if not out.is_contiguous():
            raise ValueError("out must be contiguous")
        if _needs_grad(out):
            raise ValueError("out is written in place: it may not require a gradient")
    if _needs_grad(dout):
        raise ValueError("embedding_grad is not differentiable: detach dout")
    _no_tangents("embedding_grad", dout, out)
    return _embedding_backward(tokens, dout, vocab, scale, padding, out)


def _embedding_backward(tokens, dout, vocab, scale, padding, out=None):
    tokens, dout = tokens.contiguous(), dout.contiguous()
    dim, count = dout.shape[-1], tokens.numel()
    with _on(dout.device) as stream:
        grad = torch.empty(vocab, dim, device=dout.device, dtype=dout.dtype) if out is None else out
        space = _scratch(lib().yuf_embedding_grad_workspace(count, vocab, dim), dout.device)
        entry = lib().yuf_embedding_grad_f32 if dout.dtype == torch.float32 else lib().yuf_embedding_grad_bf16
        check(entry(count, vocab, dim, tokens.data_ptr(), 8 * tokens.element_size(), dout.data_ptr(), float(scale), padding,
                    int(out is not None), grad.data_ptr(), space.data_ptr(), stream))
    if out is not None:
        torch.autograd.graph.increment_version(out)  # as an in-place operation of torch's does
    return grad


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding):
        ctx.how = (weight.shape[0], scale, padding)
        ctx.save_for_backward(tokens)
        return _embedding_forward(tokens, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        _not_captured("embedding")
        (tokens,) = ctx.saved_tensors
        return None, _embedding_backward(tokens, dout, *ctx.how), None, None


# ------------------------------------------------------------- weight update
_NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # Jordan's, of the Muon optimiser


def _pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def _check_matrices(name: str, matrices, device, dtype) -> None:
    for x in matrices:
        if x.ndim != 2:
            raise ValueError(f"{name} must be matrices, got shape {list(x.shape)}")
        if not x.is_cuda or x.device != device:
            raise ValueError(f"{name} must be on the same GPU")
        if x.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}")


def _check_size(rows: int, cols: int) -> None:
    padded = (rows + 127) // 128 * ((cols + 127) // 128) << 14
    if rows and cols and (max(rows, cols) > 1 << 22 or padded > 1 << 28):
        raise ValueError(f"matrices of shape {[rows, cols]} are too large")


def _check_apart(written, read) -> None:
    """Contiguous tensors that are written share memory with none of the others."""
    def end(x):
        return x.data_ptr() + x.element_size() * (1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride())))

    runs = sorted((x.device.index, x.data_ptr(), end(x), kind) for kind, xs in ((True, written), (False, read)) for x in xs if x.numel())
    device, any_end, written_end = None, 0, 0
    for index, begin, stop, kind in runs:
        if index != device:
            device, any_end, written_end = index, 0, 0
        if begin < written_end or (kind and begin < any_end):
            raise ValueError("params, grads and momenta may not overlap")
        any_end = max(any_end, stop)
        if kind:
            written_end = max(written_end, stop)


def newton_schulz(x, steps: int = 5, coefficients=_NS_COEFFICIENTS, eps: float = 1e-7):
    """Matrices orthogonalised by Newton-Schulz products: ``X = x / (|x|_F + eps)``, then
    ``steps`` times ``A = X X^T, X <- a X + (b A + c A A) X``, on the transpose where there
    are more rows than columns.

    ``x``: [..., R, C], or a list of [R, C] of one shape (and a list is returned); float32
    or bfloat16.  Products are of operands with 22 bits, summed in float32 (about the error of
    float32 products); the result is rounded to x's type once.  Not differentiable.
    """
    several = isinstance(x, (list, tuple))
    if several:
        if not x:
            return []
        first = x[0]
        if any(m.shape != first.shape for m in x):
            raise ValueError("matrices of a list must have one shape")
    else:
        first = x
    if first.ndim < 2 or (several and first.ndim != 2):
        raise ValueError("x must have shape [..., R, C], or be a list of [R, C]")
    if not first.is_cuda:
        raise ValueError("x must be on the GPU")
    if first.dtype not in _FLOATS:
        raise TypeError("newton_schulz takes float32 or bfloat16")
    if several:
        _check_matrices("x", x, first.device, first.dtype)
    _no_tangents("newton_schulz", *(x if several else (x,)))
    if _needs_grad(*(x if several else (x,))):
        raise ValueError("newton_schulz is not differentiable: detach its input")
    a, b, c = coefficients
    rows, cols = first.shape[-2:]
    _check_size(rows, cols)
    with _on(first.device) as stream:
        if several:
            taken = [m.contiguous() for m in x]
            out = [torch.empty_like(m) for m in taken]
            sources, targets, count = _pointers(taken), _pointers(out), len(x)
        else:
            taken = x.contiguous()
            out = torch.empty_like(taken)
            count = out.numel() // (rows * cols) if out.numel() else 0
            size = rows * cols * out.element_size()
            sources, targets = ((ctypes.c_void_p * count)(*[t.data_ptr() + i * size for i in range(count)]) for t in (taken, out))
        space = _scratch(lib().yuf_newton_schulz_workspace(count, rows, cols), first.device)
        entry = lib().yuf_newton_schulz_f32 if first.dtype == torch.float32 else lib().yuf_newton_schulz_bf16
        check(entry(count, rows, cols, sources, targets, int(steps), float(a), float(b), float(c), float(eps),
                    space.data_ptr(), stream))
    return out


def muon_step(params, grads, momenta, lr: float, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
              steps: int = 5, coefficients=_NS_COEFFICIENTS, eps: float = 1e-7) -> None:
    """One update of weight matrices by their orthogonalised momenta, in place:
    ``m <- momentum m + (1 - momentum) g``; ``u = momentum m + (1 - momentum) g`` (or ``m`` without
    ``nesterov``); ``p <- (1 - lr weight_decay) p - lr sqrt(max(1, rows / cols)) newton_schulz(u)``.

    Lists of matrices, of any shapes; those of one shape are updated together.  A weight
    without a gradient is left out of all three.  ``params`` and ``grads`` float32 or bfloat16,
    ``momenta`` float32.  ``params`` and ``momenta`` must be contiguous.  Parameters that
    require a gradient are updated like an optimiser does, without being recorded.
    """
    if not len(params) == len(grads) == len(momenta):
        raise ValueError(f"as many grads and momenta as params: got {len(params)}, {len(grads)} and {len(momenta)}")
    a, b, c = coefficients
    groups = {}
    for p, g, m in zip(params, grads, momenta):
        for name, x in (("params", p), ("grads", g), ("momenta", m)):
            if not isinstance(x, torch.Tensor):
                raise TypeError(f"{name} must be tensors, got {type(x).__name__}: leave a weight without a gradient out of all three lists")
        if not p.is_cuda:
            raise ValueError("params must be on the GPU")
        if p.dtype not in _FLOATS:
            raise TypeError("muon_step takes float32 or bfloat16 params")
        _check_matrices("params", (p,), p.device, p.dtype)
        _check_like("grads", g, p.shape, p.device, p.dtype)
        _check_like("momenta", m, p.shape, p.device)
        if not p.is_contiguous() or not m.is_contiguous():
            raise ValueError("params and momenta must be contiguous")
        _check_size(*p.shape)
        groups.setdefault((p.shape, p.dtype, p.device), []).append((p, g, m))
    _no_tangents("muon_step", *params, *grads, *momenta)
    if len(groups) > 1:  # the library sees one group at a time, and all are refused before one is updated
        _check_apart((*params, *momenta), grads)
    for ((rows, cols), dtype, device), members in groups.items():
        ps, gs, ms = zip(*members)
        with _on(device) as stream:
            gs = [g.contiguous() for g in gs]
            space = _scratch(lib().yuf_newton_schulz_workspace(len(ps), rows, cols), device)
            entry = lib().yuf_muon_step_f32 if dtype == torch.float32 else lib().yuf_muon_step_bf16
            check(entry(len(ps), rows, cols, _pointers(ps), _pointers(gs), _pointers(ms), float(lr), float(momentum),
                        int(bool(nesterov)), float(weight_decay), int(steps), float(a), float(b), float(c), float(eps),
                        space.data_ptr(), stream))
        for x in (*ps, *ms):
            torch.autograd.graph.increment_version(x)  # as an in-place operation of torch's does
