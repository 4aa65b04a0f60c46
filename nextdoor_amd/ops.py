"""Operators of models that train on samples, on torch tensors of the GPU.

Walks are sequences of different lengths whose words are the vertices of the graph.  A training step
over a batch of them needs

* :func:`packed_attention`: causal attention within each walk of a packed batch, with grouped heads;
* :func:`dropout`: from the samplers' own random stream, the mask never stored;
* :func:`vocabulary_loss`: softmax cross entropy over all vertices, the logits never stored.

Each has a ``_forward`` and a ``_backward`` function and a differentiable form that calls both.  They
enqueue the library's HIP kernels (include/nextdoor_amd.h) on torch's current stream of the tensors'
device and wait for nothing; results are new tensors.  There is no other implementation: CPU tensors,
types and shapes that the kernels do not have are errors (:class:`NextDoorError`).

Import this module (or torch) before the first call into the library: torch brings its own HIP
runtime, and streams and memory can only be shared within one.
"""
import ctypes as C
import functools
import math

import numpy as np
import torch

from . import _capi
from ._capi import NextDoorError, PackedAttention, VocabularyLoss, check

__all__ = ["PackedSequences", "packed_attention", "packed_attention_forward", "packed_attention_backward",
           "vocabulary_loss", "vocabulary_loss_forward", "vocabulary_loss_backward", "dropout", "dropout_forward",
           "dropout_backward", "NextDoorError"]

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # ND_F32, ND_F16, ND_BF16
_lib = None


def _library():
    global _lib
    if _lib is None:
        handle = _capi.lib()
        with open("/proc/self/maps") as maps:
            runtimes = {line.split()[-1] for line in maps if "libamdhip64" in line}
        if len(runtimes) > 1:
            raise NextDoorError("the library was loaded before torch, on a HIP runtime of its own: import torch (or "
                                "nextdoor_amd.ops) before the first call into nextdoor_amd")
        _lib = handle
    return _lib


def _on_gpu(what, first, *others):
    """Checks that all are tensors on one GPU; returns its index."""
    try:
        index = first.get_device()
        for t in others:
            if t.get_device() != index:
                index = -1
    except AttributeError:
        index = -1
    if index < 0:
        if not all(isinstance(t, torch.Tensor) and t.is_cuda for t in (first, *others)):
            raise NextDoorError("%s: tensors on the GPU only" % what)
        raise NextDoorError("%s: tensors on different devices" % what)
    return index


_raw_stream = torch._C._cuda_getCurrentRawStream  # what torch.cuda.current_stream wraps in an object


def _run(index, fn, *args):
    """Calls an entry point that takes a stream last, on torch's current one, with the device current."""
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        check(rc)


# ---- dropout -------------------------------------------------------------------------------------


def _dropout(x, p, seed, step, residual):
    index = _on_gpu("dropout", x) if residual is None else _on_gpu("dropout", x, residual)
    if x.dtype not in _DTYPES:
        raise NextDoorError("dropout: no kernel for %s" % x.dtype)
    if not 0.0 <= p <= 1.0:
        raise NextDoorError("dropout: p is a probability, %r given" % (p,))
    if not 0 <= seed < 1 << 64:
        raise NextDoorError("dropout: a seed has 64 bits, %r given" % (seed,))
    if not 0 <= step < 1 << 31:
        raise NextDoorError("dropout: step numbers are below 2^31, %r given" % (step,))
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise NextDoorError("dropout: the residual is of another shape or type")
        residual = residual.contiguous()
    x = x.contiguous()
    out = torch.empty_like(x)
    _run(index, _library().nd_dropout, x.data_ptr(), None if residual is None else residual.data_ptr(), out.data_ptr(),
         x.numel(), _DTYPES[x.dtype], p, seed, step)
    return out


def dropout_forward(x, p, seed, step, residual=None):
    """x / (1 - p) where an element is kept, 0 where it is dropped (whatever it holds), plus the residual.  Element o
    (in row-major order) is kept if ``philox_fill_uniform(seed, step, o, 1, step_size=2) >= p``: give each
    dropout of a training step its own ``step``.  Sums are rounded once."""
    return _dropout(x, p, seed, step, residual)


def dropout_backward(dout, p, seed, step):
    """The gradient of x; the residual's is ``dout`` itself."""
    return _dropout(dout, p, seed, step, None)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, step):
        ctx.how = p, seed, step
        ctx.has_residual = residual is not None
        return _dropout(x, p, seed, step, residual)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        dx = dropout_backward(dout, *ctx.how) if ctx.needs_input_grad[0] else None
        return dx, dout if ctx.has_residual and ctx.needs_input_grad[1] else None, None, None, None


def dropout(x, p, seed, step, residual=None):
    """:func:`dropout_forward`, differentiable in x and the residual."""
    return _Dropout.apply(x, residual, p, seed, step)


# ---- packed attention ------------------------------------------------------------------------------


class PackedSequences:
    """Where the sequences of a packed batch lie: sequence i is tokens ``starts[i] .. starts[i + 1] - 1``.

    ``starts`` (a list, a numpy array or a tensor; integers) begins with 0 and does not fall; a tensor on the GPU is
    read back to be checked, which waits for it.  ``n_tokens`` (default: ``starts[-1]``) may be larger: tokens after
    the last sequence belong to none.  Make one per batch; every layer and both directions use it (30 to 50 us on the host).
    Like any tensor it is filled on the stream that is current here: a call on another stream has to come after that
    (``stream.wait_stream``), and it has to live until such a call is done.  Not while a graph is recorded."""

    def __init__(self, starts, n_tokens=None, device=None):
        if isinstance(starts, torch.Tensor):
            if starts.is_floating_point():
                raise NextDoorError("packed sequences: starts are integers")
            device = device if device is not None or not starts.is_cuda else starts.device
            starts = starts.cpu().numpy()
        starts = np.asarray(starts)
        if not (starts.ndim == 1 and len(starts) >= 1 and starts.dtype.kind in "iu"):
            raise NextDoorError("packed sequences: starts is a list of integers, one more than there are sequences")
        if not (starts.min() >= 0 and starts.max() <= 2147483392):
            raise NextDoorError("packed sequences: starts out of range")
        starts = np.ascontiguousarray(starts, dtype=np.int32)
        self.device = torch.device("cuda" if device is None else device)
        if self.device.type != "cuda":
            raise NextDoorError("packed sequences: on a GPU only")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.n_sequences, self.n_covered = len(starts) - 1, int(starts[-1])
        self.n_tokens = self.n_covered if n_tokens is None else int(n_tokens)
        lib = _library()
        size = lib.nd_packed_plan_bytes(self.n_tokens)
        if size < 0:
            raise NextDoorError("packed sequences: no plan for %d tokens" % self.n_tokens)
        on_device = torch.from_numpy(starts).to(self.device)
        self.plan = torch.empty(max(size, 16), dtype=torch.uint8, device=self.device)
        sizes = (C.c_int64 * 3)()
        _run(self.device.index, lib.nd_packed_plan, starts.ctypes.data, self.n_sequences, self.n_tokens,
             on_device.data_ptr(), self.plan.data_ptr(), sizes)
        self.sizes = tuple(sizes)
        self.workspace_sizes = {}  # of attention calls over this batch


def _heads(what, x, tokens, dim):
    """A [token, head, dim] tensor as the kernels read it - dim side by side, the rest strided by multiples of 16 bytes -
    and its strides.  Anything else is copied."""
    shape = x.shape
    if not (len(shape) == 3 and shape[0] == tokens):
        raise NextDoorError("packed attention: %s is not [%d tokens, heads, dim]" % (what, tokens))
    if shape[2] != dim:
        raise NextDoorError("packed attention: %s has another head size" % what)
    a, b, c = x.stride()
    # (of one token or one head the stride is never used, but torch keeps it, also in contiguous() and clone())
    a, b = a if tokens > 1 else 0, b if shape[1] > 1 else 0
    if (c != 1 and dim > 1) or a % 8 or b % 8 or a > 16777216 or x.data_ptr() % 16:
        x = torch.empty(shape, dtype=x.dtype, device=x.device).copy_(x)
        a, b = x.stride()[:2]
    return x, a, b


def _attention(sequences, q, k, v, scale, dout=None):
    """Checked arguments: (device index, the tensors read, the struct's first fields, shape of lse)."""
    index = _on_gpu("packed attention", q, k, v, sequences.plan)
    dtype = q.dtype
    if not (dtype is torch.bfloat16 or dtype is torch.float16):
        raise NextDoorError("packed attention: 16-bit types only, %s given" % dtype)
    if not (k.dtype is dtype and v.dtype is dtype):
        raise NextDoorError("packed attention: q, k and v are of different types")
    tokens, dim = sequences.n_tokens, q.shape[-1] if q.dim() else 0
    q, q_token, q_head = _heads("q", q, tokens, dim)
    k, k_token, k_head = _heads("k", k, tokens, dim)
    v, v_token, v_head = _heads("v", v, tokens, dim)
    if k.shape != v.shape:
        raise NextDoorError("packed attention: k and v are of different shapes")
    heads = q.shape[1]
    d_at, d_token, d_head = None, 0, 0
    if dout is not None:
        if not (dout.shape == q.shape and dout.dtype is dtype):
            raise NextDoorError("packed attention: dout is of another shape or type than q")
        dout, d_token, d_head = _heads("dout", dout, tokens, dim)
        d_at = dout.data_ptr()
    scale = 1 / math.sqrt(max(dim, 1)) if scale is None else scale
    fields = (tokens, sequences.n_covered, *sequences.sizes, heads, k.shape[1], dim, _DTYPES[dtype], scale,
              sequences.plan.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), d_at,
              q_token, q_head, k_token, k_head, v_token, v_head, d_token, d_head)
    return index, (q, k, v, dout), fields, (heads, tokens)


def _workspace(sequences, a, sizes, backward, device):
    """The workspace of a call, if it needs one (a call that no kernel can do has none: the call says why)."""
    key = sizes, backward
    size = sequences.workspace_sizes.get(key)
    if size is None:
        size = sequences.workspace_sizes[key] = _library().nd_packed_attention_workspace(a, backward)
    if size <= 0:
        return None
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), size
    return workspace


def packed_attention_forward(q, k, v, sequences, scale=None):
    """Causal attention within each sequence: (out, lse).

    q, out: [tokens, heads, dim]; k, v: [tokens, kv_heads, dim], ``heads / kv_heads`` query heads to each; dim a
    multiple of 8 up to 128; float16 or bfloat16.  Slices of one projection are read in place.  lse:
    [heads, tokens], float32, for the backward pass.  ``scale`` is 1 / sqrt(dim) unless given.  Rows of tokens that
    belong to no sequence are 0 (lse -inf) and their inputs are not read.  Weights are rounded to the type of q before they
    meet v, results once."""
    index, keep, fields, rows = _attention(sequences, q, k, v, scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(rows, dtype=torch.float32, device=q.device)
    a = PackedAttention(*fields, out.data_ptr(), lse.data_ptr())
    workspace = _workspace(sequences, a, (q.shape, k.shape, q.dtype), 0, q.device)
    _run(index, _library().nd_packed_attention_forward, a)
    del keep, workspace
    return out, lse


def packed_attention_backward(dout, q, k, v, out, lse, sequences, scale=None):
    """(dq, dk, dv) for the gradient ``dout`` of ``out``, which with ``lse`` is the forward pass's.  Weights and their gradients
    are rounded to the type of q before their second product (float16: times a power of two, so that small ones are not
    lost).  The first token of a sequence, which sees itself only, has dq = 0 exactly."""
    _on_gpu("packed attention", q, dout, out, lse)
    index, keep, fields, rows = _attention(sequences, q, k, v, scale, dout)
    if not (out.shape == q.shape and out.dtype is q.dtype and out.is_contiguous() and lse.is_contiguous() and
            lse.dtype is torch.float32 and lse.shape == rows):
        raise NextDoorError("packed attention: out and lse are not a forward pass's")
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk, dv = (torch.empty(k.shape, dtype=q.dtype, device=q.device) for _ in range(2))
    a = PackedAttention(*fields, out.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr())
    workspace = _workspace(sequences, a, (q.shape, k.shape, q.dtype), 1, q.device)
    _run(index, _library().nd_packed_attention_backward, a)
    del keep, workspace
    return dq, dk, dv


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, sequences, scale):
        out, lse = packed_attention_forward(q, k, v, sequences, scale)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.how = sequences, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        return (*packed_attention_backward(dout, q, k, v, out, lse, *ctx.how), None, None)


def packed_attention(q, k, v, sequences, scale=None):
    """The ``out`` of :func:`packed_attention_forward`, differentiable in q, k and v."""
    return _PackedAttention.apply(q, k, v, sequences, scale)


# ---- cross entropy over the vocabulary -----------------------------------------------------------------


def _vectors(x):
    if x.shape[1] % 8:  # the kernels read 16 bytes at a time
        x = torch.nn.functional.pad(x, (0, 8 - x.shape[1] % 8))
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


@functools.lru_cache(maxsize=256)
def _loss_workspace(rows, classes, dim, backward):
    return _library().nd_vocabulary_loss_workspace(rows, classes, dim, backward)


def _loss(hidden, weight, target, backward):
    """Checked arguments: (device index, the tensors read, the struct's first fields, workspace, its size)."""
    index = _on_gpu("vocabulary loss", hidden, weight, target)
    dtype = hidden.dtype
    if not (dtype is torch.bfloat16 or dtype is torch.float16):
        raise NextDoorError("vocabulary loss: 16-bit types only, %s given" % dtype)
    if weight.dtype is not dtype:
        raise NextDoorError("vocabulary loss: hidden and weight are of different types")
    if not (hidden.dim() == 2 and weight.dim() == 2 and hidden.shape[1] == weight.shape[1]):
        raise NextDoorError("vocabulary loss: hidden and weight are not matrices of equally long rows")
    hidden, weight = _vectors(hidden), _vectors(weight)
    rows, dim = hidden.shape
    classes = weight.shape[0]
    if not (target.dim() == 1 and target.shape[0] == rows):
        raise NextDoorError("vocabulary loss: one target for each row of hidden")
    if target.dtype not in (torch.int32, torch.int64):
        raise NextDoorError("vocabulary loss: targets are int32 or int64")
    if target.dtype is torch.int64:  # (what is no class stays none: 2^31 - 1 is above every class)
        target = torch.where((target < 0) | (target > 2147483647), 2147483647, target).to(torch.int32)
    target = target.contiguous()
    size = _loss_workspace(rows, classes, dim, backward)
    if size < 0:
        raise NextDoorError("vocabulary loss: no kernel for %d rows, %d classes, vectors of %d" % (rows, classes, dim))
    workspace = torch.empty(max(size, 16), dtype=torch.uint8, device=hidden.device)
    fields = (rows, classes, dim, _DTYPES[dtype], hidden.data_ptr(), weight.data_ptr(), target.data_ptr())
    return index, (hidden, weight, target), fields, workspace, size


def vocabulary_loss_forward(hidden, weight, target):
    """(loss, lse) of each row, float32: ``lse_i = log sum_v exp(hidden_i . weight_v)``, ``loss_i = lse_i - hidden_i .
    weight_{target_i}``.  hidden: [rows, dim], weight: [classes, dim], float16 or bfloat16 (a dim that is no
    multiple of 8 costs a copy); target: int32 or int64.  A row whose target is no class - the samplers' INVALID is
    |V| - has loss 0."""
    index, keep, fields, workspace, size = _loss(hidden, weight, target, 0)
    loss, lse = (torch.empty(fields[0], dtype=torch.float32, device=hidden.device) for _ in range(2))
    _run(index, _library().nd_vocabulary_loss_forward,
         VocabularyLoss(*fields, loss.data_ptr(), lse.data_ptr(), None, None, None, workspace.data_ptr(), size))
    del keep
    return loss, lse


def vocabulary_loss_backward(dloss, hidden, weight, target, lse):
    """(dhidden, dweight) for the gradient ``dloss`` of each row's loss; lse is the forward pass's.  Rows without a
    target send nothing back, whatever their ``dloss``.  bfloat16: ``dloss`` below 2^95."""
    _on_gpu("vocabulary loss", hidden, dloss, lse)
    index, keep, fields, workspace, size = _loss(hidden, weight, target, 1)
    width = hidden.shape[1]
    if tuple(dloss.shape) != fields[:1] or tuple(lse.shape) != fields[:1] or lse.dtype is not torch.float32:
        raise NextDoorError("vocabulary loss: dloss and lse have one value for each row")
    dloss, lse = dloss.to(torch.float32).contiguous(), lse.contiguous()
    dhidden, dweight = torch.empty_like(keep[0]), torch.empty_like(keep[1])
    _run(index, _library().nd_vocabulary_loss_backward,
         VocabularyLoss(*fields, None, lse.data_ptr(), dloss.data_ptr(), dhidden.data_ptr(), dweight.data_ptr(),
                        workspace.data_ptr(), size))
    del keep
    if width != fields[2]:
        dhidden, dweight = dhidden[:, :width].contiguous(), dweight[:, :width].contiguous()
    return dhidden, dweight


class _VocabularyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target):
        loss, lse = vocabulary_loss_forward(hidden, weight, target)
        ctx.save_for_backward(hidden, weight, target, lse)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        return (*vocabulary_loss_backward(dloss, *ctx.saved_tensors), None)


def vocabulary_loss(hidden, weight, target):
    """The loss of each row (:func:`vocabulary_loss_forward`), differentiable in hidden and weight."""
    return _VocabularyLoss.apply(hidden, weight, target)
