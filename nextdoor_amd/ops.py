"""Operators of models that train on samples, on torch tensors of the GPU.

Walks are sequences of different lengths whose words are the vertices of the graph.  A training step
over a batch of them needs

* :func:`packed_attention`: causal attention within each walk of a packed batch, with grouped heads;
* :func:`dropout`: from the samplers' own random stream, the mask never stored;
* :func:`vocabulary_loss`: softmax cross entropy over all vertices, the logits never stored;
* :func:`layer_norm`: of each row, with the gradients of its weight and bias;
* :func:`linear`: a matrix product with bias, activation and residual in one kernel;
* :func:`mlp`: the feed-forward part of a block, gated or not.

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
from torch.autograd import forward_ad

from . import _capi
from ._capi import LayerNorm, Linear, Mlp, NextDoorError, PackedAttention, VocabularyLoss, check

__all__ = ["PackedSequences", "packed_attention", "packed_attention_forward", "packed_attention_backward",
           "vocabulary_loss", "vocabulary_loss_forward", "vocabulary_loss_backward", "dropout", "dropout_forward",
           "dropout_backward", "layer_norm", "layer_norm_forward", "layer_norm_backward", "linear", "linear_forward",
           "linear_backward", "mlp", "mlp_forward", "mlp_backward", "NextDoorError"]

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
_current_device = torch._C._cuda_getDevice  # torch.cuda.current_device without the check for a first use: there is a tensor


def _run(index, fn, *args):
    """Calls an entry point that takes a stream last, on torch's current one, with the device current."""
    if _current_device() == index:
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


# ---- layer norm ------------------------------------------------------------------------------------------


def _rows_in_place(x, dim, multiple):
    """x as [rows, dim] and the elements between its rows, a multiple of ``multiple``.  What cannot be read so is copied."""
    x = x.reshape(-1, dim) if x.dim() != 2 else x
    rows, step = x.shape[0], x.stride(0)
    if rows <= 1 or dim == 0:
        step = dim + -dim % multiple  # (never used, but torch keeps one)
    if (x.stride(1) != 1 and dim > 1) or step % multiple or step > 4194304 or (multiple > 1 and x.data_ptr() % 16):
        x = torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x)
        step = dim
    return x, step


def _norm(x, weight, bias, eps, *others):
    """Checked arguments: (device index, x as rows, the struct's first fields, weight, bias)."""
    given = [x, *others]
    if weight is not None:
        given.append(weight)
    if bias is not None:
        given.append(bias)
    index = _on_gpu("layer norm", *given)
    dtype = x.dtype
    code = _DTYPES.get(dtype)
    if code is None:
        raise NextDoorError("layer norm: no kernel for %s" % dtype)
    if x.dim() == 0:
        raise NextDoorError("layer norm: x has no rows")
    dim = x.shape[-1]
    weight_dtype = dtype
    for t in given[1 + len(others):]:
        if t.shape != (dim,):
            raise NextDoorError("layer norm: weight or bias is not [%d]" % dim)
        weight_dtype = t.dtype
        if weight_dtype is not dtype and weight_dtype is not torch.float32:
            raise NextDoorError("layer norm: weight or bias is neither of the type of x nor float32")
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise NextDoorError("layer norm: weight and bias are of different types")
    if not 0.0 <= eps < math.inf:
        raise NextDoorError("layer norm: eps is a number of at least 0, %r given" % (eps,))
    if not 1 <= dim <= 16384:
        raise NextDoorError("layer norm: rows of 1 to 16384 values, %d given" % dim)
    x, x_row = _rows_in_place(x, dim, 1)
    weight, bias = None if weight is None else weight.contiguous(), None if bias is None else bias.contiguous()
    return index, x, (x.shape[0], dim, code, _DTYPES[weight_dtype], eps), x_row, weight, bias


def _pointer(t):
    return None if t is None else t.data_ptr()


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5):
    """(out, mean, rstd): each row of x (its last dimension, up to 16384 values) less its mean, over its standard deviation
    (``rstd = 1 / sqrt(variance + eps)``), times weight (1 unless given), plus bias (0).  float32, float16 or bfloat16; weight and bias
    of that type or float32.  mean and rstd: [rows], float32, for the backward pass.  Sums are in 32 bits, results rounded
    once."""
    index, rows, fields, x_row, weight, bias = _norm(x, weight, bias, eps)
    device = x.device
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean, rstd = torch.empty(fields[0], dtype=torch.float32, device=device), torch.empty(fields[0], dtype=torch.float32, device=device)
    _run(index, _library().nd_layer_norm_forward,
         LayerNorm(*fields, x_row, 0, rows.data_ptr(), _pointer(weight), _pointer(bias), out.data_ptr(), mean.data_ptr(), rstd.data_ptr()))
    return out, mean, rstd


def layer_norm_backward(dout, x, weight, mean, rstd, needs=(True, True, True), dtype=None):
    """(dx, dweight, dbias) for the gradient ``dout`` of ``out``; mean and rstd are the forward pass's, ``weight`` None if there was
    none.  dweight and dbias are of the type of weight; without one of ``dtype``, that of x or float32, by default that of x.
    ``needs``: which to compute; the others are None."""
    index, rows, fields, x_row, weight, _ = _norm(x, weight, None, 0.0, dout, mean, rstd)
    if weight is None and dtype is not None:
        if dtype is not x.dtype and dtype is not torch.float32:
            raise NextDoorError("layer norm: gradients of the type of x or float32, not %s" % dtype)
        fields = (*fields[:3], _DTYPES[dtype], fields[4])
    if dout.shape != x.shape or dout.dtype is not x.dtype:
        raise NextDoorError("layer norm: dout is of another shape or type than x")
    if not (mean.shape == rstd.shape == (fields[0],) and mean.dtype is rstd.dtype is torch.float32 and
            mean.is_contiguous() and rstd.is_contiguous()):
        raise NextDoorError("layer norm: mean and rstd are not a forward pass's")
    dout, dout_row = _rows_in_place(dout, fields[1], 1)
    kind = weight.dtype if weight is not None else x.dtype if dtype is None else dtype
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if needs[0] else None
    dweight = mean.new_empty(fields[1], dtype=kind) if needs[1] else None
    dbias = mean.new_empty(fields[1], dtype=kind) if needs[2] else None
    a = LayerNorm(*fields, x_row, dout_row, rows.data_ptr(), _pointer(weight), None, None, mean.data_ptr(), rstd.data_ptr(),
                  dout.data_ptr(), _pointer(dx), _pointer(dweight), _pointer(dbias))
    workspace = _room(a, _library().nd_layer_norm_workspace(a), mean.device) if needs[1] or needs[2] else None
    _run(index, _library().nd_layer_norm_backward, a)
    del workspace
    return dx, dweight, dbias


def _room(a, size, device):
    """A workspace of the size that a call needs, if any (a call that no kernel can do has none: the call says why)."""
    if size <= 0:
        return None
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), size
    return workspace


def _nothing_to_derive():
    """Whether a call may pass autograd by, which costs some 5 us: gradients are off, and so is forward mode, which no_grad
    leaves on and which has to see the call to refuse it."""
    return not torch.is_grad_enabled() and forward_ad._current_level < 0


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        out, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        x, weight, mean, rstd = ctx.saved_tensors
        return (*layer_norm_backward(dout, x, weight, mean, rstd, ctx.needs_input_grad[:3], ctx.bias_dtype), None)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """The ``out`` of :func:`layer_norm_forward`, differentiable in x, weight and bias."""
    if _nothing_to_derive():
        return layer_norm_forward(x, weight, bias, eps)[0]
    return _LayerNorm.apply(x, weight, bias, eps)


# ---- linear maps -------------------------------------------------------------------------------------------

_ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}  # ND_NO_ACTIVATION ...


def _activation(what, name):
    try:
        return _ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise NextDoorError("%s: no activation %r; there are None, %s" % (what, name, ", ".join(sorted(filter(None, _ACTIVATIONS))))) from None


def _types(what, first, *others):
    dtype = first.dtype
    if not (dtype is torch.bfloat16 or dtype is torch.float16):
        raise NextDoorError("%s: 16-bit types only, %s given" % (what, dtype))
    for t in others:
        if t is not None and t.dtype is not dtype:
            raise NextDoorError("%s: tensors of different types" % what)


def _matrix(t):
    """A weight or a bias as the kernels read it; a last dimension that is no multiple of 8, or a matrix's first, is
    filled up with zeros, which costs a copy."""
    if t is None:
        return None
    if any([size % 8 for size in t.shape]):
        t = torch.nn.functional.pad(t, [n for size in reversed(t.shape) for n in (0, -size % 8)])
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _vectors_in_place(x, dim):
    """x as [rows, a multiple of 8], filled up with zeros if need be, and the elements between its rows."""
    if dim % 8:
        x = torch.nn.functional.pad(x.reshape(-1, dim), (0, -dim % 8))
    return _rows_in_place(x, dim + -dim % 8, 8)


def _check_rows(what, name, t, shape, dtype):
    if t.shape != shape or t.dtype is not dtype:
        raise NextDoorError("%s: %s is of another shape or type than the result" % (what, name))


def _result(x, wanted, *shape):
    """Room for a result that the kernels write as a matrix or vector of `shape`, in the shape that is wanted where both are the same."""
    return x.new_empty(wanted if wanted[-1] == shape[-1] else shape)


def _cut(t, *shape):
    """The part of a filled-up result that was asked for."""
    if t is None or t.shape == shape:
        return t
    for i, n in enumerate(shape):
        t = t.narrow(i, 0, n)
    return t.contiguous()


def _shaped(t, rows, dim, wanted):
    """The rows of a result of :func:`_result` as the caller wants them."""
    return t if t is None or t.shape == wanted else _cut(t, rows, dim).view(wanted)


def _linear_arguments(what, x, weight, bias):
    if not (x.dim() >= 1 and weight.dim() == 2 and x.shape[-1] == weight.shape[1]):
        raise NextDoorError("%s: x and weight are not vectors and a matrix of equally long rows" % what)
    out_dim, dim = weight.shape
    if bias is not None and bias.shape != (out_dim,):
        raise NextDoorError("%s: a bias is not [%d]" % (what, out_dim))
    if not (1 <= dim <= 1048576 and 1 <= out_dim <= 1048576):
        raise NextDoorError("%s: vectors of 1 to 1048576 places, %d and %d given" % (what, dim, out_dim))
    return out_dim, dim


def linear_forward(x, weight, bias=None, activation=None, residual=None, keep=False):
    """``activation(x weight^T + bias) + residual``, or with ``keep`` (out, z), z being what the backward pass reads (None without an
    activation).

    x: [..., dim], weight: [out_dim, dim], bias: [out_dim], residual: [..., out_dim], float16 or bfloat16; activation: None,
    "relu", "gelu", "gelu_tanh" or "silu".  Slices whose rows begin at multiples of 16 bytes are read in place; dims that are no
    multiples of 8 cost copies.  Sums are in 32 bits; the result, and z, are rounded once."""
    index = _on_gpu("linear", x, weight, *(t for t in (bias, residual) if t is not None))
    _types("linear", x, weight, bias, residual)
    code = _activation("linear", activation)
    out_dim, dim = _linear_arguments("linear", x, weight, bias)
    shape = (*x.shape[:-1], out_dim)
    wide = out_dim + -out_dim % 8
    rows, x_row = _vectors_in_place(x, dim)
    residual_row = 0
    if residual is not None:
        _check_rows("linear", "the residual", residual, shape, x.dtype)
        residual, residual_row = _vectors_in_place(residual, out_dim)
    weight, bias = _matrix(weight), _matrix(bias)
    n = rows.shape[0]
    out = _result(x, shape, n, wide)
    z = x.new_empty((n, wide)) if keep and code else None
    a = Linear(n, weight.shape[1], wide, _DTYPES[x.dtype], code, x_row, residual_row, 0, rows.data_ptr(), weight.data_ptr(), _pointer(bias),
               _pointer(residual), out.data_ptr(), _pointer(z))
    workspace = _room(a, _library().nd_linear_workspace(a, 0), x.device)
    _run(index, _library().nd_linear_forward, a)
    del workspace
    if z is not None and wide > out_dim:
        z[:, out_dim:].zero_()  # (0 times a place of x that is not finite)
    out = _shaped(out, n, out_dim, shape)
    return (out, z) if keep else out


def linear_backward(dout, x, weight, z=None, activation=None, with_bias=True, needs=(True, True)):
    """(dx, dweight, dbias) for the gradient ``dout`` of ``out``; z is what the forward pass kept.  The residual's gradient is
    ``dout`` itself.  ``needs``: whether dx and dweight are wanted; what is not is None.  With an activation the gradient of z is
    rounded to 16 bits before its products (float16: held times a power of two, so that small ones are not lost)."""
    index = _on_gpu("linear", x, dout, weight, *(() if z is None else (z,)))
    _types("linear", x, dout, weight, z)
    code = _activation("linear", activation)
    out_dim, dim = _linear_arguments("linear", x, weight, None)
    _check_rows("linear", "dout", dout, (*x.shape[:-1], out_dim), x.dtype)
    rows, x_row = _vectors_in_place(x, dim)
    dout, dout_row = _vectors_in_place(dout, out_dim)
    weight = _matrix(weight)
    n, wide, high = rows.shape[0], out_dim + -out_dim % 8, dim + -dim % 8
    if code and not (z is not None and z.shape == (n, wide) and z.is_contiguous()):
        raise NextDoorError("linear: z is not what a forward pass kept")
    dx = _result(x, x.shape, n, high) if needs[0] else None
    dweight = torch.empty_like(weight) if needs[1] else None
    dbias = x.new_empty(wide) if with_bias else None
    a = Linear(n, high, wide, _DTYPES[x.dtype], code, x_row, 0, dout_row, rows.data_ptr(), weight.data_ptr(), None, None, None,
               _pointer(z) if code else None, dout.data_ptr(), _pointer(dx), _pointer(dweight), _pointer(dbias))
    workspace = _room(a, _library().nd_linear_workspace(a, 1), x.device)
    _run(index, _library().nd_linear_backward, a)
    del workspace
    return _shaped(dx, n, dim, x.shape), _cut(dweight, out_dim, dim), _cut(dbias, out_dim)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        keep = activation is not None and any(ctx.needs_input_grad[:3])
        out = linear_forward(x, weight, bias, activation, residual, keep)
        out, z = out if keep else (out, None)
        ctx.save_for_backward(x, weight, z)
        ctx.activation = activation
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        x, weight, z = ctx.saved_tensors
        needs = ctx.needs_input_grad
        got = (None, None, None)
        if any(needs[:3]):
            got = linear_backward(dout, x, weight, z, ctx.activation, needs[2], needs[:2])
        return (*got, dout if needs[3] else None, None)


def linear(x, weight, bias=None, activation=None, residual=None):
    """:func:`linear_forward`, differentiable in x, weight, bias and the residual."""
    if _nothing_to_derive():  # (nothing is kept)
        return linear_forward(x, weight, bias, activation, residual)
    return _Linear.apply(x, weight, bias, residual, activation)


# ---- feed-forward parts ------------------------------------------------------------------------------------


def _mlp_arguments(x, up, down, up_bias, down_bias, activation, gated):
    if not (down.dim() == 2 and up.dim() == 2):
        raise NextDoorError("mlp: up and down are matrices")
    inner = down.shape[1]
    if up.shape[0] != (2 * inner if gated else inner):
        raise NextDoorError("mlp: up has %d rows, down has rows of %d: %s" %
                            (up.shape[0], inner, "a gated part has twice as many" if gated else "they are as many"))
    wide, dim = _linear_arguments("mlp", x, up, up_bias)
    if down_bias is not None and down_bias.shape != (down.shape[0],):
        raise NextDoorError("mlp: a bias is not [%d]" % down.shape[0])
    if not 1 <= down.shape[0] <= 1048576:
        raise NextDoorError("mlp: vectors of 1 to 1048576 places, %d given" % down.shape[0])
    return dim, inner, down.shape[0], _activation("mlp", activation)


def _up(t, inner, gated):
    """The rows of both projections, each filled up to a multiple of 8."""
    if t is None or not gated or inner % 8 == 0:
        return _matrix(t)
    halves = [torch.nn.functional.pad(half, (0, 0) * (t.dim() - 1) + (0, -inner % 8)) for half in t.split(inner)]
    return _matrix(torch.cat(halves))


def _up_cut(t, inner, gated, *rest):
    """The gradient of up or its bias without what was filled up."""
    if t is None or not gated or inner % 8 == 0:
        return _cut(t, inner * (2 if gated else 1), *rest)
    return torch.cat([_cut(half, inner, *rest) for half in t.split(t.shape[0] // 2)])


def mlp_forward(x, up, down, up_bias=None, down_bias=None, activation="silu", gated=True, residual=None, keep=False):
    """The feed-forward part of a block: ``h down^T + down_bias + residual``, or with ``keep`` (out, z, h), which the backward
    pass reads (z of a gated part holds 24 bits of each value, as bytes).

    z = x up^T + up_bias; gated: ``h = activation(g) u`` with ``g, u = z.chunk(2, -1)``, else ``h = activation(z)``.  x: [..., dim];
    up: [2 inner or inner, dim]; down: [out_dim, inner]; activations, types and sizes as in :func:`linear_forward`.  Both
    projections, the activation and the product are one kernel (and one more where few rows share out the sums); h is rounded to 16 bits
    before the second, which makes an infinity of what is 65520 or more in float16."""
    index = _on_gpu("mlp", x, up, down, *(t for t in (up_bias, down_bias, residual) if t is not None))
    _types("mlp", x, up, down, up_bias, down_bias, residual)
    gated = bool(gated)
    dim, inner, out_dim, code = _mlp_arguments(x, up, down, up_bias, down_bias, activation, gated)
    shape = (*x.shape[:-1], out_dim)
    rows, x_row = _vectors_in_place(x, dim)
    residual_row = 0
    if residual is not None:
        _check_rows("mlp", "the residual", residual, shape, x.dtype)
        residual, residual_row = _vectors_in_place(residual, out_dim)
    up, up_bias, down, down_bias = _up(up, inner, gated), _up(up_bias, inner, gated), _matrix(down), _matrix(down_bias)
    n, wide = rows.shape[0], down.shape[0]

    out, h = _result(x, shape, n, wide), x.new_empty((n, down.shape[1]))
    z = None
    if keep and gated:
        z = torch.empty((n, 3 * up.shape[0]), dtype=torch.uint8, device=x.device)
    elif keep and code:
        z = x.new_empty((n, up.shape[0]))
    a = Mlp(n, up.shape[1], down.shape[1], wide, _DTYPES[x.dtype], code, gated, x_row, residual_row, 0, rows.data_ptr(), up.data_ptr(),
            _pointer(up_bias), down.data_ptr(), _pointer(down_bias), _pointer(residual), out.data_ptr(), _pointer(z), h.data_ptr())
    a.inner_filled = down.shape[1] - inner
    workspace = _room(a, _library().nd_mlp_workspace(a, 0), x.device)
    _run(index, _library().nd_mlp_forward, a)
    del workspace
    out = _shaped(out, n, out_dim, shape)
    return (out, z, h) if keep else out


def mlp_backward(dout, x, up, down, z, h, activation="silu", gated=True, with_up_bias=True, with_down_bias=True,
                 needs=(True, True, True)):
    """(dx, dup, ddown, dup_bias, ddown_bias) for the gradient ``dout`` of ``out``; z and h are what the forward pass kept.  The
    residual's gradient is ``dout`` itself.  ``needs``: whether dx, dup and ddown are wanted; what is not is None (ddown alone reads h, dx,
    dup and dup_bias read z: what nothing reads may be None).  The gradient of z
    is rounded to 16 bits before its products (float16: held times a power of two, so that small ones are not lost, and large ones do
    not become infinite)."""
    index = _on_gpu("mlp", x, dout, up, down, *(t for t in (z, h) if t is not None))
    _types("mlp", x, dout, up, down, h)
    gated = bool(gated)
    dim, inner, out_dim, code = _mlp_arguments(x, up, down, None, None, activation, gated)
    _check_rows("mlp", "dout", dout, (*x.shape[:-1], out_dim), x.dtype)
    rows, x_row = _vectors_in_place(x, dim)
    dout, dout_row = _vectors_in_place(dout, out_dim)
    up, down = _up(up, inner, gated), _matrix(down)
    n = rows.shape[0]
    if needs[2] if h is None else not (h.shape == (n, down.shape[1]) and h.is_contiguous()):
        raise NextDoorError("mlp: h is not what a forward pass kept")
    if gated or code:
        kept = ((n, 3 * up.shape[0]), torch.uint8) if gated else ((n, up.shape[0]), x.dtype)
        if needs[0] or needs[1] or with_up_bias if z is None else (z.shape, z.dtype) != kept or not z.is_contiguous():
            raise NextDoorError("mlp: z is not what a forward pass kept")

    dx = _result(x, x.shape, n, up.shape[1]) if needs[0] else None
    dup, ddown = torch.empty_like(up) if needs[1] else None, torch.empty_like(down) if needs[2] else None
    dup_bias, ddown_bias = x.new_empty(up.shape[0]) if with_up_bias else None, x.new_empty(down.shape[0]) if with_down_bias else None
    a = Mlp(n, up.shape[1], down.shape[1], down.shape[0], _DTYPES[x.dtype], code, gated, x_row, 0, dout_row, rows.data_ptr(), up.data_ptr(),
            None, down.data_ptr(), None, None, None, _pointer(z), _pointer(h), dout.data_ptr(), _pointer(dx), _pointer(dup),
            _pointer(dup_bias), _pointer(ddown), _pointer(ddown_bias))
    a.inner_filled = down.shape[1] - inner
    workspace = _room(a, _library().nd_mlp_workspace(a, 1), x.device)
    _run(index, _library().nd_mlp_backward, a)
    del workspace
    return (_shaped(dx, n, dim, x.shape), _up_cut(dup, inner, gated, dim), _cut(ddown, out_dim, inner), _up_cut(dup_bias, inner, gated),
            _cut(ddown_bias, out_dim))


class _Mlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, up, down, up_bias, down_bias, activation, gated, residual):
        needs = ctx.needs_input_grad
        first = needs[0] or needs[1] or needs[3]  # (what of z and h no gradient reads is not kept)
        keep = first or needs[2]
        got = mlp_forward(x, up, down, up_bias, down_bias, activation, gated, residual, keep)
        out, z, h = got if keep else (got, None, None)
        ctx.save_for_backward(x, up, down, z if first else None, h if needs[2] else None)
        ctx.how = activation, gated
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        x, up, down, z, h = ctx.saved_tensors
        needs = ctx.needs_input_grad
        got = (None,) * 5
        if any(needs[:5]):
            got = mlp_backward(dout, x, up, down, z, h, *ctx.how, needs[3], needs[4], needs[:3])
        return (*got, None, None, dout if needs[7] else None)


def mlp(x, up, down, up_bias=None, down_bias=None, activation="silu", gated=True, residual=None):
    """:func:`mlp_forward`, differentiable in x, the weights, the biases and the residual."""
    if _nothing_to_derive():
        return mlp_forward(x, up, down, up_bias, down_bias, activation, gated, residual)
    return _Mlp.apply(x, up, down, up_bias, down_bias, activation, gated, residual)
