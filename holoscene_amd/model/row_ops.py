"""Operators on rows (samples, tokens, frames) beside the fused networks: learned codes looked up by index, a gated feed-forward block and
dropout, each with its backward pass, on the kernels of csrc/embed_rows.hip, csrc/gated_mlp*.hip and csrc/dropout.hip.

    codes = embedding_rows(frame_ids, table)                     # table[frame_ids], gradient by sorted indices
    y = gated_mlp_rows(x, w_gate, w_up, w_down, "silu")          # (silu(x Wg^T) * (x Wu^T)) Wd^T
    y = dropout_rows(y, 0.1, rng, residual=x)                    # x + dropout(y), the mask recomputed from a counter

float32, bfloat16 and float16 storage, fp32 arithmetic, one rounding per result.  As everywhere in this package there is no CPU path: a tensor
that is not on the GPU, or a type or shape the kernels do not take, raises RuntimeError.  The work runs on the current stream of the tensors' device
and can be captured into a HIP graph (with a backward pass: capture before an eager graph of the same leaves is built, or drop it first -- its
gradient accumulators belong to the eager stream); results do not depend on the launch (no floating-point atomics).  Gradients of gradients are not provided.
"""
import contextlib
import math

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from ..hashencoder import backend as _be

ACTIVATIONS = tuple(_be.ROW_ACTIVATIONS)
_INDICES = (torch.int32, torch.int64)


def _check_tensor(t, name, device=None, dtype=None, dtypes=_be.ROW_DTYPES):
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.layout is not torch.strided:
        raise RuntimeError(f"{name} must be a dense tensor")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")
    if dtype is not None and t.dtype is not dtype:
        raise RuntimeError(f"{name} must be a {dtype} tensor, got {t.dtype}")
    if t.dtype not in dtypes:
        raise RuntimeError(f"{name}: unsupported type {t.dtype}")


def _on(t):
    """t's device as the current one while a kernel is launched (a launch goes to the current device, whatever its stream)."""
    return _HERE if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


_HERE = contextlib.nullcontext()


def _recorded(*tensors):
    """Whether autograd will want a backward pass."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _once(backward):
    """once_differentiable, without its guard where gradients are off anyway (every backward pass but create_graph=True; the guard is 5 us of the host)."""
    guarded = once_differentiable(backward)
    return lambda ctx, g: guarded(ctx, g) if torch.is_grad_enabled() else backward(ctx, g)


def _as_rows(t):
    """[..., n] -> 2-D with consecutive elements in a row: the tensor itself (any row distance >= n), else a copy."""
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    if t.is_contiguous():
        return t
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _embed(indices, table, scale, out_dtype):
    out = torch.empty(*indices.shape, table.shape[1], device=table.device, dtype=out_dtype)
    if out.numel():
        with _on(table):
            _be._backend.embed_fwd(indices, _as_rows(table), out, scale)
    return out


class _embedding_rows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, indices, table, scale, padding_idx, out_dtype):
        ctx.save_for_backward(indices)
        ctx.args = (table.shape, table.dtype, scale, -1 if padding_idx is None else padding_idx)
        return _embed(indices, table, scale, out_dtype)

    @staticmethod
    @_once
    def backward(ctx, g):
        indices, = ctx.saved_tensors
        shape, dtype, scale, padding = ctx.args
        g_table = torch.empty(shape, device=g.device, dtype=dtype)
        if g_table.numel():
            with _on(g):
                _be._backend.embed_bwd(indices, _as_rows(g), g_table, scale, padding)
        return None, g_table, None, None, None


def embedding_rows(indices, table, scale=1.0, padding_idx=None, out_dtype=None):
    """scale * table[indices]: indices int32 / int64 of any shape, table [V, D] -> [*indices.shape, D] of `out_dtype` (default: the table's type).

    An index outside [0, V) reads zeros and takes no gradient (as a point outside the hash grid does); row `padding_idx` is read like any other and
    takes no gradient.  The gradient is dense [V, D], summed in fp32 in the order of the positions, the same from run to run."""
    _check_tensor(table, "table")
    _check_tensor(indices, "indices", device=table.device, dtypes=_INDICES)
    if table.dim() != 2:
        raise RuntimeError(f"table must be [V, D], got {tuple(table.shape)}")
    if padding_idx is not None and not 0 <= padding_idx < table.shape[0]:
        raise RuntimeError(f"padding_idx {padding_idx} is outside the table's {table.shape[0]} rows")
    out_dtype = table.dtype if out_dtype is None else out_dtype
    if out_dtype not in _be.ROW_DTYPES:
        raise RuntimeError(f"out_dtype: unsupported type {out_dtype}")
    indices = indices.contiguous()
    if not _recorded(table):
        return _embed(indices, table, float(scale), out_dtype)
    return _embedding_rows.apply(indices, table, float(scale), padding_idx, out_dtype)


def _gated(rows, wg, wu, wd, activation, save):
    """(y, what the backward pass reads) for 2-D rows."""
    y = torch.empty_like(rows, memory_format=torch.contiguous_format)
    with _on(rows):
        return y, _be._backend.gated_mlp_fwd(rows, wg, wu, wd, activation, y, save)


class _gated_mlp_rows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        rows, wg, wu, wd = (_as_rows(t) for t in (x, w_gate, w_up, w_down))
        ctx.activation, ctx.lead = activation, x.shape[:-1]
        ctx.empty = rows.numel() == 0 or wg.numel() == 0
        if ctx.empty:
            ctx.save_for_backward(x, w_gate, w_up, w_down)
            return torch.zeros_like(x)
        y, saved = _gated(rows, wg, wu, wd, activation, True)
        ctx.save_for_backward(rows, wg, wu, wd, saved)
        return y.view(x.shape)

    @staticmethod
    @_once
    def backward(ctx, g):
        if ctx.empty:
            return tuple(torch.zeros_like(t) if need else None for t, need in zip(ctx.saved_tensors, ctx.needs_input_grad)) + (None,)
        rows, wg, wu, wd, saved = ctx.saved_tensors
        gx, ggate, gup, gdown = (torch.empty_like(t, memory_format=torch.contiguous_format) if need else None
                                 for t, need in zip((rows, wg, wu, wd), ctx.needs_input_grad))
        with _on(g):
            _be._backend.gated_mlp_bwd(_as_rows(g), rows, wg, wu, wd, ctx.activation, saved, gx, ggate, gup, gdown)
        return None if gx is None else gx.view(*ctx.lead, rows.shape[1]), ggate, gup, gdown, None


def gated_mlp_rows(x, w_gate, w_up, w_down, activation="silu"):
    """(act(x Wg^T) * (x Wu^T)) Wd^T for x [..., dim], w_gate and w_up [hidden, dim], w_down [dim, hidden], all of one type.

    dim and hidden are at most 2^21.  activation: "silu", "gelu" (g Phi(g)), "gelu_tanh" (its tanh form), "sigmoid", "relu".  float32 operands are multiplied as three bf16 planes each
    (24 bits, as linear_rows under HOLOSCENE_FP32_GEMM=split3; an infinity among them gives NaN).  Rows may be strided; 16-bit operands whose
    rows are not 16-byte aligned are copied once per call.  The forward keeps the gated product for the backward pass, with dim > 768 both projections in fp32 as well."""
    _check_tensor(x, "x")
    if x.dim() < 1:
        raise RuntimeError("x must be [..., dim]")
    device, dtype = x.device, x.dtype
    for t, name in ((w_gate, "w_gate"), (w_up, "w_up"), (w_down, "w_down")):
        _check_tensor(t, name, device, dtype)
        if t.dim() != 2:
            raise RuntimeError(f"{name} must be a matrix, got {tuple(t.shape)}")
    hidden, dim = w_gate.shape
    if x.shape[-1] != dim or w_up.shape != w_gate.shape or w_down.shape != (dim, hidden):
        raise RuntimeError(f"x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)}, w_down {tuple(w_down.shape)}: expected [..., dim], "
                           "[hidden, dim], [hidden, dim], [dim, hidden]")
    if max(hidden, dim) > 1 << 21:
        raise RuntimeError(f"dim {dim} and hidden {hidden} must be at most {1 << 21}")
    if activation not in _be.ROW_ACTIVATIONS:
        raise RuntimeError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    if _recorded(x, w_gate, w_up, w_down):
        return _gated_mlp_rows.apply(x, w_gate, w_up, w_down, activation)
    if x.numel() == 0 or hidden == 0:
        return torch.zeros_like(x)
    y = _gated(_as_rows(x), _as_rows(w_gate), _as_rows(w_up), _as_rows(w_down), activation, False)[0]
    return y if x.dim() == 2 else y.view(x.shape)


def _dropout(x, residual, drop, rng):
    x = x.contiguous()
    y = torch.empty_like(x)
    if y.numel():
        with _on(x):
            _be._backend.dropout_rows(x, None if residual is None else residual.contiguous(), y, drop, rng)
    return y


class _dropout_rows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, drop, rng):
        ctx.save_for_backward(rng)          # (autograd refuses the backward if rng has been written in the meantime)
        ctx.drop = drop
        return _dropout(x, residual, drop, rng)

    @staticmethod
    @_once
    def backward(ctx, g):
        rng, = ctx.saved_tensors
        return _dropout(g, None, ctx.drop, rng) if ctx.needs_input_grad[0] else None, g if ctx.needs_input_grad[1] else None, None, None


def dropout_rows(x, p, rng, residual=None):
    """Zeroes elements of x with probability p, scales the others by 1 / (1 - p), adds `residual` (same shape and type) if given.

    rng: int64 [2] on x's device = (seed, number of the call).  The mask is a function of these two and the element's position in x (row-major,
    whatever the strides) -- Philox-4x32-10, 16 bits an element, so p counts in steps of 2^-16 -- and is never stored: the backward pass computes it again
    from the same rng, which therefore must not be written in between (autograd raises if it is).  Give every call its own number; inside a captured
    graph add to rng[1] after the backward pass, so that each replay draws anew."""
    _check_tensor(x, "x")
    _check_tensor(rng, "rng", device=x.device, dtypes=_INDICES[1:])
    if tuple(rng.shape) != (2,) or not rng.is_contiguous():
        raise RuntimeError("rng must be two consecutive int64 (seed, number of the call)")
    if residual is not None:
        _check_tensor(residual, "residual", device=x.device, dtype=x.dtype)
        if residual.shape != x.shape:
            raise RuntimeError(f"residual {tuple(residual.shape)} must have x's shape {tuple(x.shape)}")
    if not 0.0 <= p <= 1.0:
        raise RuntimeError(f"p must be in [0, 1], got {p}")
    drop = math.floor(p * 65536 + 0.5)
    return _dropout_rows.apply(x, residual, drop, rng) if _recorded(x, residual) else _dropout(x, residual, drop, rng)


class RowEmbedding(nn.Module):
    """A table of `num` learned codes of `dim` elements, looked up by index (embedding_rows)."""

    def __init__(self, num, dim, scale=1.0, padding_idx=None, std=1e-4):
        super().__init__()
        self.scale, self.padding_idx = scale, padding_idx
        self.weight = nn.Parameter(torch.empty(num, dim).normal_(0.0, std))
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx].zero_()

    def forward(self, indices):
        return embedding_rows(indices, self.weight, self.scale, self.padding_idx)


class GatedMLP(nn.Module):
    """The gated feed-forward block (gated_mlp_rows) with its three weights."""

    def __init__(self, dim, hidden, activation="silu"):
        super().__init__()
        if activation not in _be.ROW_ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
        self.activation = activation
        self.w_gate = nn.Parameter(nn.Linear(dim, hidden, bias=False).weight.detach().clone())
        self.w_up = nn.Parameter(nn.Linear(dim, hidden, bias=False).weight.detach().clone())
        self.w_down = nn.Parameter(nn.Linear(hidden, dim, bias=False).weight.detach().clone())

    def forward(self, x):
        return gated_mlp_rows(x, self.w_gate, self.w_up, self.w_down, self.activation)


class RowDropout(nn.Module):
    """Dropout (dropout_rows) with a generator state of its own: a buffer (seed, number of the next call), advanced on the device by every
    call in training mode, so that eager calls and replays of a captured graph alike draw a new mask each time.  A pass that is run twice
    (activation checkpointing) draws twice: call dropout_rows with a state of your own there.  Give every rank its own seed, and keep
    DistributedDataParallel from copying rank 0's buffer (broadcast_buffers=False)."""

    def __init__(self, p, seed=0):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p must be in [0, 1], got {p}")
        self.p = p
        self.register_buffer("rng", torch.tensor([seed, 0], dtype=torch.int64))

    def forward(self, x, residual=None):
        if not self.training or self.p == 0.0:
            return x if residual is None else x + residual
        used = self.rng.clone()
        self.rng[1:].add_(1)
        return dropout_rows(x, self.p, used, residual)
