"""Operators on rows (samples, tokens, frames) beside the fused networks: learned codes looked up by index, a gated feed-forward block and
dropout, each with its backward pass, on the kernels of csrc/embed_rows.hip, csrc/gated_mlp*.hip and csrc/dropout.hip.

    codes = embedding_rows(frame_ids, table)                     # table[frame_ids], gradient by sorted indices
    y = gated_mlp_rows(x, w_gate, w_up, w_down, "silu")          # (silu(x Wg^T) * (x Wu^T)) Wd^T
    y = dropout_rows(y, 0.1, rng, residual=x)                    # x + dropout(y), the mask recomputed from a counter

float32, bfloat16 and float16 storage, fp32 arithmetic, one rounding per result.  As everywhere in this package there is no CPU path: a tensor
that is not on the GPU, or a type or shape the kernels do not take, raises RuntimeError.  The work runs on the current stream of the tensors' device
and can be captured into a HIP graph (with a backward pass: capture before an eager graph of the same leaves is built, or drop it first -- its
gradient accumulators belong to the eager stream); results do not depend on the launch (no floating-point atomics).

Gradients of gradients are not provided: with create_graph=True the gradients come back, and a backward pass that reaches them raises RuntimeError.  Those of
embedding_rows and dropout_rows, linear operators, depend on the incoming gradient only; where that is a constant, so are they.  A tensor with a
tangent (forward mode) and a call under torch.jit.trace are refused.
"""
import torch
import torch.nn as nn

from ..hashencoder import backend as _be

ACTIVATIONS = tuple(_be.ROW_ACTIVATIONS)


def _check_tensor(t, name):
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor")


def embedding_rows(indices, table, scale=1.0, padding_idx=None, out_dtype=None):
    """scale * table[indices]: indices int32 / int64 of any shape, table [V, D] -> [*indices.shape, D] of `out_dtype` (default: the table's type).

    An index outside [0, V) reads zeros and takes no gradient (as a point outside the hash grid does); row `padding_idx` is read like any other and
    takes no gradient.  The gradient is dense [V, D], summed in fp32 in the order of the positions, the same from run to run."""
    _check_tensor(indices, "indices")
    _check_tensor(table, "table")
    return _be.row_autograd().embedding_rows(indices, table, scale, padding_idx, out_dtype)


def gated_mlp_rows(x, w_gate, w_up, w_down, activation="silu", planes=None):
    """(act(x Wg^T) * (x Wu^T)) Wd^T for x [..., dim], w_gate and w_up [hidden, dim], w_down [dim, hidden], all of one type.

    dim and hidden are at most 2^21.  activation: "silu", "gelu" (g Phi(g)), "gelu_tanh" (its tanh form), "sigmoid", "relu".  float32 operands are
    multiplied as three bf16 planes each (24 bits, as linear_rows under HOLOSCENE_FP32_GEMM=split3; an infinity among them gives NaN).  Rows may be
    strided; 16-bit operands whose rows are not 16-byte aligned are copied once per call.  The forward keeps the gated product for the backward pass, and both
    projections in fp32 where reading them back costs less than computing them again (dim > 768, in float32 > 128).  The gated product and its two
    gradients are rounded to x's type between the products: in float16 they are infinite beyond 65 504, and less than 3e-8 is zero.

    planes (bfloat16 and float16): in how many values of the type each element of these three is held -- 1: results are 1.4 times as far from exact as their own
    rounding takes them; 2: no further than that, for up to twice the time; None: 2 where results are few (min(rows, hidden) dim <= 2 048), else 1.  float32
    always holds them in its three planes."""
    for t, name in ((x, "x"), (w_gate, "w_gate"), (w_up, "w_up"), (w_down, "w_down")):
        _check_tensor(t, name)
    if activation not in _be.ROW_ACTIVATIONS:
        raise RuntimeError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    if planes not in _be.ROW_PLANES:
        raise RuntimeError(f"planes must be None, 1 or 2, got {planes!r}")
    return _be.row_autograd().gated_mlp_rows(x, w_gate, w_up, w_down, _be.ROW_ACTIVATIONS[activation] | _be.ROW_PLANES[planes])


def dropout_rows(x, p, rng, residual=None):
    """Zeroes elements of x with probability p, scales the others by 1 / (1 - p), adds `residual` (same shape and type) if given.

    rng: int64 [2] on x's device = (seed, number of the call).  The mask is a function of these two and the element's position in x (row-major,
    whatever the strides) -- Philox-4x32-10, 16 bits an element, so p counts in steps of 2^-16 -- and is never stored: the backward pass computes it again
    from the same rng, which therefore must not be written in between (autograd raises if it is).  Give every call its own number; inside a captured
    graph add to rng[1] after the backward pass, so that each replay draws anew."""
    _check_tensor(x, "x")
    _check_tensor(rng, "rng")
    if residual is not None:
        _check_tensor(residual, "residual")
    return _be.row_autograd().dropout_rows(x, p, rng, residual)


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

    def __init__(self, dim, hidden, activation="silu", planes=None):
        super().__init__()
        if planes not in _be.ROW_PLANES:
            raise ValueError(f"planes must be None, 1 or 2, got {planes!r}")
        if activation not in _be.ROW_ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
        self.activation, self.planes = activation, planes
        self.w_gate = nn.Parameter(nn.Linear(dim, hidden, bias=False).weight.detach().clone())
        self.w_up = nn.Parameter(nn.Linear(dim, hidden, bias=False).weight.detach().clone())
        self.w_down = nn.Parameter(nn.Linear(hidden, dim, bias=False).weight.detach().clone())

    def forward(self, x):
        return gated_mlp_rows(x, self.w_gate, self.w_up, self.w_down, self.activation, self.planes)


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
