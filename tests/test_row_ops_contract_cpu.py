"""CPU: what the row operators (model/row_ops.py, include/holoscene_hip.h section 10) refuse before they look at a device."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from holoscene_amd.model import row_ops


def calls(t):
    idx, rng = torch.zeros(3, dtype=torch.long), torch.zeros(2, dtype=torch.long)
    w, d = torch.zeros(5, 4), torch.zeros(4, 5)
    yield lambda: row_ops.embedding_rows(idx, t)
    yield lambda: row_ops.dropout_rows(t, 0.5, rng)
    yield lambda: row_ops.gated_mlp_rows(t, w, w, d)


def test_forward_mode_is_refused():
    """A tangent would be dropped: the value alone came back."""
    x = torch.zeros(3, 4)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="x has a tangent"):
            row_ops.dropout_rows(fwd.make_dual(x, x), 0.5, torch.zeros(2, dtype=torch.long))
        with pytest.raises(RuntimeError, match="table has a tangent"):
            row_ops.embedding_rows(torch.zeros(3, dtype=torch.long), fwd.make_dual(x, x))
        with pytest.raises(RuntimeError, match="x has a tangent"):
            row_ops.gated_mlp_rows(fwd.make_dual(x, x), torch.zeros(5, 4), torch.zeros(5, 4), torch.zeros(4, 5))


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_tracing_is_refused():
    """A trace would hold the result's allocation and not the launch that fills it."""
    x = torch.zeros(3, 4)
    for k in range(3):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(lambda t: list(calls(t))[k](), (x,))
