"""CPU: what the row operators (model/row_ops.py, include/holoscene_hip.h section 10) refuse before they look at a device."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from holoscene_amd.hashencoder import backend
from holoscene_amd.model import row_ops
from test_row_ops_cpu import I64, gated, lib
from test_row_ops_gpu import keep_reference


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


# ------------------------------------------------------------------------------------------------ sizes, from C
def test_work_space_queries_refuse_empty_blocks():
    """Without rows, columns or hidden elements there is no product to plan (the plan divided by the number of its tiles: SIGFPE)."""
    for dtype in (0, 1, 2):
        for bad in (dict(rows=0), dict(dim=0), dict(hidden=0), dict(rows=100, dim=0), dict(rows=100, hidden=0), dict(rows=0, dim=0, hidden=0)):
            args = gated(dtype=dtype, gx=256, gw_gate=256, gw_up=256, gw_down=256, **bad)
            assert lib().hs_gated_mlp_fwd_ws_bytes(args) == -1 and lib().hs_gated_mlp_bwd_ws_bytes(args) == -1, (dtype, bad)
            assert lib().hs_gated_mlp_saved_bytes(args) == -1, (dtype, bad)


def test_lookup_work_space_of_an_empty_table():
    """A table without rows takes no pass of the sort (which the plan divided by: SIGFPE); its gradient needs nothing."""
    f = lib().hs_embed_bwd_ws_bytes
    for n in (0, 1, 5000, 1 << 20):
        assert f(I64(n), I64(0), I64(16)) == 0 and f(I64(n), I64(5), I64(0)) == 0
    assert f(I64(0), I64(5), I64(16)) >= 8


def test_most_rows_of_a_block():
    """The weight gradients contract over the rows, in steps of 64 counted in 32 bits: the last step must end below 2^31."""
    most = (1 << 31) - 128
    for dtype in (0, 1, 2):
        for f in (lib().hs_gated_mlp_saved_bytes, lib().hs_gated_mlp_fwd_ws_bytes, lib().hs_gated_mlp_bwd_ws_bytes):
            assert f(gated(rows=most, dtype=dtype, gw_down=256)) >= 0
            assert all(f(gated(rows=rows, dtype=dtype, gw_down=256)) == -1 for rows in (most + 1, (1 << 31) - 63, (1 << 31) - 1, 1 << 31))
        for f in (lib().hs_gated_mlp_fwd, lib().hs_gated_mlp_bwd):
            assert all(f(gated(rows=rows, dtype=dtype, gw_down=256, ws_bytes=1 << 62), None) == -1 for rows in (most + 1, (1 << 31) - 63, (1 << 31) - 1, 1 << 31))


# ------------------------------------------------------------------------------------------------ planes
def test_planes_refusals_and_sizes():
    one, two = 0x100, 0x200
    f = lib().hs_gated_mlp_saved_bytes
    for act in range(5):
        assert f(gated(activation=act | one)) < f(gated(activation=act | two)) == f(gated(activation=act))        # (4 x 16: few results)
        wide = dict(rows=500, dim=16, hidden=32)
        big = dict(rows=5000, dim=256, ldx=256, ld_gate=256, ld_up=256)
        assert f(gated(activation=act | one, **wide)) < f(gated(activation=act | two, **wide))
        assert f(gated(activation=act | one, **big)) == f(gated(activation=act, **big)) < f(gated(activation=act | two, **big))
    for bad in (5, 5 | one, one | two, 0x400, 0x10000 | one, -1):
        assert f(gated(activation=bad)) == -1 and lib().hs_gated_mlp_fwd(gated(activation=bad), None) == -1 and lib().hs_gated_mlp_bwd(gated(activation=bad), None) == -1
    assert f(gated(activation=one, dtype=0)) == -1 and f(gated(activation=two, dtype=0)) == -1        # (fp32: always three)
    t = torch.zeros(4, 8)
    for planes in (0, 3, "two"):
        with pytest.raises(RuntimeError, match="planes must be"):
            row_ops.gated_mlp_rows(t, t, t, t.t(), planes=planes)
        with pytest.raises(ValueError, match="planes must be"):
            row_ops.GatedMLP(8, 16, planes=planes)


# ------------------------------------------------------------------------------------------------ the two libraries
def test_nodes_are_bound_to_their_own_abi_only():
    nodes = backend.row_autograd()
    assert lib().hs_abi_version() == backend.ABI_VERSION
    for version in (backend.ABI_VERSION - 1, backend.ABI_VERSION + 1):
        with pytest.raises(RuntimeError, match="ABI version"):
            nodes.bind({}, version)


# ------------------------------------------------------------------------------------------------ the oracles of the GPU tests
def test_philox_known_answer_through_the_oracle():
    """The published vector of Philox-4x32-10 (counter and key all ones -> 408f276d 41c83b0e a20bc7c6 6d5451fd) read out of keep_reference, which the kernel is
    compared with: element e is kept at drop = u_e and not at u_e + 1."""
    ones = (1 << 64) - 1
    words = [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    halves = [h for w in words for h in (w & 0xffff, w >> 16)]
    for e, u in enumerate(halves):
        assert bool(keep_reference(8, u, ones, ones, first=ones)[e]) and not bool(keep_reference(8, u + 1, ones, ones, first=ones)[e])
