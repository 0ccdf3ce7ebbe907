"""CPU: refusals of the row operators (include/holoscene_hip.h section 10, model/row_ops.py) -- error codes come before any launch, a tensor that is
not on the GPU raises -- and the sizes of their work spaces."""
import ctypes

import pytest
import torch

from holoscene_amd.hashencoder import backend
from holoscene_amd.model import row_ops

ONE = ctypes.c_void_p(256)          # never dereferenced on these paths
I64 = ctypes.c_int64
F = ctypes.c_float


def lib():
    return backend.load_library()


def embed_fwd(idx=ONE, ib=8, table=ONE, ld=16, out=ONE, n=4, V=10, D=16, td=0, od=0):
    return lib().hs_embed_fwd(idx, ib, table, I64(ld), out, I64(n), I64(V), I64(D), F(1.0), td, od, None)


def embed_bwd(idx=ONE, ib=8, grad=ONE, ld=16, gt=ONE, n=4, V=10, D=16, gd=0, td=0, ws=ONE, nbytes=1 << 20):
    return lib().hs_embed_bwd(idx, ib, grad, I64(ld), gt, I64(n), I64(V), I64(D), F(1.0), I64(-1), gd, td, ws, I64(nbytes), None)


def test_embed_refusals():
    assert embed_fwd(n=0) == 0 and embed_fwd(D=0) == 0                       # nothing to do: no launch
    assert embed_fwd(ib=2) == -1 and embed_fwd(td=3) == -1 and embed_fwd(od=-1) == -1 and embed_fwd(ld=15) == -1 and embed_fwd(n=-1) == -1
    assert embed_fwd(n=1 << 31) == -1 and embed_fwd(V=0x7fffffff) == -1 and embed_fwd(D=(1 << 20) + 1, ld=1 << 21) == -1
    assert embed_fwd(idx=None) == -3 and embed_fwd(out=None) == -3 and embed_fwd(table=None) == -3
    assert embed_bwd(V=0) == 0 and embed_bwd(D=0) == 0
    assert embed_bwd(ib=1) == -1 and embed_bwd(gd=7) == -1 and embed_bwd(td=7) == -1 and embed_bwd(ld=3) == -1
    assert embed_bwd(gt=None) == -3 and embed_bwd(grad=None) == -3 and embed_bwd(ws=None) == -3
    assert embed_bwd(nbytes=lib().hs_embed_bwd_ws_bytes(I64(4), I64(10), I64(16)) - 1) == -1


def test_embed_work_space_grows_with_its_parts():
    f = lib().hs_embed_bwd_ws_bytes
    assert f(I64(-1), I64(1), I64(1)) == -1
    assert f(I64(1), I64(1), I64(1)) >= 8
    for n, V, D in ((4096, 50021, 2048), (4097, 100, 7), (131072, 1024, 32), (1 << 20, 1 << 22, 64)):
        multi = n > 4096
        passes = 1 if V < 1 << 11 else -(-V.bit_length() // 9)
        assert f(I64(n), I64(V), I64(D)) >= 8 * n * (2 if multi and passes > 1 else 1) + (n // 32) * D * 4


def test_dropout_refusals():
    def call(x=ONE, y=ONE, n=8, dt=0, drop=100, rng=ONE):
        return lib().hs_dropout_rows(x, None, y, I64(n), dt, drop, rng, None)
    assert call(n=0) == 0
    assert call(n=-1) == -1 and call(dt=3) == -1 and call(drop=-1) == -1 and call(drop=65537) == -1
    assert call(x=None) == -3 and call(y=None) == -3 and call(rng=None) == -3


class hsGatedMlp(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("x", "w_gate", "w_up", "w_down")] + [(n, ctypes.c_int64) for n in ("ldx", "ld_gate", "ld_up", "ld_down", "rows", "dim", "hidden")]
                + [("dtype", ctypes.c_int32), ("activation", ctypes.c_int32), ("y", ctypes.c_void_p), ("saved", ctypes.c_void_p), ("grad", ctypes.c_void_p),
                   ("ld_grad", ctypes.c_int64)] + [(n, ctypes.c_void_p) for n in ("gx", "gw_gate", "gw_up", "gw_down", "ws")] + [("ws_bytes", ctypes.c_int64)])


def gated(**kw):
    a = hsGatedMlp(x=256, w_gate=256, w_up=256, w_down=256, ldx=16, ld_gate=16, ld_up=16, ld_down=32, rows=4, dim=16, hidden=32, dtype=1, activation=0, y=256,
                           saved=256, grad=256, ld_grad=16, ws=256, ws_bytes=1 << 40)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_gated_mlp_refusals():
    fwd, bwd = lib().hs_gated_mlp_fwd, lib().hs_gated_mlp_bwd
    for fn in (fwd, bwd):
        assert fn(None, None) == -3
        for bad in (dict(rows=0), dict(dim=0), dict(hidden=0), dict(rows=-1), dict(ldx=15), dict(ld_gate=1), dict(ld_up=1), dict(ld_down=31), dict(activation=5),
                    dict(activation=-1), dict(dtype=3), dict(hidden=(1 << 21) + 1, ld_down=1 << 23)):
            assert fn(gated(**bad), None) == -1, bad
        for name in ("x", "w_gate", "w_up", "w_down"):
            assert fn(gated(**{name: None}), None) == -3
    assert fwd(gated(y=None), None) == -3
    assert bwd(gated(grad=None), None) == -3 and bwd(gated(saved=None), None) == -3 and bwd(gated(ld_grad=3), None) == -1
    assert bwd(gated(gx=256, ws=None), None) == -3 and bwd(gated(gx=256, ws_bytes=8), None) == -1
    assert fwd(gated(saved=None, ws_bytes=8), None) == -1                    # (without a saved buffer the product lies in the work space)
    assert lib().hs_gated_mlp_saved_bytes(None) == -3 and lib().hs_gated_mlp_saved_bytes(gated(dtype=9)) == -1


def test_gated_mlp_work_space_counts_the_copies():
    ws = lib().hs_gated_mlp_fwd_ws_bytes
    assert ws(gated()) == 0 and ws(gated(x=258)) == 0                        # few rows: everything is read where it is
    plain = ws(gated(rows=100))
    assert ws(gated(rows=100, x=258)) - plain >= 100 * 16 * 2                # more: an operand that is not aligned is copied
    assert ws(gated(rows=100, w_down=264)) - plain >= 16 * 32 * 2
    assert ws(gated(rows=100, dtype=0)) >= 3 * 2 * (100 * 16 + 3 * 16 * 32)  # fp32: three planes of every operand
    assert lib().hs_gated_mlp_saved_bytes(gated()) >= 4 * 32 * 2             # the gated product; with wide rows both projections in fp32 too
    assert lib().hs_gated_mlp_saved_bytes(gated(dim=2048, ldx=2048, ld_gate=2048, ld_up=2048)) >= 4 * 32 * (2 + 8)
    assert lib().hs_gated_mlp_bwd_ws_bytes(gated(gx=256)) >= 2 * 4 * 32 * 2


def test_cpu_tensors_are_refused():
    t = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        row_ops.embedding_rows(torch.zeros(3, dtype=torch.long), t)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        row_ops.gated_mlp_rows(t, t, t, t.t())
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        row_ops.dropout_rows(t, 0.1, torch.zeros(2, dtype=torch.long))
    with pytest.raises(ValueError, match="activation"):
        row_ops.GatedMLP(8, 16, activation="tanh")
    with pytest.raises(ValueError, match="p must be"):
        row_ops.RowDropout(1.5)
    drop = row_ops.RowDropout(0.5).eval()
    assert drop(t) is t                                                      # outside training: nothing is drawn, nothing launched
