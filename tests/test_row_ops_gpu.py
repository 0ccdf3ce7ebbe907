"""GPU: the row operators (model/row_ops.py) against their definitions in 64 bits.

Tolerances are bounds, not observations: `half(t)` = eps / 2 for the rounding of a result, H32 = 2^-24 for each fp32 operation; a sum of n fp32 terms is off by
at most n 2^-24 times the sum of their magnitudes (the matrix instruction's own order and roundings: counted twice)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
H32 = 2.0 ** -24


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):        # half a step among the type's subnormals
    return {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[t]


def ops():
    from holoscene_amd.model import row_ops
    return row_ops


def within(got, want, bound, what):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound, worst error {float(err.max()):.3e}, bound there {float(bound.reshape(-1)[err.argmax()] if bound.numel() > 1 else bound):.3e}"


# ------------------------------------------------------------------------------------------------ codes by index
def embed_reference(idx, table, g, scale, padding):
    table, g, idx = table.double().cpu(), g.double().cpu(), idx.cpu().long()
    ok = (idx >= 0) & (idx < table.shape[0])
    out = torch.where(ok[..., None], table[idx.clamp(0, table.shape[0] - 1)] * scale, 0.0)
    flat, rows = idx.reshape(-1), g.reshape(-1, g.shape[-1])
    take = ok.reshape(-1) if padding is None else ok.reshape(-1) & (flat != padding)
    sums = torch.zeros_like(table).index_add_(0, flat[take], rows[take]) * scale
    mags = torch.zeros_like(table).index_add_(0, flat[take], rows[take].abs()) * abs(scale)
    count = torch.zeros(table.shape[0], dtype=torch.float64).index_add_(0, flat[take], torch.ones(int(take.sum()), dtype=torch.float64))
    return out, sums, mags, count


def check_embed(idx, table, scale=1.0, padding=None, out_dtype=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    out_dtype = out_dtype or table.dtype
    g = torch.randn(*idx.shape, table.shape[1], generator=gen).to(out_dtype).to(DEV)
    leaf = table.detach().requires_grad_()
    out = ops().embedding_rows(idx, leaf, scale=scale, padding_idx=padding, out_dtype=out_dtype)
    gt, = torch.autograd.grad(out, leaf, g)
    w_out, w_sum, mags, count = embed_reference(idx, table, g, scale, padding)
    assert out.shape == w_out.shape and out.dtype == out_dtype and gt.shape == table.shape and gt.dtype == table.dtype
    within(out.cpu(), w_out, w_out.abs() * (half(out_dtype) + 2 * H32) + tiny(out_dtype), "lookup")
    # a term passes through at most 32 additions in its chunk, count / 32 partials and 256 slots; or `count` in all when the run is short
    adds = torch.minimum(count, 32 + count / 32 + 256) + 3
    within(gt.cpu(), w_sum, w_sum.abs() * half(table.dtype) + mags * (adds * H32)[:, None] + tiny(table.dtype), "gradient")
    again, = torch.autograd.grad(ops().embedding_rows(idx, leaf, scale=scale, padding_idx=padding, out_dtype=out_dtype), leaf, g)
    assert torch.equal(gt, again), "the same sums in the same order"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (1, 7, 8), (5, 3, 33), (63, 2, 4), (64, 1, 8), (65, 1, 16), (1000, 17, 100), (1025, 5000, 12), (4097, 300, 65), (16384, 70000, 8), (4096, 66000, 5), (65537, 3, 6), (140001, 4500, 9),
                                   (16385, 9, 24), (20000, 3000, 3), (40000, 5001, 520)])
def test_embedding_sizes(n, V, D, dtype):
    gen = torch.Generator().manual_seed(n + V + D)
    idx = torch.randint(0, V, (n,), generator=gen).to(DEV)
    check_embed(idx, torch.randn(V, D, generator=gen).to(dtype).to(DEV), scale=1.0 if D % 2 else math.sqrt(D), seed=n)


@pytest.mark.parametrize("n", [0, 1, 64, 200, 16384, 131072])
def test_embedding_one_index_takes_everything(n):
    gen = torch.Generator().manual_seed(n)
    table = torch.randn(50, 32, generator=gen).to(DEV)
    check_embed(torch.full((n,), 7, device=DEV), table)
    check_embed(torch.full((n,), 49, dtype=torch.int32, device=DEV), table, padding=49)         # nothing is left


@pytest.mark.parametrize("n", [5000, 70000])
@pytest.mark.parametrize("V", [1, 2, 511, 512, 2046, 2047, 2048, 2049, 300000])
def test_embedding_digits(n, V):
    """Tables at the edges of the sort's digits and passes, 32-bit indices, a padding row."""
    gen = torch.Generator().manual_seed(n + V)
    idx = torch.randint(-1, V + 1, (n,), generator=gen, dtype=torch.int32).to(DEV)
    check_embed(idx, torch.randn(V, 12, generator=gen).to(torch.bfloat16).to(DEV), padding=V // 2)


def test_embedding_long_runs_and_gaps():
    gen = torch.Generator().manual_seed(3)
    for V, frames in ((1024, [5, 5, 900, 1023, 0, 0, 5, 77]), (3_000_000, [2_999_999, 12, 0, 2_048_001])):
        idx = torch.tensor(frames)[torch.arange(30011) * len(frames) // 30011].to(DEV)
        check_embed(idx, torch.randn(V, 4, generator=gen).to(DEV))


def test_embedding_indices_outside_and_padding():
    gen = torch.Generator().manual_seed(4)
    for n in (300, 20000):
        idx = torch.randint(-5, 25, (n,), generator=gen)
        idx[:3] = torch.tensor([2 ** 62, -2 ** 62, 2 ** 32 + 1])                # (their low 32 bits are rows of the table)
        check_embed(idx.to(DEV), torch.randn(20, 40, generator=gen).to(DEV), padding=4)
    table = torch.full((3, 8), float("nan"), device=DEV)
    out = ops().embedding_rows(torch.tensor([-1, 3], device=DEV), table)
    assert torch.equal(out, torch.zeros(2, 8, device=DEV)), "nothing of the table is read"


@pytest.mark.parametrize("dtype,out", [(torch.float32, torch.bfloat16), (torch.float32, torch.float16), (torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16)])
def test_embedding_mixed_types_shapes_and_strides(dtype, out):
    gen = torch.Generator().manual_seed(5)
    wide = torch.randn(31, 77, generator=gen).to(dtype).to(DEV)
    idx = torch.randint(0, 31, (6, 14), generator=gen).to(torch.int32).to(DEV)
    check_embed(idx, wide[:, 3:51], out_dtype=out)                              # rows of a wider table, not aligned
    check_embed(idx.t(), wide[:, :64], out_dtype=out, scale=-0.37)
    check_embed(idx[::2], wide.t(), out_dtype=out)                              # a transposed table
    assert ops().embedding_rows(idx, wide[:, :0]).shape == (6, 14, 0)


def test_embedding_gradient_of_broadcast_and_strided_results():
    gen = torch.Generator().manual_seed(6)
    idx = torch.randint(0, 9, (50,), generator=gen).to(DEV)
    table = torch.randn(9, 16, generator=gen).to(DEV).requires_grad_()
    gt, = torch.autograd.grad(ops().embedding_rows(idx, table).sum(), table)
    assert torch.equal(gt, torch.bincount(idx, minlength=9).float()[:, None].expand(9, 16))
    g = torch.randn(50, 40, generator=gen).to(DEV)
    a, = torch.autograd.grad(ops().embedding_rows(idx, table), table, g[:, 7:23])
    b, = torch.autograd.grad(ops().embedding_rows(idx, table), table, g[:, 7:23].contiguous())
    assert torch.equal(a, b)


def test_embedding_beyond_32_bits():
    """More result elements than a grid has threads, gradients behind 4 GiB."""
    n, V, D = 65600, 5, 65537
    gen = torch.Generator().manual_seed(8)
    idx = torch.randint(-1, V, (n,), generator=gen).to(DEV)
    table = torch.randn(V, D, generator=gen).to(torch.bfloat16).to(DEV).requires_grad_()
    out = ops().embedding_rows(idx, table)
    assert out.numel() > 1 << 32
    for v in range(V):
        at = (idx == v).nonzero()[:, 0]
        assert all(torch.equal(out[i], table[v]) for i in (int(at[0]), int(at[len(at) // 2]), int(at[-1])))
    for i in range(0, n, 4100):
        part = idx[i:i + 4100, None]
        assert torch.equal(out[i:i + 4100], torch.where(part >= 0, table.detach()[part[:, 0].clamp(min=0)], torch.zeros((), dtype=table.dtype, device=DEV)))
    # whole numbers below 2^24: the sums are exact; every row ends in a value of its own
    g = torch.ones_like(out)
    g[:, -1] = (torch.arange(n, device=DEV) % 3).to(g.dtype)
    gt, = torch.autograd.grad(out, table, g)
    want = torch.stack([(idx == v).sum() for v in range(V)]).float().to(gt.dtype)[:, None].expand(V, D).clone()
    want[:, -1] = torch.stack([(torch.arange(n, device=DEV) % 3)[idx == v].sum() for v in range(V)]).float().to(gt.dtype)
    assert torch.equal(gt, want)


def test_embedding_refusals():
    f, table, idx = ops().embedding_rows, torch.zeros(4, 8, device=DEV), torch.zeros(3, dtype=torch.long, device=DEV)
    for bad in (dict(indices=idx.float()), dict(indices=idx.short()), dict(table=table[0]), dict(table=table.double()), dict(padding_idx=4), dict(padding_idx=-1),
                dict(out_dtype=torch.float64), dict(indices=idx.cpu()), dict(table=table.to_sparse())):
        with pytest.raises(RuntimeError):
            f(**{**dict(indices=idx, table=table), **bad})


# ------------------------------------------------------------------------------------------------ dropout
def keep_reference(n, drop, seed, call, first=0):
    """Philox-4x32-10 in Python integers: elements 8 first, 8 first + 1, .. n of them."""
    out = []
    for grp in range(first, first + (n + 7) // 8):
        c, k = [grp & 0xffffffff, grp >> 32, call & 0xffffffff, call >> 32], [seed & 0xffffffff, seed >> 32]
        for _ in range(10):
            a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(b >> 32) ^ c[1] ^ k[0], b & 0xffffffff, (a >> 32) ^ c[3] ^ k[1], a & 0xffffffff]
            k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
        for w in c:
            out += [w & 0xffff, w >> 16]
    return torch.tensor(out[:n]) >= drop


def test_philox_known_answer():
    """The published test vector of Philox-4x32-10: counter and key all ones -> 408f276d 41c83b0e a20bc7c6 6d5451fd."""
    want = [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    c, k = [0xffffffff] * 4, [0xffffffff] * 2
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xffffffff, (a >> 32) ^ c[3] ^ k[1], a & 0xffffffff]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    assert c == want


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,p,seed,call", [(1, 0.5, 1, 0), (7, 0.1, 2, 3), (8, 0.0, 3, 1), (9, 1.0, 4, 1), (2049, 0.3, (1 << 63) - 1, 1 << 40), (5000, 0.9, -7, -1), (4096, 1e-6, 5, 5)])
def test_dropout_mask_and_values(n, p, seed, call, dtype):
    gen = torch.Generator().manual_seed(n)
    x, r, g = (torch.randn(n, generator=gen).to(dtype) for _ in range(3))
    drop = math.floor(p * 65536 + 0.5)
    keep = keep_reference(n, drop, seed % (1 << 64), call % (1 << 64))
    s = 65536 / (65536 - drop) if drop < 65536 else 0.0
    rng = torch.tensor([seed, call], dtype=torch.int64, device=DEV)
    x_, r_ = x.to(DEV).requires_grad_(), r.to(DEV).requires_grad_()
    for res in (None, r_):
        y = ops().dropout_rows(x_, p, rng, residual=res)
        kept = torch.where(keep, x.double() * s, 0.0)
        want = kept + (0 if res is None else r.double())
        within(y.cpu(), want, want.abs() * half(dtype) + (kept.abs() * 2 + want.abs()) * H32 * (1 + half(dtype)) + tiny(dtype), "value")
        grads = torch.autograd.grad(y, [x_] if res is None else [x_, r_], g.to(DEV))
        want = torch.where(keep, g.double() * s, 0.0)
        within(grads[0].cpu(), want, want.abs() * (half(dtype) + 3 * H32) + tiny(dtype), "gradient")
        assert torch.equal(grads[0].cpu() != 0, keep & (g != 0)) or drop == 65536
        if res is not None:
            assert torch.equal(grads[1].cpu(), g)
    assert torch.equal(rng.cpu(), torch.tensor([seed, call])), "rng is read only"


def test_dropout_dropped_infinities_strides_and_shares():
    x = torch.full((64, 33), float("inf"), device=DEV)
    x[::2] = float("nan")
    rng = torch.tensor([11, 2], device=DEV)
    y = ops().dropout_rows(x, 0.5, rng)
    keep = keep_reference(64 * 33, 32768, 11, 2).view(64, 33).to(DEV)
    assert torch.equal(y[~keep], torch.zeros_like(y[~keep])) and not bool(torch.isfinite(y[keep]).any())
    base = torch.randn(40, 70, device=DEV)
    for v in (base.t(), base[:, 5:48], base[1:], base[:1].expand(9, 70), base.view(4, 10, 70)):
        assert torch.equal(ops().dropout_rows(v, 0.3, rng), ops().dropout_rows(v.contiguous(), 0.3, rng))
    flat = torch.randn(3001, device=DEV)
    assert torch.equal(ops().dropout_rows(flat[1:], 0.3, rng), ops().dropout_rows(flat[1:].clone(), 0.3, rng)), "any alignment"
    n = 1 << 20
    for p in (0.1, 0.5):
        share = float((ops().dropout_rows(torch.ones(n, device=DEV), p, rng) == 0).float().mean())
        assert abs(share - p) < 6 * math.sqrt(p * (1 - p) / n) + 2.0 ** -17      # six standard deviations
    other = ops().dropout_rows(base, 0.5, torch.tensor([11, 3], device=DEV))
    assert not torch.equal(other == 0, ops().dropout_rows(base, 0.5, rng) == 0), "another call, another mask"
    assert ops().dropout_rows(base[:0], 0.5, rng).shape == (0, 70)


def test_dropout_beyond_32_bits():
    n = (1 << 33) + 2051                   # the last groups' counters have more than 30 bits, their elements more than 33
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    y = ops().dropout_rows(x, 0.5, torch.tensor([9, 4], device=DEV))
    for first, count in ((0, 64), ((1 << 29) - 4, 64), (1 << 29, 2051)):
        want = keep_reference(count, 32768, 9, 4, first)
        assert torch.equal(y[8 * first:8 * first + count].cpu(), want.to(torch.bfloat16) * 2)


def test_dropout_refusals():
    x, rng = torch.zeros(4, 4, device=DEV), torch.zeros(2, dtype=torch.long, device=DEV)
    for args, kw in (((x, -0.1, rng), {}), ((x, 1.1, rng), {}), ((x, float("nan"), rng), {}), ((x.double(), 0.1, rng), {}), ((x, 0.1, rng.int()), {}),
                     ((x, 0.1, torch.zeros(4, dtype=torch.long, device=DEV)[::2]), {}), ((x, 0.1, rng[:1]), {}), ((x, 0.1, rng.cpu()), {}),
                     ((x, 0.1, rng), dict(residual=x[:1])), ((x, 0.1, rng), dict(residual=x.half()))):
        with pytest.raises(RuntimeError):
            ops().dropout_rows(*args, **kw)
    leaf = torch.randn(8, device=DEV, requires_grad=True)
    y = ops().dropout_rows(leaf, 0.5, rng)
    rng[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ------------------------------------------------------------------------------------------------ gated block
ACTS = ["silu", "gelu", "gelu_tanh", "sigmoid", "relu"]
# bounds of |act'| and |act''|
SLOPE = dict(silu=1.1, gelu=1.13, gelu_tanh=1.13, sigmoid=0.25, relu=1.0)
CURVE = dict(silu=0.5, gelu=0.8, gelu_tanh=0.81, sigmoid=0.1, relu=0.0)


def gated_reference(x, wg, wu, wd, act, gy):
    """Values and error bounds of y, gx, gWg, gWu, gWd in 64 bits on the GPU (2-D operands)."""
    t = x.dtype
    # results; operands of a second product (few results, 16-bit types: two planes, each rounded by half a step of what the first leaves)
    e, eo = half(t), (H32 if t == torch.float32 else half(t) ** 2 if min(x.shape[0], wg.shape[0]) * x.shape[1] <= 2048 else half(t))
    x, wg, wu, wd, gy = (v.detach().double() for v in (x, wg, wu, wd, gy))

    def acc(k):             # fp32 accumulation over k products, counted twice; fp32 operands: their dropped plane products too
        return (k + 16) * 2 * H32
    M, D, F = x.shape[0], x.shape[1], wg.shape[0]
    g, u = x @ wg.t(), x @ wu.t()
    dg, du = acc(D) * (x.abs() @ wg.abs().t()), acc(D) * (x.abs() @ wu.abs().t())
    leaf = g.clone().requires_grad_()
    fn = dict(silu=torch.nn.functional.silu, gelu=torch.nn.functional.gelu, sigmoid=torch.sigmoid, relu=torch.relu,
              gelu_tanh=lambda v: torch.nn.functional.gelu(v, approximate="tanh"))[act]
    a = fn(leaf)
    da, = torch.autograd.grad(a.sum(), leaf)
    a = a.detach()
    fn_err = 8 * H32 * (1 + a.abs())                                    # the activation's own fp32 arithmetic, absolute: |terms| <= 1 + |g|
    d_a = SLOPE[act] * dg + fn_err
    h = a * u
    dh = d_a * (u.abs() + du) + (a.abs() + d_a) * du + 2 * H32 * h.abs()
    dh = dh + eo * (h.abs() + dh) + tiny(t)
    y = h @ wd.t()
    dy = dh @ wd.abs().t() + acc(F) * ((h.abs() + dh) @ wd.abs().t())
    dy = dy + e * (y.abs() + dy) + tiny(t)
    gh = gy @ wd
    dgh = acc(D) * (gy.abs() @ wd.abs())
    dgs, dus = dg + e * (g.abs() + dg) + tiny(t), du + e * (u.abs() + du) + tiny(t)     # as kept for the backward pass
    das = SLOPE[act] * dgs + fn_err
    dda = CURVE[act] * dgs + 8 * H32 * (1 + g.abs()) + ((g.abs() <= dgs).double() if act == "relu" else 0.0)
    gg, gu = gh * u * da, gh * a

    def product(parts):     # error of a product of (value, error) pairs
        val, err = parts[0]
        for v, d in parts[1:]:
            val, err = val * v, err * (v.abs() + d) + val.abs() * d
        return err + 3 * H32 * (val.abs() + err)
    dgg, dgu = product([(gh, dgh), (u, dus), (da, dda)]), product([(gh, dgh), (a, das)])
    dgg, dgu = dgg + eo * (gg.abs() + dgg) + tiny(t), dgu + eo * (gu.abs() + dgu) + tiny(t)

    def mm(a_, da_, b_, k):
        v = a_ @ b_
        d = da_ @ b_.abs() + acc(k) * ((a_.abs() + da_) @ b_.abs())
        return v, d

    def done(v, d):
        return v, d + e * (v.abs() + d) + tiny(t)
    gx1, dgx1 = mm(gg, dgg, wg, 2 * F)
    gx2, dgx2 = mm(gu, dgu, wu, 2 * F)
    out = [done(y, dy - e * y.abs() * 0), done(gx1 + gx2, dgx1 + dgx2), done(*mm(gg.t(), dgg.t(), x, M)), done(*mm(gu.t(), dgu.t(), x, M))]
    gwd, dgwd = (h.t() @ gy).t(), (dh.t() @ gy.abs()).t() + acc(M) * ((h.abs() + dh).t() @ gy.abs()).t()
    return out + [done(gwd, dgwd)]


def gated_inputs(M, D, F, dtype, seed=0):
    gen = torch.Generator().manual_seed(1000 * M + 10 * D + F + seed)
    return [(torch.randn(*s, generator=gen) * k).to(dtype).to(DEV) for s, k in (((M, D), 1.0), ((F, D), D ** -0.5), ((F, D), D ** -0.5), ((D, F), F ** -0.5), ((M, D), 1.0))]


def check_gated(x, wg, wu, wd, gy, act):
    ref = gated_reference(x.reshape(-1, x.shape[-1]), wg, wu, wd, act, gy.reshape(-1, x.shape[-1]))
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu, wd)]
    y = ops().gated_mlp_rows(*leaves, activation=act)
    grads = torch.autograd.grad(y, leaves, gy)
    with torch.no_grad():
        alone = ops().gated_mlp_rows(x, wg, wu, wd, activation=act)
    assert torch.equal(alone, y), "with and without a gradient: the same numbers"
    assert y.dtype == x.dtype and y.shape == x.shape
    for got, (want, bound), what in zip((y, *grads), ref, ("y", "gx", "gw_gate", "gw_up", "gw_down")):
        within(got.reshape(want.shape), want, bound, f"{what} {act}")
    for t, g in zip(leaves, grads):
        assert g.shape == t.shape and g.dtype == t.dtype


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,D,F", [(1, 1, 1), (1, 8, 8), (2, 3, 5), (16, 64, 32), (17, 33, 65), (31, 264, 40), (64, 64, 64), (65, 72, 130), (130, 256, 96), (257, 100, 300), (300, 264, 520),
                                   (1, 512, 1000), (13, 250, 170), (1000, 24, 16), (500, 1000, 4), (1, 2048, 24), (2, 1024, 300), (2, 1025, 300), (300, 13, 157), (300, 13, 158), (700, 1000, 2)])
def test_gated_sizes(M, D, F, dtype):
    check_gated(*gated_inputs(M, D, F, dtype), act=ACTS[(M + D + F) % 5])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_gated_activations(act, dtype):
    x, wg, wu, wd, gy = gated_inputs(40, 48, 72, dtype)
    check_gated(x * 4, wg, wu, wd, gy, act)          # (gates of several units: both tails of the activation)


@pytest.mark.parametrize("dtype,M,D,F", [(torch.float32, 50, 1101, 7700), (torch.float32, 64, 4000, 2100), (torch.bfloat16, 1, 4096, 2200), (torch.float16, 20, 1501, 4099), (torch.bfloat16, 4096, 64, 1600), (torch.float16, 2000, 1000, 1210), (torch.bfloat16, 20000, 256, 128), (torch.float32, 3000, 72, 700),
                                         (torch.bfloat16, 513, 1536, 2056)])
def test_gated_large_tiles_and_slices(dtype, M, D, F):
    check_gated(*gated_inputs(M, D, F, dtype), act="silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,D,F", [(2500, 200, 90), (1500, 333, 777), (900, 2100, 130), (5000, 40, 500), (33, 700, 1300), (6000, 300, 17)])
def test_gated_uneven_slices(M, D, F, dtype):
    check_gated(*gated_inputs(M, D, F, dtype), "silu")


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_strides_and_alignment(dtype):
    M, D, F = 70, 64, 96
    x, wg, wu, wd, gy = gated_inputs(M, D, F, dtype)

    def window(t, ahead, behind):
        wide = torch.full((t.shape[0], t.shape[1] + ahead + behind), float("nan"), dtype=t.dtype, device=DEV)      # what lies beside the rows is never used
        wide[:, ahead:ahead + t.shape[1]] = t
        return wide[:, ahead:ahead + t.shape[1]]
    for ahead, behind in ((8, 8), (1, 2), (0, 3)):
        check_gated(window(x, ahead, behind), window(wg, ahead, behind), window(wu, 8, 16), window(wd, ahead, behind), window(gy, ahead, behind), "gelu")
    check_gated(x, wg.t().contiguous().t(), wu, wd.t().contiguous().t(), gy.t().contiguous().t(), "silu")
    check_gated(x.view(7, 10, D), wg, wu, wd, gy.view(7, 10, D), "silu")
    check_gated(x[:1].expand(33, D), wg, wu, wd, gy[:1].expand(33, D), "silu")
    for odd in (60, 61):        # odd widths inside wider rows
        check_gated(window(x[:, :odd], 4, 4), window(wg[:, :odd], 4, 4), window(wu[:, :odd], 4, 4), wd[:odd].contiguous(), window(gy[:, :odd], 4, 4), "silu")


def test_gated_partial_gradients():
    x, wg, wu, wd, gy = gated_inputs(50, 40, 56, torch.bfloat16)
    full = [t.detach().requires_grad_() for t in (x, wg, wu, wd)]
    want = torch.autograd.grad(ops().gated_mlp_rows(*full), full, gy)
    for pick in ((0,), (1,), (2,), (3,), (0, 3), (1, 2), (2, 3)):
        some = [t.detach().requires_grad_(i in pick) for i, t in enumerate((x, wg, wu, wd))]
        got = torch.autograd.grad(ops().gated_mlp_rows(*some), [some[i] for i in pick], gy)
        assert all(torch.equal(a, want[i]) for a, i in zip(got, pick))


def test_gated_beyond_32_bits():
    """A hidden layer of more than 2^32 elements: rows at its start, behind 2^31 and at its end."""
    M, D, F = (1 << 20) + 77, 64, 4104
    x, wg, wu, wd, _ = gated_inputs(200, D, F, torch.bfloat16)
    at = torch.cat([torch.arange(64), torch.arange(64) + M // 2 + 100, torch.arange(72) + M - 72]).to(DEV)
    rows, gy = torch.zeros(M, D, dtype=x.dtype, device=DEV), torch.zeros(M, D, dtype=x.dtype, device=DEV)
    rows[at] = x
    gy[at] = torch.randn(200, D, generator=torch.Generator().manual_seed(9)).to(x.dtype).to(DEV)
    leaves = [t.requires_grad_() for t in (rows, wg, wu, wd)]
    y = ops().gated_mlp_rows(*leaves)
    grads = torch.autograd.grad(y, leaves, gy)
    # rows of zeros give zeros everywhere: the sums over the rows have 200 terms
    ref = gated_reference(x, wg, wu, wd, "silu", gy[at])
    for got, (want, bound), what in zip((y[at], grads[0][at], *grads[1:]), ref, ("y", "gx", "gw_gate", "gw_up", "gw_down")):
        within(got, want, bound, what)
    rest = torch.ones(M, dtype=torch.bool, device=DEV)
    rest[at] = False
    assert not bool(y[rest].any()) and not bool(grads[0][rest].any())


@pytest.mark.parametrize("M,D,F", [(0, 8, 16), (4, 8, 0), (0, 0, 0), (3, 0, 5)])
def test_gated_empty(M, D, F):
    t = [torch.randn(*s, device=DEV).requires_grad_() for s in ((M, D), (F, D), (F, D), (D, F))]
    y = ops().gated_mlp_rows(*t)
    assert y.shape == (M, D) and not bool(y.any())
    for g, v in zip(torch.autograd.grad(y, t, torch.randn(M, D, device=DEV)), t):
        assert g.shape == v.shape and not bool(g.any())


def test_gated_gradient_against_differences():
    x, wg, wu, wd, gy = gated_inputs(9, 12, 20, torch.float32)
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
    gen = torch.Generator().manual_seed(9)
    for act in ("silu", "gelu", "gelu_tanh", "sigmoid"):
        grads = torch.autograd.grad(ops().gated_mlp_rows(*leaves, activation=act), leaves, gy)
        for i in range(4):
            d = torch.randn(leaves[i].shape, generator=gen).to(DEV)
            d /= d.norm()
            step = 2.0 ** -7
            with torch.no_grad():
                ends = [(ops().gated_mlp_rows(*[t + s * step * d if j == i else t for j, t in enumerate(leaves)], activation=act).double() * gy.double()).sum() for s in (1, -1)]
            slope, want = float(ends[0] - ends[1]) / (2 * step), float((grads[i].double() * d.double()).sum())
            # central difference: step^2 / 6 of a third derivative of order |gy| |y| (sums of 108 terms of order one), and fp32 noise 2^-22 / step of the sum
            assert abs(slope - want) < 3e-3 * (1 + float(grads[i].norm())), (act, i, slope, want)


def test_gated_not_finite_stays_in_its_row():
    for dtype in TYPES:
        x, wg, wu, wd, gy = gated_inputs(40, 64, 64, dtype)
        clean = ops().gated_mlp_rows(x, wg, wu, wd)
        x[7, 3], x[20, 0] = float("nan"), float("inf")
        y = ops().gated_mlp_rows(x, wg, wu, wd)
        rows = torch.ones(40, dtype=torch.bool)
        rows[[7, 20]] = False
        assert torch.equal(y[rows], clean[rows]) and bool(torch.isnan(y[7]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
def test_gated_far_preactivations(act, dtype):
    """Preactivations whose square passes the largest float: the functions and their slopes have reached their limits."""
    for rows, D in ((3, 8), (70, 8), (70, 1000)):           # few rows; slopes from G computed again, and from G kept
        x = torch.zeros(rows, D, device=DEV, dtype=dtype)
        x[:, 0] = 1
        wg, wu, wd = (torch.zeros(s, device=DEV, dtype=dtype) for s in ((16, D), (16, D), (D, 16)))
        wg[:, 0] = torch.tensor([1e20, -1e20, 1.0, -1.0]).repeat(4).to(dtype).to(DEV)
        wu[:, 0] = 0.5
        wd[0, :] = 2.0 ** -60
        leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
        y = ops().gated_mlp_rows(*leaves, activation=act)
        grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
        assert all(bool(torch.isfinite(t).all()) for t in (y, *grads)), (rows, D)
        slope = {"sigmoid": [0.0, 0.0], "relu": [1.0, 0.0]}.get(act, [1.0, 0.0])
        want = torch.tensor(slope, dtype=torch.float64) * 0.5 * 2.0 ** -60 * rows
        within(grads[1][:2, 0].cpu(), want, want * (rows + 8) * half(dtype), "slope")


def test_embedding_gradient_ignores_what_takes_none():
    """Not a number in the gradient of padded and outside positions."""
    for n in (100, 5000, 40000):
        idx = torch.arange(n, device=DEV) % 7 - 1
        table, g = torch.randn(5, 40, device=DEV).requires_grad_(), torch.ones(n, 40, device=DEV)
        g[(idx < 0) | (idx > 4) | (idx == 2)] = float("nan")
        gt, = torch.autograd.grad(ops().embedding_rows(idx, table, padding_idx=2), table, g)
        want = torch.bincount(idx[(idx >= 0) & (idx < 5) & (idx != 2)], minlength=5).float()[:, None].expand(5, 40)
        assert torch.equal(gt, want)


@pytest.mark.parametrize("tied", [(1, 2), (0, 0)])
def test_gated_shared_operands(tied):
    """One tensor as both projections; x as its own residual in dropout."""
    x, wg, wu, wd, gy = gated_inputs(70, 64, 96, torch.float32)
    if tied == (1, 2):
        w = wg.clone().requires_grad_()
        g, = torch.autograd.grad(ops().gated_mlp_rows(x, w, w, wd), w, gy)
        a, b = wg.clone().requires_grad_(), wg.clone().requires_grad_()
        ga, gb = torch.autograd.grad(ops().gated_mlp_rows(x, a, b, wd), (a, b), gy)
        assert torch.equal(g, ga + gb)
    else:
        t, rng = x.clone().requires_grad_(), torch.tensor([1, 2], device=DEV)
        g, = torch.autograd.grad(ops().dropout_rows(t, 0.4, rng, residual=t), t, gy)
        assert torch.equal(g, ops().dropout_rows(gy, 0.4, rng) + gy)


def test_calls_from_two_threads():
    """Two host threads, a stream each: nothing is shared between calls."""
    import threading
    inputs = [_chain_inputs(torch.bfloat16, n=200 + 37 * k, seed=k) for k in range(2)]
    want = [_chain(*i) for i in inputs]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = _chain(*inputs[k])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                    bad.append(k)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_gated_refusals():
    x, wg, wu, wd, _ = gated_inputs(4, 8, 16, torch.float32)
    f = ops().gated_mlp_rows
    for args in ((x.double(), wg, wu, wd), (x, wg.half(), wu, wd), (x, wg, wu[:8], wd), (x, wg, wu, wd.t()), (x[:, :4], wg, wu, wd), (x, wg, wu, wd[0]), (x.cpu(), wg, wu, wd),
                 (x, wg, wu.cpu(), wd), (torch.zeros((), device=DEV), wg, wu, wd)):
        with pytest.raises(RuntimeError):
            f(*args)
    with pytest.raises(RuntimeError, match="activation"):
        f(x, wg, wu, wd, activation="tanh")
    leaf = x.requires_grad_()
    g, = torch.autograd.grad(f(leaf, wg, wu, wd).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("lead", [(6,), (2, 3)])
def test_saved_operands_are_guarded(lead):
    """A second backward pass, or one after an operand has been written, is refused as for torch's own operators."""
    x, wg, wu, wd, _ = gated_inputs(6, 8, 16, torch.float32)
    x, leaf = x.view(*lead, 8), wg.clone().requires_grad_()
    y = ops().gated_mlp_rows(x, leaf, wu, wd)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    for t in (x, wu):
        y = ops().gated_mlp_rows(x, leaf, wu, wd)
        t.mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    idx, table = torch.arange(4, device=DEV), torch.randn(5, 8, device=DEV, requires_grad=True)
    out = ops().embedding_rows(idx, table)
    idx += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_second_derivatives_are_refused():
    x, wg, wu, wd, gy = gated_inputs(6, 8, 16, torch.float32)
    rng, idx = torch.tensor([3, 4], device=DEV), torch.arange(6, device=DEV)
    for f, leaf in ((lambda t: ops().gated_mlp_rows(t, wg, wu, wd), x), (lambda t: ops().dropout_rows(t, 0.5, rng), x), (lambda t: ops().dropout_rows(x, 0.5, rng, residual=t), x),
                    (lambda t: ops().embedding_rows(idx, t), x)):
        leaf, g = leaf.clone().requires_grad_(), gy.clone().requires_grad_()
        first, = torch.autograd.grad(f(leaf), leaf, g, create_graph=True)
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            first.sum().backward()


# ------------------------------------------------------------------------------------------------ together
def _chain(idx, table, ws, rng, gy):
    """Codes -> dropout -> gated block -> dropout + residual, and all gradients."""
    leaves = [t.detach().requires_grad_() for t in (table, *ws)]
    r = ops()
    x = r.embedding_rows(idx, leaves[0], scale=4.0, padding_idx=0)
    x = r.dropout_rows(x, 0.1, rng[0])
    y = r.dropout_rows(r.gated_mlp_rows(x, *leaves[1:]), 0.2, rng[1], residual=x)
    return [y.detach(), *torch.autograd.grad(y, leaves, gy)]


def _chain_inputs(dtype, n=200, seed=0):
    gen = torch.Generator().manual_seed(70 + seed)
    x, wg, wu, wd, gy = gated_inputs(n, 40, 72, dtype, seed)
    idx = torch.randint(0, 30, (n,), generator=gen).to(DEV)
    rng = [torch.tensor([seed + 1, k], device=DEV) for k in (1, 2)]
    return idx, (torch.randn(30, 40, generator=gen) * 0.25).to(dtype).to(DEV), (wg, wu, wd), rng, gy


@pytest.mark.parametrize("dtype", TYPES)
def test_chain_matches_its_definition(dtype):
    idx, table, ws, rng, gy = _chain_inputs(dtype)
    got = _chain(idx, table, ws, rng, gy)
    n, D = gy.shape
    leaves = [t.double().requires_grad_() for t in (table, *ws)]
    m1, m2 = (keep_reference(n * D, math.floor(p * 65536 + 0.5), 1, c).view(n, D).to(DEV) * (65536 / (65536 - math.floor(p * 65536 + 0.5))) for p, c in ((0.1, 1), (0.2, 2)))
    x = torch.nn.functional.embedding(idx, leaves[0], padding_idx=0) * 4.0 * m1
    y = m2 * ((torch.nn.functional.silu(x @ leaves[1].t()) * (x @ leaves[2].t())) @ leaves[3].t()) + x
    want = [y, *torch.autograd.grad(y, leaves, gy.double())]
    # every tensor between two operators is rounded to the type (5 of them forward, 5 backward), each rounding relative to its own size; sums over 72 or 200
    # such terms of either sign grow like their norm.  Norms: 10 roundings of half(t) each, and the fp32 arithmetic (2^-18 covers sums of 200 terms)
    for g, w, what in zip(got, want, ("y", "table", "w_gate", "w_up", "w_down")):
        rel = float((g.detach().double() - w).norm() / w.norm())
        assert rel < 10 * half(dtype) + 2.0 ** -18, (what, rel)


def test_chain_on_another_stream_and_in_a_graph():
    idx, table, ws, rng, gy = _chain_inputs(torch.bfloat16)
    want = _chain(idx, table, ws, rng, gy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _chain(idx, table, ws, rng, gy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _chain(idx, table, ws, rng, gy)
        rng[0][1:].add_(10)
        rng[1][1:].add_(10)
    graph2 = torch.cuda.CUDAGraph()         # a second graph of other sizes lives beside it
    other = _chain_inputs(torch.bfloat16, n=333, seed=5)
    want2 = _chain(*other)
    with torch.cuda.graph(graph2):
        out2 = _chain(*other)
    start = [r.clone() for r in rng]
    for k in range(4):
        new = _chain_inputs(torch.bfloat16, seed=k)
        for dst, src in zip((idx, table, *ws, gy), (new[0], new[1], *new[2], new[4])):
            dst.copy_(src)
        step = [s + torch.tensor([0, 10 * k], device=DEV) for s in start]
        graph.replay()
        graph2.replay()
        torch.cuda.synchronize()
        want = _chain(idx, table, ws, step, gy)
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        assert all(torch.equal(a, b) for a, b in zip(out2, want2)), k


def test_modules_train_together():
    """The modules in one model: they run, draw a new mask every call, and give gradients to every parameter."""
    r = ops()
    torch.manual_seed(0)
    emb, mlp, drop = r.RowEmbedding(12, 32, std=1.0, padding_idx=0).to(DEV), r.GatedMLP(32, 48).to(DEV), r.RowDropout(0.25, seed=3).to(DEV)
    idx = torch.arange(60, device=DEV) % 12
    outs = []
    for _ in range(2):
        x = emb(idx)
        y = drop(mlp(x), residual=x)
        y.square().mean().backward()
        outs.append(y.detach())
    assert not torch.equal(*outs) and int(drop.rng[1]) == 2
    for p in (emb.weight, mlp.w_gate, mlp.w_up, mlp.w_down):
        assert p.grad is not None and bool(p.grad.abs().sum() > 0)
    assert not bool(emb.weight.grad[0].any())
    drop.eval()
    assert torch.equal(drop(outs[0], residual=outs[1]), outs[0] + outs[1]) and int(drop.rng[1]) == 2


def test_training_step_in_a_graph():
    """The modules' forward and backward() captured as one graph, the leaves' gradients written by every replay, against the same steps run eagerly."""
    r = ops()
    torch.manual_seed(1)

    def make():
        torch.manual_seed(2)
        return r.RowEmbedding(40, 64, std=1.0).to(DEV), r.GatedMLP(64, 96, "gelu").to(DEV), r.RowDropout(0.2, seed=5).to(DEV)

    def step(mods, idx, gy):
        emb, mlp, drop = mods
        x = emb(idx)
        y = drop(mlp(x), residual=x)
        y.backward(gy)
        return y.detach()
    idx, gy = torch.arange(300, device=DEV) * 7 % 40, torch.randn(300, 64, device=DEV)
    captured, eager = make(), make()
    params = [[p for m in mods for p in m.parameters()] for mods in (captured, eager)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(captured, idx, gy)
    torch.cuda.current_stream().wait_stream(side)
    for p in params[0]:
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(captured, idx, gy)
    eager[2].rng.copy_(captured[2].rng)
    gen = torch.Generator().manual_seed(3)
    for k in range(4):
        idx.copy_(torch.randint(0, 40, (300,), generator=gen))
        gy.copy_(torch.randn(300, 64, generator=gen))
        graph.replay()
        for p in params[1]:
            p.grad = None
        want = step(eager, idx, gy)
        torch.cuda.synchronize()
        assert torch.equal(out, want), k
        assert all(torch.equal(a.grad, b.grad) for a, b in zip(*params)), k
    assert torch.equal(captured[2].rng, eager[2].rng)
