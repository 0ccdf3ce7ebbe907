"""GPU: what the row operators (model/row_ops.py) owe a caller beside their values: gradients that are asked to be differentiable, results that are written in
place, operands that are not finite, lazily negated operands, transforms that would lose the operators without a word."""
import pytest
import torch

from test_row_ops_gpu import DEV, TYPES, gated_inputs, ops

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ gradients of gradients
@pytest.mark.parametrize("which", [0, 1, 2, 3])
@pytest.mark.parametrize("form", ["rows", "leading dims", "copied"])
def test_gradient_penalty_is_refused(which, form):
    """grad(y, t, ones, create_graph=True): the incoming gradient is a constant, the block's gradients still depend on its operands."""
    x, wg, wu, wd, _ = gated_inputs(6, 8, 16, torch.float32)
    if form == "leading dims":
        x = x.view(2, 3, 8)
    if form == "copied":
        x, wg = x.t().contiguous().t(), wg.t().contiguous().t()
    leaves = [t.clone().requires_grad_(i == which or (which == 3 and i == 0)) for i, t in enumerate((x, wg, wu, wd))]        # (Wd's gradient depends on the others only)
    y = ops().gated_mlp_rows(*leaves)
    first, = torch.autograd.grad(y, leaves[which], torch.ones_like(y), create_graph=True)
    want, = torch.autograd.grad(ops().gated_mlp_rows(*leaves), leaves[which], torch.ones_like(y))
    assert torch.equal(first, want) and first.requires_grad
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        (y.mean() + (first.norm() - 1) ** 2).backward()


def test_gradients_that_depend_on_nothing_are_constants():
    """Lookup, dropout, and Wd's gradient where nothing else takes one: linear, so with a constant incoming gradient there is nothing to differentiate."""
    x, wg, wu, wd, _ = gated_inputs(6, 8, 16, torch.float32)
    rng, idx = torch.tensor([3, 4], device=DEV), torch.arange(6, device=DEV)
    for f, leaf in ((lambda t: ops().embedding_rows(idx, t), x), (lambda t: ops().dropout_rows(t, 0.5, rng), x), (lambda t: ops().dropout_rows(x, 0.5, rng, residual=t), x),
                    (lambda t: ops().gated_mlp_rows(x, wg, wu, t), wd)):
        leaf = leaf.clone().requires_grad_()
        y = f(leaf)
        first, = torch.autograd.grad(y, leaf, torch.ones_like(y), create_graph=True)
        (y.mean() + (first.norm() - 1) ** 2).backward()
        alone, = torch.autograd.grad(f(leaf).mean(), leaf)
        assert torch.equal(leaf.grad, alone)


def test_backward_with_create_graph_keeps_its_values():
    x, wg, wu, wd, gy = gated_inputs(40, 24, 32, torch.float32)
    a, b = ([t.clone().requires_grad_() for t in (x, wg, wu, wd)] for _ in range(2))
    ops().gated_mlp_rows(*a).backward(gy)
    grads = torch.autograd.grad(ops().gated_mlp_rows(*b), b, gy, create_graph=True)
    assert all(torch.equal(s.grad, t) for s, t in zip(a, grads))


# ------------------------------------------------------------------------------------------------ transforms
def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd
    x, wg, wu, wd, gy = gated_inputs(6, 8, 16, torch.float32)
    rng, idx = torch.tensor([3, 4], device=DEV), torch.arange(6, device=DEV)
    with fwd.dual_level():
        d = fwd.make_dual(x, gy)
        for f in (lambda: ops().gated_mlp_rows(d, wg, wu, wd), lambda: ops().gated_mlp_rows(x, wg, wu, fwd.make_dual(wd, wd)), lambda: ops().embedding_rows(idx, d),
                  lambda: ops().dropout_rows(d, 0.5, rng), lambda: ops().dropout_rows(x, 0.5, rng, residual=d)):
            with pytest.raises(RuntimeError, match="has a tangent"):
                f()


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_tracing_is_refused():
    x, wg, wu, wd, _ = gated_inputs(6, 8, 16, torch.float32)
    rng, idx = torch.tensor([3, 4], device=DEV), torch.arange(6, device=DEV)
    for f in (lambda t: ops().gated_mlp_rows(t, wg, wu, wd), lambda t: ops().embedding_rows(idx, t), lambda t: ops().dropout_rows(t, 0.5, rng)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, (x,))


# ------------------------------------------------------------------------------------------------ operands that are not finite
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,D,F", [(40, 64, 100), (40, 64, 104), (300, 264, 130), (300, 1000, 130), (65, 1024, 77), (2100, 33, 250)])
def test_an_infinity_is_what_the_definition_makes_of_it(M, D, F, dtype):
    """Positive operands, one infinite element of x and one of the incoming gradient: their rows' results are infinite, not NaN, whatever hidden % 8 is (the
    columns that fill the last group of eight are multiplied by zeros)."""
    x, wg, wu, wd, gy = (t.abs() + 2.0 ** -6 for t in gated_inputs(M, D, F, dtype))
    for t in (x, wg, wu, wd, gy):
        t[t > 4] = 4
    scale = 2.0 ** -8
    x, gy = x * scale, gy * scale              # (finite results stay below 65 504)
    bad_x, bad_g = M // 2, M - 1
    x[bad_x, D - 1] = float("inf")
    gy[bad_g, 0] = float("inf")
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    y = ops().gated_mlp_rows(*leaves, activation="relu")
    got = [y.detach(), *torch.autograd.grad(y, leaves, gy)]
    ref = [t.double().clone().requires_grad_() for t in (x, wg, wu, wd)]
    z = (torch.relu(ref[0] @ ref[1].t()) * (ref[0] @ ref[2].t())) @ ref[3].t()
    want = [z.detach(), *torch.autograd.grad(z, ref, gy.double())]
    for a, b, what in zip(got, want, ("y", "gx", "gw_gate", "gw_up", "gw_down")):
        same = bool((torch.isinf(a) == torch.isinf(b)).all()) and bool((torch.isnan(a) == torch.isnan(b)).all())
        assert same, what
    assert bool(torch.isinf(y[bad_x]).all()) and bool(torch.isinf(got[1][bad_g]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("where", ["x and gradient", "w_gate", "w_up", "w_down"])
@pytest.mark.parametrize("M,D,F", [(1, 1, 1), (5, 24, 13), (20, 100, 300), (70, 24, 9), (70, 800, 1), (70, 1024, 2), (1, 2040, 300), (20000, 16, 100), (4001, 33, 60)])
def test_an_infinity_beside_two_planes(M, D, F, where, dtype):
    """Few results: H, gg and gu in two planes, the lower of which is any small number, zero among them, where the definition has one finite factor."""
    x, wg, wu, wd, gy = (t.abs().clamp(2.0 ** -6, 4) for t in gated_inputs(M, D, F, dtype))
    x, gy = x * 2.0 ** -8, gy * 2.0 ** -8
    if where == "x and gradient":
        x[M // 2, D - 1] = float("inf")
        gy[M - 1, 0] = float("inf")
    else:
        t = {"w_gate": wg, "w_up": wu, "w_down": wd}[where]
        t[t.shape[0] // 2, t.shape[1] // 3] = float("inf")
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    y = ops().gated_mlp_rows(*leaves, activation="relu")
    got = [y.detach(), *torch.autograd.grad(y, leaves, gy)]
    ref = [t.double().clone().requires_grad_() for t in (x, wg, wu, wd)]
    z = (torch.relu(ref[0] @ ref[1].t()) * (ref[0] @ ref[2].t())) @ ref[3].t()
    want = [z.detach(), *torch.autograd.grad(z, ref, gy.double())]
    for a, b, what in zip(got, want, ("y", "gx", "gw_gate", "gw_up", "gw_down")):
        same = bool((torch.isinf(a) == torch.isinf(b)).all()) and bool((torch.isnan(a) == torch.isnan(b)).all())
        assert same, what


# ------------------------------------------------------------------------------------------------ results written in place
@pytest.mark.parametrize("lead", [(6,), (2, 3), (1, 6, 1), ()])
def test_results_can_be_written_in_place(lead):
    """The result belongs to the caller: writing it in place is as good as writing a copy, with any number of leading dims."""
    rows = 1
    for n in lead:
        rows *= n
    x, wg, wu, wd, gy = gated_inputs(rows, 8, 16, torch.float32)
    table, idx, rng = torch.randn(9, 8, device=DEV), (torch.arange(rows, device=DEV) * 5 % 9).view(lead), torch.tensor([7, 1], device=DEV)
    x, gy = x.view(*lead, 8), gy.view(*lead, 8)
    calls = ((lambda t: ops().gated_mlp_rows(t, wg, wu, wd), x), (lambda t: ops().dropout_rows(t, 0.5, rng), x), (lambda t: ops().dropout_rows(t, 0.5, rng, residual=x), x),
             (lambda t: ops().embedding_rows(idx, t), table))
    for f, t in calls:
        leaf = t.clone().requires_grad_()
        want = f(leaf) * 3 + x
        want_grad, = torch.autograd.grad(want, leaf, gy)
        y = f(leaf)
        y.mul_(3).add_(x)
        grad, = torch.autograd.grad(y, leaf, gy)
        assert torch.equal(y, want) and torch.equal(grad, want_grad)


# ------------------------------------------------------------------------------------------------ lazily negated operands
@pytest.mark.parametrize("lazy", [lambda t: torch.complex(torch.zeros_like(t), -t).conj().imag, lambda t: torch._neg_view(-t)], ids=["conjugate", "contiguous"])
@pytest.mark.parametrize("D", [1, 8])
def test_lazily_negated_operands(lazy, D):
    """The imaginary part of a conjugate is a view whose elements are negated when they are read."""
    x, wg, wu, wd, gy = gated_inputs(6, D, 7, torch.float32)
    table, rng, idx = gated_inputs(6, D, 7, torch.float32, seed=1)[0], torch.tensor([2, 9], device=DEV), torch.tensor([0, 3, 3, 1, 2, 5], device=DEV)
    assert lazy(x).is_neg() and torch.equal(lazy(x), x)
    f, args = ops().gated_mlp_rows, [x, wg, wu, wd]
    for i in range(4):
        assert torch.equal(f(*[lazy(t) if k == i else t for k, t in enumerate(args)]), f(*args)), i
    assert torch.equal(ops().dropout_rows(lazy(x), 0.25, rng, residual=lazy(gy)), ops().dropout_rows(x, 0.25, rng, residual=gy))
    assert torch.equal(ops().embedding_rows(idx, lazy(table)), table[idx])
    assert torch.equal(ops().embedding_rows(torch._neg_view(-idx), table), table[idx])
    with pytest.raises(RuntimeError, match="rng"):
        ops().dropout_rows(x, 0.25, torch._neg_view(-rng))
    for g, leaf in ((lambda t: f(t, wg, wu, wd), x), (lambda t: ops().dropout_rows(t, 0.25, rng), x), (lambda t: ops().embedding_rows(idx, t), table)):
        leaf = leaf.clone().requires_grad_()
        want, = torch.autograd.grad(g(leaf), leaf, gy)
        got, = torch.autograd.grad(g(leaf), leaf, lazy(gy))
        assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------ two planes
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [2, 20, 40, 100])
@pytest.mark.parametrize("D", [8, 100, 1000])
def test_the_lower_plane_is_what_the_upper_one_leaves(D, M, dtype):
    """Few results, H, gg and gu in two planes.  Gate and up projection are 1 + 2^-12 in one row and 1 in another: H there is (1 + 2^-12)^2, which as a float lies
    half way between two neighbours in float16 and unrounded does not, and both values must come from one rounding of it."""
    F = 2
    x, wg, wd, gy = (torch.zeros(s, dtype=dtype, device=DEV) for s in ((M, D), (F, D), (D, F), (M, D)))
    x[:, 0] = 1
    x[M - 1, 1] = wg[:, 1].fill_(2.0 ** -6)[0]
    wg[:, 0] = 1
    wd[0] = 1
    gy[M - 1, 0], gy[0, 0] = 1, -1
    leaves = [t.clone().requires_grad_() for t in (x, wg, wg, wd)]
    for act in ("relu", "silu", "gelu"):
        gx, gwg, gwu, gwd = torch.autograd.grad(ops().gated_mlp_rows(*leaves, activation=act), leaves, gy)
        ref = [t.detach().double().requires_grad_() for t in leaves]
        fn = dict(relu=torch.relu, silu=torch.nn.functional.silu, gelu=torch.nn.functional.gelu)[act]
        want = torch.autograd.grad((fn(ref[0] @ ref[1].t()) * (ref[0] @ ref[2].t())) @ ref[3].t(), ref, gy.double())
        e = torch.finfo(dtype).eps / 2
        # each term, at most 1.3, is off by the square of the rounding and by the activation's fp32 arithmetic (8 2^-24 of 1 + |g|); their difference by a rounding too
        for got, exact, what in ((gwg, want[1], "gw_gate"), (gwu, want[2], "gw_up"), (gwd.t(), want[3].t(), "gw_down")):
            err = (got[:, 0].double() - exact[:, 0]).abs().max()
            assert float(err) <= 2 * 1.3 * (e * e + 20 * 2.0 ** -24) + e * float(exact[:, 0].abs().max()), (act, what)


# ------------------------------------------------------------------------------------------------ what is rounded, and how often
H32 = 2.0 ** -24


def block_bounds(x, wg, wu, wd, act, gy, planes):
    """(value in 64 bits, bound) of y, gx, gWg, gWu, gWd, in 2-D operands: fp32 sums (k 2^-24 of the sum of magnitudes, counted twice for the matrix instruction's own
    order and roundings), H, gg and gu rounded once in `planes` values of the type (3: fp32's planes, to 2^-24), G and U not at all, each result rounded once."""
    t = x.dtype
    e, under = torch.finfo(t).eps / 2, {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[t]
    e_in = H32 if planes == 3 else e ** planes         # (a second value holds what the first left, to half a step of that)
    x, wg, wu, wd, gy = (v.detach().double() for v in (x, wg, wu, wd, gy))
    M, D, F = x.shape[0], x.shape[1], wg.shape[0]

    def mm(a, da, b, k):                # of a known to da, b exact
        return a @ b, da @ b.abs() + (k + 16) * 2 * H32 * ((a.abs() + da) @ b.abs())

    def times(*parts):                  # product of (value, error) pairs in fp32
        val, err = parts[0]
        for v, d in parts[1:]:
            val, err = val * v, err * (v.abs() + d) + val.abs() * d
        return val, err + 3 * H32 * (val.abs() + err)

    def rounded(v, d, step):
        return v, d + step * (v.abs() + d) + under
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    g, u = mm(x, zero.expand_as(x), wg.t(), D), mm(x, zero.expand_as(x), wu.t(), D)
    leaf = g[0].clone().requires_grad_()
    fn = dict(silu=torch.nn.functional.silu, relu=torch.relu)[act]
    value = fn(leaf)
    slope, = torch.autograd.grad(value.sum(), leaf)
    own = 8 * H32 * (1 + g[0].abs())    # the activation's fp32 arithmetic
    flips = (g[0].abs() <= g[1]).double() if act == "relu" else 0.0
    a = value.detach(), dict(silu=1.1, relu=1.0)[act] * g[1] + own
    s = slope, dict(silu=0.5, relu=0.0)[act] * g[1] + own + flips
    h = rounded(*times(a, u), e_in)
    gh = mm(gy, zero.expand_as(gy), wd, D)
    gg, gu = rounded(*times(gh, u, s), e_in), rounded(*times(gh, a), e_in)
    gx1, gx2 = mm(*gg, wg, 2 * F), mm(*gu, wu, 2 * F)
    gwd, dgwd = mm(h[0].t(), h[1].t(), gy, M)
    return [rounded(*p, e) for p in (mm(*h, wd.t(), F), (gx1[0] + gx2[0], gx1[1] + gx2[1]), mm(gg[0].t(), gg[1].t(), x, M), mm(gu[0].t(), gu[1].t(), x, M), (gwd.t(), dgwd.t()))]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("planes", [None, 1, 2])
@pytest.mark.parametrize("M,D,F", [(1, 8, 8), (1, 2048, 24), (1, 2049, 24), (13, 250, 170), (31, 264, 40), (33, 130, 65), (70, 72, 130), (300, 264, 157), (70, 1000, 300), (2500, 96, 777), (1500, 1001, 65)])
def test_planes_hold_what_they_say(M, D, F, planes, dtype):
    if dtype == torch.float32 and planes is not None:
        with pytest.raises(RuntimeError, match="16-bit types"):
            ops().gated_mlp_rows(*gated_inputs(M, D, F, dtype)[:4], planes=planes)
        return
    act = "relu" if (M + D) % 2 else "silu"
    x, wg, wu, wd, gy = gated_inputs(M, D, F, dtype, seed=3)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    y = ops().gated_mlp_rows(*leaves, activation=act, planes=planes)
    with torch.no_grad():
        assert torch.equal(ops().gated_mlp_rows(x, wg, wu, wd, activation=act, planes=planes), y)
    held = 3 if dtype == torch.float32 else planes or (2 if min(M, F) * D <= 2048 else 1)
    for got, (want, bound), what in zip((y, *torch.autograd.grad(y, leaves, gy)), block_bounds(x, wg, wu, wd, act, gy, held), ("y", "gx", "gw_gate", "gw_up", "gw_down")):
        bad = (got.double() - want).abs() > bound
        assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()}, by at most {float(((got.double() - want).abs() / bound).max()):.2f} bounds"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [2, 40, 300])
@pytest.mark.parametrize("D", [8, 1000, 1024])
def test_projections_are_not_rounded(D, M, dtype):
    """G and U are 1 + 2^-12 in one row and 1 in another, both 1 in a 16-bit type: what a difference of the rows leaves shows whether they were kept."""
    F = 16
    x, wg, wd, gy = (torch.zeros(s, dtype=dtype, device=DEV) for s in ((M, D), (F, D), (D, F), (M, D)))
    x[:, 0] = 1
    x[M - 1, 1] = wg[:, 1].fill_(2.0 ** -6)[0]
    wg[:, 0] = 1
    wd[0] = 1
    gy[M - 1, 0], gy[0, 0] = 1, -1
    leaves = [t.clone().requires_grad_() for t in (x, wg, wg, wd)]
    y = ops().gated_mlp_rows(*leaves, activation="relu", planes=2)
    gx, gwg, gwu, gwd = torch.autograd.grad(y, leaves, gy)
    assert bool((gwg[:, 0] == 2.0 ** -12).all()) and bool((gwu[:, 0] == 2.0 ** -12).all())
    assert bool((gwd[0] == 2.0 ** -11).all())                      # (1 + 2^-12)^2 - 1, rounded to the type
    # and in one plane, as the docstring says, they do not show
    one = torch.autograd.grad(ops().gated_mlp_rows(*leaves, activation="relu", planes=1), leaves, gy)
    assert not bool(one[1][:, 0].any()) and not bool(one[2][:, 0].any())


def test_planes_of_the_module():
    x, wg, wu, wd, _ = gated_inputs(200, 64, 96, torch.bfloat16)
    mods = [ops().GatedMLP(64, 96, "silu", planes=p).to(DEV, torch.bfloat16) for p in (None, 1, 2)]
    for m in mods:
        with torch.no_grad():
            for p, w in ((m.w_gate, wg), (m.w_up, wu), (m.w_down, wd)):
                p.copy_(w)
    y = [m(x) for m in mods]
    assert torch.equal(y[0], y[1]) and not torch.equal(y[1], y[2])
    assert all(torch.equal(y[k], ops().gated_mlp_rows(x, wg, wu, wd, "silu", planes=p)) for k, p in enumerate((None, 1, 2)))


# ------------------------------------------------------------------------------------------------ what the backward pass reads
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,D,F", [(6, 8, 16), (70, 40, 100), (300, 1000, 130)])
def test_a_kept_graph_gives_its_gradients_again(M, D, F, dtype):
    """Nothing that the forward pass has kept is written by a backward pass; and it may be kept elsewhere in the meantime."""
    x, wg, wu, wd, gy = gated_inputs(M, D, F, dtype)
    wide = torch.cat([x, x], 1)[:, 1:D + 1]                                  # (rows of a wider tensor: another row distance when it comes back)
    leaves = [t.detach().requires_grad_() for t in (wide, wg.t().contiguous().t(), wu, wd)]
    rng, idx, table = torch.tensor([3, 4], device=DEV), torch.arange(M, device=DEV) % 5, x[:5].clone().requires_grad_()

    def run():
        rows = ops().dropout_rows(leaves[0], 0.2, rng, residual=ops().embedding_rows(idx, table))
        return ops().gated_mlp_rows(rows, *leaves[1:])
    y = run()
    first = torch.autograd.grad(y, [*leaves, table], gy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, [*leaves, table], gy)))
    with torch.autograd.graph.save_on_cpu():
        y = run()
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, [*leaves, table], gy)))
