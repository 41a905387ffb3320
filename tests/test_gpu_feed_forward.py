"""The feed-forward operators (fpn.feed_forward) against their formulas in float64 on the same inputs.

Tolerance.  With u the type's half step (2^-24, 2^-11, 2^-8) an output has one rounding of its own; what lies before
it adds
  * fp32 accumulation of K products: at most K 2^-24 of the sum of their magnitudes, in practice its square root;
    taken as 2^-24 (4 + sqrt K) of the root of the sum of the squared products, times the largest of the output's
    values in units of its standard deviation (6);
  * in the backward pass of 16-bit types the rounded dpre (dg, du), a relative half step on one factor of every product:
    u of the same root (pre-activations are kept in fp32);
  * in gated_feed_forward h likewise: sqrt(2) u.
  * in the backward pass the forward sums' own error: a pre-activation is off by delta = 6 2^-24 (4 + sqrt cin) S(x, w)
    + u |pre|; slopes move by at most delta (curvature <= 1), values by 1.13 delta, and the products' terms with them
    (`moved`).
All of them are measured against the root of the sum of squares S = sqrt(a^2 @ b^2) of the product's terms (for a
column sum, of the summed values): |got - want| <= u |want| + 6 c S with c as above.  An activation's slope is at most
1.13 and its curvature at most 1 in magnitude, so a half step on a pre-activation v changes the activation by 1.13 u |v|.
"""
import contextlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": (torch.float32, 2.0 ** -24), "bf16": (torch.bfloat16, 2.0 ** -8), "f16": (torch.float16, 2.0 ** -11)}
ACTS = [None, "relu", "silu", "sigmoid", "gelu", "gelu_tanh"]


def f64(t):
    return t.detach().double().cpu()


def act64(v, act):
    """(value, derivative) in float64"""
    v = v.clone().requires_grad_()
    y = {None: lambda: v * 1, "relu": lambda: torch.relu(v), "silu": lambda: v / (1 + torch.exp(-v)),
         "sigmoid": lambda: 1 / (1 + torch.exp(-v)), "gelu": lambda: v * 0.5 * torch.special.erfc(-v / 2 ** 0.5),
         "gelu_tanh": lambda: 0.5 * v * (1 + torch.tanh((2 / np.pi) ** 0.5 * (v + 0.044715 * v ** 3)))}[act]()
    (d,) = torch.autograd.grad(y.sum(), v)
    return y.detach(), d


def make(device, dtype, rows, cin, cout, seed=0, cols=False, hidden=None):
    g = torch.Generator().manual_seed(seed + 7 * rows + 131 * cin + cout)
    n = hidden or cout

    def r(*shape, s=1.0):
        return (torch.randn(shape, generator=g) * s).to(dtype).to(device)

    def w(k, m):
        return r(m, k, s=k ** -0.5).t() if cols else r(k, m, s=k ** -0.5)
    return {"x": r(rows, cin), "w": w(cin, cout), "wg": w(cin, n), "wu": w(cin, n), "wd": w(n, cout), "b": r(cout, s=0.3),
            "bg": r(n, s=0.3), "bu": r(n, s=0.3), "res": r(rows, cout), "dy": r(rows, cout), "dh": r(rows, n)}


def check(got, want, s, k, u, halves=0.0, what="", moved=0.0):
    """|got - want| <= u |want| + 6 (2^-24 (4 + sqrt k) + halves u) s, and what fp16 loses below its normal numbers"""
    got = f64(got)
    assert got.shape == want.shape, what
    c = 2.0 ** -24 * (4 + k ** 0.5) + (halves * u if u > 2.0 ** -20 else 2.0 ** -24 * halves)
    # fp16's subnormal numbers lie 2^-24 apart, so that a rounding below 2^-14 errs by up to 2^-25 whatever the value: once
    # in the result, and where d was rounded (halves) once in each of the k terms, times a factor of unit spread
    tiny = 2.0 ** -25 if u == 2.0 ** -11 else 0.0
    tol = u * want.abs() + 6 * c * s + 6 * moved + tiny * (1 + (6 * k ** 0.5 if halves else 0))
    off = (got - want).abs()
    assert torch.isfinite(got).all(), what
    assert (off <= tol).all(), "%s: %.3g of the tolerance" % (what, float((off / tol).max()))


def root(a, b):
    return (a.square() @ b.square()).sqrt()


def sum_error(a, b, k):
    return 6 * 2.0 ** -24 * (4 + k ** 0.5) * root(a, b)


def dense_case(device, t, rows, cin, cout, act, bias, residual, cols, seed=0):
    from fpn import feed_forward as F
    dtype, u = TYPES[t]
    d = make(device, dtype, rows, cin, cout, seed, cols)
    b, r = d["b"] if bias else None, d["res"] if residual else None
    y, pre = F.dense(d["x"], d["w"], b, act, r, keep=True)
    y2 = F.dense(d["x"], d["w"], b, act, r)
    assert torch.equal(y, y2)
    x, w, dy = f64(d["x"]), f64(d["w"]), f64(d["dy"])
    p = x @ w + (f64(b) if bias else 0)
    a, slope = act64(p, act)
    want = a + (f64(r) if residual else 0)
    s = root(x, w) + a.abs() + want.abs()
    check(y, want, 1.2 * s, cin, u, what="y")
    if act:
        check(pre, p, s + p.abs(), cin, 2.0 ** -24, what="pre")
    dx, dw, db = F.dense_grad(d["dy"], d["x"], d["w"], pre, act, bias=True)
    if act == "relu":                                     # the step of the derivative goes by the kernel's own sums
        slope = (f64(pre) > 0).double()
    e = dy * slope
    spread = dy.abs() * (1.2 + p.abs())                   # what a half step of pre and of e is relative to
    off = dy.abs() * sum_error(x, w, cin) if act else 0 * dy
    check(dx, e @ w.t(), root(spread, w.t()), cout, u, 1 if act else 0, "dx", root(off, w.t()))
    check(dw, x.t() @ e, root(x.t(), spread), rows, u, 1 if act else 0, "dw", root(x.t(), off))
    check(db, e.sum(0), spread.square().sum(0).sqrt(), rows, u, 1 if act else 0, "db", off.square().sum(0).sqrt())


SIZES = [(1, 1, 1), (1, 5, 3), (2, 3, 7), (5, 4, 8), (1, 1027, 512), (7, 64, 64), (33, 63, 65), (64, 128, 128), (65, 129, 127),
         (130, 515, 259), (300, 200, 100), (1000, 3, 64), (515, 1091, 2), (129, 640, 264)]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows,cin,cout", SIZES)
def test_dense(device, t, rows, cin, cout):
    i = SIZES.index((rows, cin, cout))
    for j, cols in enumerate((False, True)):
        dense_case(device, t, rows, cin, cout, ACTS[(i + 3 * j) % 6], bias=(i + j) % 3 != 0, residual=(i + j) % 2 == 0, cols=cols)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("act", ACTS)
def test_dense_activations(device, t, act):
    dense_case(device, t, 96, 72, 40, act, True, True, False, seed=5)


def gated_case(device, t, rows, cin, cout, act, bias, cols, seed=0):
    from fpn import feed_forward as F
    dtype, u = TYPES[t]
    d = make(device, dtype, rows, cin, cout, seed, cols)
    bg, bu = (d["bg"], d["bu"]) if bias else (None, None)
    h, gate, up = F.gated(d["x"], d["wg"], d["wu"], bg, bu, act, keep=True)
    assert torch.equal(h, F.gated(d["x"], d["wg"], d["wu"], bg, bu, act))
    x, wg, wu, dh = f64(d["x"]), f64(d["wg"]), f64(d["wu"]), f64(d["dh"])
    pg, pu = x @ wg + (f64(bg) if bias else 0), x @ wu + (f64(bu) if bias else 0)
    a, slope = act64(pg, act)
    sg, su = root(x, wg) + pg.abs(), root(x, wu) + pu.abs()
    check(gate, pg, sg, cin, 2.0 ** -24, what="gate")
    check(up, pu, su, cin, 2.0 ** -24, what="up")
    check(h, a * pu, 1.2 * sg * pu.abs() + su * a.abs() + (a * pu).abs(), cin, u, what="h")
    dx, dwg, dwu, dbg, dbu = F.gated_grad(d["dh"], d["x"], d["wg"], d["wu"], gate, up, act, bias=True)
    if act == "relu":
        slope = (f64(gate) > 0).double()
    eg, eu = dh * pu * slope, dh * a
    tg, tu = dh.abs() * (pu.abs() + 2.0 ** -24 * su) * (1.2 + pg.abs()), dh.abs() * (1.2 * pg.abs() + a.abs())
    og = dh.abs() * (1.13 * sum_error(x, wu, cin) + pu.abs() * sum_error(x, wg, cin))
    ou = dh.abs() * 1.13 * sum_error(x, wg, cin)
    check(dx, eg @ wg.t() + eu @ wu.t(), (root(tg, wg.t()).square() + root(tu, wu.t()).square()).sqrt(), 2 * cout, u, 1, "dx",
          root(og, wg.t()) + root(ou, wu.t()))
    check(dwg, x.t() @ eg, root(x.t(), tg), rows, u, 1, "dwg", root(x.t(), og))
    check(dwu, x.t() @ eu, root(x.t(), tu), rows, u, 1, "dwu", root(x.t(), ou))
    check(dbg, eg.sum(0), tg.square().sum(0).sqrt(), rows, u, 1, "dbg", og.square().sum(0).sqrt())
    check(dbu, eu.sum(0), tu.square().sum(0).sqrt(), rows, u, 1, "dbu", ou.square().sum(0).sqrt())


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows,cin,cout", SIZES)
def test_gated(device, t, rows, cin, cout):
    i = SIZES.index((rows, cin, cout))
    for j, cols in enumerate((False, True)):
        gated_case(device, t, rows, cin, cout, ACTS[(i + 3 * j + 1) % 6], bias=(i + j) % 2 != 0, cols=cols)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("act", ACTS)
def test_gated_activations(device, t, act):
    gated_case(device, t, 96, 72, 40, act, True, False, seed=5)


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_exact_on_small_integers(device, t):
    """Small whole numbers: every product and sum is exact in fp32 and in the results, so layouts, orders, splits and
    ends are checked bit for bit, at sizes on every side of the tiles and at every way of cutting k."""
    from fpn import feed_forward as F
    dtype, _ = TYPES[t]
    g = torch.Generator().manual_seed(1)
    for rows, cin, cout in [(1, 2048, 256), (16, 4096, 130), (17, 4100, 96), (255, 257, 300), (256, 512, 256), (700, 96, 1000),
                            (40000, 70, 33), (20000, 64, 128), (2048, 130, 2049), (1536, 2048, 1024)]:
        x = torch.randint(-1, 2, (rows, cin), generator=g).to(dtype)
        w = torch.randint(-1, 2, (cin, cout), generator=g).to(dtype)
        x, w = x.to(device), w.to(device)
        # (few nonzero weights: sums stay under bf16's 256)
        keep = (torch.rand((cin, cout), generator=g) < 30.0 / cin).to(dtype).to(device)
        w = w * keep
        want = (x.double() @ w.double()).to(dtype)
        for ww in (w, w.t().contiguous().t()):
            assert torch.equal(F.dense(x, ww), want), (rows, cin, cout)
            assert torch.equal(F.gated(x, ww, ww, activation=None), (want.double() ** 2).to(dtype)), (rows, cin, cout)
        dy = (torch.randint(-1, 2, (rows, cout), generator=g) * (torch.rand((rows, cout), generator=g) < min(1.0, 20.0 / max(rows, cout)))).to(dtype).to(device)
        for ww in (w, w.t().contiguous().t()):
            dx, dw, db = F.dense_grad(dy, x, ww, bias=True)
            assert dw.stride() == ww.stride()
            assert torch.equal(dx, (dy.double() @ w.double().t()).to(dtype)), (rows, cin, cout)
            assert torch.equal(dw, (x.double().t() @ dy.double()).to(dtype)), (rows, cin, cout)
            assert torch.equal(db, dy.double().sum(0).to(dtype)), (rows, cin, cout)


@pytest.mark.parametrize("t", list(TYPES))
def test_strided_operands_and_untouched_memory(device, t):
    """Column slices of wider buffers at odd offsets: read and written in place, nothing beside them touched; a
    broadcast x and residual row; out = residual."""
    from fpn import feed_forward as F
    dtype, _ = TYPES[t]
    g = torch.Generator().manual_seed(2)
    rows, cin, cout = 77, 131, 67
    ints = lambda *s: torch.randint(-2, 3, s, generator=g).to(dtype).to(device)      # noqa: E731
    wide = torch.full((rows, 400), float("nan"), dtype=dtype, device=device)
    wide[:, 3:3 + cin] = ints(rows, cin)
    x, out = wide[:, 3:3 + cin], wide[:, 201:201 + cout]
    wboth = torch.full((cin, 301), float("nan"), dtype=dtype, device=device)
    wboth[:, 1:1 + cout] = ints(cin, cout)
    wboth[:, 101:101 + cout] = ints(cin, cout)
    w, w2 = wboth[:, 1:1 + cout], wboth[:, 101:101 + cout]
    b, res = ints(cout), ints(rows, cout)
    before = wide.clone()
    y = F.dense(x, w, b, "relu", res, out=out)
    assert y.data_ptr() == out.data_ptr()
    want = (torch.relu(x.double() @ w.double() + b.double()) + res.double()).to(dtype)
    assert torch.equal(out, want)
    mask = torch.ones(400, dtype=torch.bool, device=device)
    mask[201:201 + cout] = False
    assert torch.equal(wide[:, mask].nan_to_num(7.0), before[:, mask].nan_to_num(7.0))
    F.gated(x, w, w2, activation="relu", out=out)
    assert torch.equal(out, (torch.relu(x.double() @ w.double()) * (x.double() @ w2.double())).to(dtype))
    assert torch.equal(wide[:, mask].nan_to_num(7.0), before[:, mask].nan_to_num(7.0))
    row = ints(1, cin)
    assert torch.equal(F.dense(row.expand(rows, cin), w, residual=b.expand(rows, cout)),
                       (row.double() @ w.double() + b.double()).to(dtype).expand(rows, cout))
    y = res.clone()
    F.dense(x, w, residual=y, out=y)
    assert torch.equal(y, (x.double() @ w.double() + res.double()).to(dtype))


@pytest.mark.parametrize("t", list(TYPES))
def test_not_finite_values_stay_in_their_rows(device, t):
    """A NaN or an infinity in a row of x reaches that row's results and no other; one in a column of w that column;
    neither leaks through the ends of tiles (rows, widths and k off every tile size)."""
    from fpn import feed_forward as F
    dtype, _ = TYPES[t]
    g = torch.Generator().manual_seed(3)
    rows, cin, cout = 70, 75, 69
    x = torch.randn((rows, cin), generator=g).to(dtype).to(device)
    w = torch.randn((cin, cout), generator=g).to(dtype).to(device)
    x[rows - 1, cin - 1], x[3, 0] = float("nan"), float("inf")
    w[cin - 1, cout - 1] = float("nan")
    for act in ACTS:
        for y in (F.dense(x, w, activation=act), F.gated(x, w, w, activation=act), F.dense(x, w.t().contiguous().t(), activation=act)):
            want = (x.float() @ w.float())
            bad = ~torch.isfinite(want)
            assert torch.isfinite(y[~bad]).all()
            assert torch.isnan(y[rows - 1]).all() and torch.isnan(y[:, cout - 1]).all()
            if act is None or act == "relu":
                assert (y[3, :-1] == (want[3, :-1] if act is None else torch.relu(want[3, :-1]))).all() or y.isnan().any()


@pytest.mark.parametrize("t", list(TYPES))
def test_far_tails_of_the_activations(device, t):
    """Pre-activations from the type's largest value down: values and slopes stay finite wherever the formula's are."""
    from fpn import feed_forward as F
    dtype, u = TYPES[t]
    top = torch.finfo(dtype).max
    v = torch.tensor([[0.0, -0.0, 1e-3, -1e-3, 1, -1, 3, -3, 6, -6, 12, -12, 80, -80, 200, -200, 3e4, -3e4, top / 4, -top / 4]],
                     dtype=torch.float64).to(dtype).to(device)
    n = v.shape[1]
    one = torch.zeros((1, 1), dtype=dtype, device=device)
    w = torch.zeros((1, n), dtype=dtype, device=device)
    for act in ACTS[1:]:
        y, pre = F.dense(one, w, v[0], act, keep=True)
        assert torch.equal(pre.abs(), v.abs())
        p = f64(v).clone().requires_grad_()
        want, slope = act64(p.detach(), act)
        z = p.detach()
        if act == "silu":                                   # (the oracle's own forms overflow far out)
            s = torch.sigmoid(z)
            want, slope = z * s, s * (1 + z * torch.sigmoid(-z))
        if act == "sigmoid":
            slope = torch.sigmoid(z) * torch.sigmoid(-z)
        if act == "gelu_tanh":
            far = z.abs() > 50
            want = torch.where(far, torch.relu(z), want)
            slope = torch.where(far, (z > 0).double(), slope)
        if act == "relu":
            slope = (z > 0).double()
        tiny = torch.finfo(dtype).tiny
        off = (f64(y) - want).abs()
        # the tail of v Phi(v) falls as exp(-v^2 / 2): v / sqrt 2, its square and the constant are each rounded to fp32,
        # a relative 2^-24 in a quantity whose logarithm's derivative is up to v^2 - together 3 v^2 2^-24
        tail = torch.where(z.abs() < 40, z * z, 0 * z) * 3 * 2.0 ** -24
        assert (off <= (u + 4e-6 + tail) * want.abs() + tiny).all(), (act, y, want)
        dy = torch.ones((1, n), dtype=dtype, device=device)
        _, _, db = F.dense_grad(dy, one, w, pre, act, bias=True, need_x=False, need_w=False)
        off = (f64(db)[None] - slope).abs()
        assert (off <= u * slope.abs() + 4e-6 * (1 + slope.abs())).all(), (act, db, slope)


def test_no_rows(device):
    from fpn import feed_forward as F
    for t in TYPES:
        dtype = TYPES[t][0]
        x, w = torch.empty((0, 40), dtype=dtype, device=device), torch.ones((40, 24), dtype=dtype, device=device)
        y, pre = F.dense(x, w, activation="silu", keep=True)
        assert y.shape == (0, 24)
        dx, dw, db = F.dense_grad(y, x, w, pre, "silu", bias=True)
        assert dx.shape == (0, 40) and not dw.any() and not db.any()
        h, g, u = F.gated(x, w, w, keep=True)
        dx, a, b, c, d = F.gated_grad(h, x, w, w, g, u, bias=True)
        assert dx.shape == (0, 40) and not a.any() and not b.any() and not c.any() and not d.any()


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows,cin,hidden", [(1, 64, 256), (3, 130, 67), (200, 96, 256), (333, 160, 328), (700, 64, 2048), (130, 72, 24)])
def test_block_runs_together_and_its_gradients(device, t, rows, cin, hidden):
    """gated_feed_forward with its residual through autograd, against the formula's gradients in float64."""
    from fpn import feed_forward as F
    dtype, u = TYPES[t]
    d = make(device, dtype, rows, cin, cin, seed=3, hidden=hidden)
    names = ["x", "wg", "wu", "wd", "bg", "bu", "b", "res"]
    leaves = [d[k].clone().requires_grad_() for k in names]
    x, wg, wu, wd, bg, bu, bd, res = leaves
    y = F.gated_feed_forward(x, wg, wu, wd, bg, bu, bd, "silu", res)
    with torch.no_grad():
        assert torch.equal(y, F.gated_feed_forward(x, wg, wu, wd, bg, bu, bd, "silu", res))
    grads = torch.autograd.grad(y, leaves, d["dy"])
    l64 = [f64(t_).requires_grad_() for t_ in leaves]
    X, WG, WU, WD, BG, BU, BD, RES = l64
    pg, pu = X @ WG + BG, X @ WU + BU
    h = torch.nn.functional.silu(pg) * pu
    Y = h @ WD + BD + RES
    want = torch.autograd.grad(Y, l64, f64(d["dy"]))
    s = root(h.detach(), WD.detach()) + root(X.detach(), WG.detach()).mean() + Y.detach().abs()
    check(y, Y.detach(), 2 * s, hidden, u, 1.5, "y")
    for name, g, w_ in zip(names, grads, want):
        scale = w_.square().mean().sqrt()                  # (every gradient's terms have about its own spread)
        check(g, w_, 2 * (w_.abs() + scale), max(rows, hidden, cin), u, 1.5, "d" + name)


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cin,hidden,cols", [(5, 24, 40, False), (260, 96, 520, False), (260, 96, 520, True), (1100, 64, 1024, False),
                                                  (257, 33, 70, True)])
def test_gradient_through_the_down_projection(device, t, rows, cin, hidden, cols):
    """gated_grad with w_down, for the kernel that makes dg and du in the product's epilogue and for the one that does not:
    against gated_grad on dh = dy w_down^T formed in float64 (rounded once, which is what the call saves: a relative u on
    every term)."""
    from fpn import feed_forward as F
    dtype, u = TYPES[t]
    d = make(device, dtype, rows, cin, cin, seed=8, hidden=hidden, cols=cols)
    for act in ("silu", "gelu_tanh"):
        _, gate, up = F.gated(d["x"], d["wg"], d["wu"], d["bg"], d["bu"], act, keep=True)
        got = F.gated_grad(d["dy"], d["x"], d["wg"], d["wu"], gate, up, act, bias=True, w_down=d["wd"])
        dh = (d["dy"].double() @ d["wd"].double().t()).to(dtype)
        want = F.gated_grad(dh, d["x"], d["wg"], d["wu"], gate, up, act, bias=True)
        assert all(torch.equal(a, b) for a, b in zip(got, F.gated_grad(d["dy"], d["x"], d["wg"], d["wu"], gate, up, act, bias=True, w_down=d["wd"])))
        for name, a, b in zip(("dx", "dwg", "dwu", "dbg", "dbu"), got, want):
            # both sides round the result (u each) and dg, du (u each); dh's rounding and fp32 sums add u and 2^-24 sqrt k
            off = float((a.double() - b.double()).norm() / b.double().norm())
            assert off <= 5 ** 0.5 * u + 4 * 2.0 ** -24 * max(rows, cin, hidden) ** 0.5, (name, off)


def test_gradients_against_differences(device):
    """The directional derivative of a random functional along a random direction, by central differences of the fp32
    forward pass: the third-order remainder at step 2^-6 and the forward's roundings over the step stay under 2e-3."""
    from fpn import feed_forward as F
    d = make(device, torch.float32, 37, 45, 45, seed=9, hidden=70)
    leaves = [d[k].clone().requires_grad_() for k in ("x", "wg", "wu", "wd", "bg", "bu", "b", "res")]
    g = torch.Generator().manual_seed(10)
    for act in ("silu", "gelu", "gelu_tanh", "sigmoid"):
        def f(ts):
            return F.gated_feed_forward(*ts[:7], act, ts[7])
        y = f(leaves)
        grads = torch.autograd.grad(y, leaves, d["dy"])
        for i, leaf in enumerate(leaves):
            v = torch.randn(leaf.shape, generator=g).to(device)
            v /= v.norm()
            eps = 2.0 ** -6
            with torch.no_grad():
                up = [t + eps * v if j == i else t for j, t in enumerate(leaves)]
                dn = [t - eps * v if j == i else t for j, t in enumerate(leaves)]
                diff = float(((f(up).double() - f(dn).double()) * d["dy"].double()).sum()) / (2 * eps)
            got = float((grads[i].double() * v.double()).sum())
            scale = float(grads[i].double().norm()) / leaf.numel() ** 0.5 + 1e-3
            assert abs(got - diff) <= 2e-3 * max(abs(diff), scale) + 1e-3 * scale * 10, (act, i, got, diff)


def test_shared_leaves_and_partial_gradients(device):
    """The same tensor in two places gets both gradients; only what is asked for is computed."""
    from fpn import feed_forward as F
    g = torch.Generator().manual_seed(11)
    x = torch.randn((9, 16), generator=g).to(device).requires_grad_()
    w = torch.randn((16, 16), generator=g).to(device).requires_grad_()
    y = F.dense(x, w, activation="gelu", residual=x)
    y = F.gated(y, w, w)
    y.sum().backward()                                       # (an expanded gradient comes in)
    X, W = f64(x).requires_grad_(), f64(w).requires_grad_()
    Y = torch.nn.functional.gelu(X @ W) + X
    Y = torch.nn.functional.silu(Y @ W) * (Y @ W)
    Y.sum().backward()
    for a, b in ((x.grad, X.grad), (w.grad, W.grad)):
        assert (f64(a) - b).norm() <= 1e-5 * b.norm()
    frozen = w.detach()
    (dx,) = torch.autograd.grad(F.gated(x, frozen, frozen).sum(), x)
    assert dx.shape == x.shape
    xb = x.detach()[:1].requires_grad_()
    (db,) = torch.autograd.grad(F.dense(xb.expand(9, 16), frozen).sum(), xb)      # a broadcast input
    assert (f64(db) - 9 * f64(frozen).sum(1)).norm() <= 1e-5 * f64(frozen).sum(1).norm() * 9


def test_repeats_bit_for_bit_and_on_another_stream(device):
    """Split sums, column sums: the same bits call after call, on another stream, and between other work."""
    from fpn import feed_forward as F
    d = make(device, torch.bfloat16, 3000, 72, 100, seed=1)
    first = None
    side = torch.cuda.Stream()
    for i in range(4):
        ctx = torch.cuda.stream(side) if i % 2 else contextlib.nullcontext()
        if i % 2:
            side.wait_stream(torch.cuda.current_stream())
        with ctx:
            h, gate, up = F.gated(d["x"], d["wg"], d["wu"], d["bg"], d["bu"], keep=True)
            out = [h] + list(F.gated_grad(d["dh"], d["x"], d["wg"], d["wu"], gate, up, bias=True))
        torch.cuda.synchronize()
        out = [o.cpu() for o in out]
        if first is None:
            first = out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_captured_step_replays(device):
    """A training step with the explicit backward pass in a graph, replayed between eager work (an eager autograd graph
    of the same leaves alive all the while): every replay equals the eager result; two graphs at once have their own
    workspaces; recording through autograd inside a capture is refused."""
    from fpn import feed_forward as F
    d = make(device, torch.bfloat16, 130, 200, 96, seed=4)
    w_leaf = d["wg"].clone().requires_grad_()
    alive = F.dense(d["x"], w_leaf, activation="silu")       # an eager graph of a leaf that the capture reads too

    def step(x, dh, wg, wu):
        h, gate, up = F.gated(x, wg, wu, keep=True)
        return (h,) + F.gated_grad(dh, x, wg, wu, gate, up, bias=True)
    with torch.no_grad():
        step(d["x"], d["dh"], w_leaf, d["wu"])
    torch.cuda.synchronize()
    graphs, outs, xs = [], [], []
    for i in range(2):
        xs.append(d["x"].clone())
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            with torch.no_grad():
                outs.append(step(xs[i], d["dh"], w_leaf, d["wu"]))
        graphs.append(gr)
    gen = torch.Generator().manual_seed(12)
    for r in range(3):
        for x in xs:
            x.copy_(torch.randn(x.shape, generator=gen).to(x.dtype))
        for gr in graphs:
            gr.replay()
        (alive.float().sum() * 0).backward(retain_graph=True)
        with torch.no_grad():
            for x, out in zip(xs, outs):
                want = step(x, d["dh"], w_leaf, d["wu"])
                torch.cuda.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(out, want)), r
    gr = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(gr):
            F.dense(d["x"], w_leaf)
    torch.cuda.synchronize()


def test_long_offsets(device):
    """Rows whose byte offsets pass 32 bits: the last rows of a 2.3 GiB x and of as large a y."""
    from fpn import feed_forward as F
    rows, cin, cout = 1_250_000, 1000, 8
    x = torch.zeros((rows, cin), dtype=torch.bfloat16, device=device)
    x[-3:] = 1
    w = torch.ones((cin, cout), dtype=torch.bfloat16, device=device)
    y = F.dense(x, w)
    assert not y[:-3].any() and (y[-3:] == 1000).all()
    dy = torch.zeros((rows, cout), dtype=torch.bfloat16, device=device)
    dy[-1] = 2
    dx, dw, _ = F.dense_grad(dy, x, w)
    assert not dx[:-1].any() and (dx[-1] == 16).all() and (dw == 2).all()
    del x, dx
    y = F.dense(torch.ones((rows, 8), dtype=torch.bfloat16, device=device), torch.ones((8, cin), dtype=torch.bfloat16, device=device))
    assert (y == 8).all()


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_larger_products(device, t):
    """Sizes that take the larger tiles, against a float64 product on the device.  Of K fp32 additions each rounds a partial
    sum, which is at most about the final one, by up to 2^-24 of it, independently: relative to the result's norm at
    most 2^-24 sqrt K, plus the result's own rounding u; a gated product has two such factors, the gate's moved by an
    activation of slope at most 1.13 (relative to its value by less than 4 where it matters to the norm)."""
    from fpn import feed_forward as F
    dtype, u = TYPES[t]

    def near(got, want, k, factor=1):
        assert float((got.double() - want).norm() / want.norm()) <= u + factor * 2.0 ** -24 * k ** 0.5
    for rows, cin, cout in [(2048, 1024, 2048), (4099, 515, 1027), (1024, 2000, 4096), (16, 4096, 4096), (70000, 64, 96), (9001, 640, 3), (4100, 515, 13)]:
        d = make(device, dtype, rows, cin, cout, seed=6)
        want = d["x"].double() @ d["w"].double()
        y = F.dense(d["x"], d["w"])
        near(y, want, cin)
        # (the largest of 10^7 normal values is under 5.8: half a bf16 step there is 2^-6)
        assert float((y.double() - want).abs().max()) <= (2.0 ** -6 + 1e-4 if t == "bf16" else 8 * 2.0 ** -24 * cin ** 0.5 * 6)
        dx, dw, _ = F.dense_grad(d["dy"], d["x"], d["w"])
        near(dx, d["dy"].double() @ d["w"].double().t(), cout)
        near(dw, d["x"].double().t() @ d["dy"].double(), rows)
        h = F.gated(d["x"], d["wg"], d["wu"])
        g, up = d["x"].double() @ d["wg"].double(), d["x"].double() @ d["wu"].double()
        near(h, torch.nn.functional.silu(g) * up, cin, 5)


@pytest.mark.parametrize("t", list(TYPES))
def test_layers(device, t):
    """tf_util's layers are the operators on the store's variables, in the inputs' type, over any leading dimensions."""
    from fpn import feed_forward as F
    from fpn import tf_util, variables
    dtype = TYPES[t][0]
    g = torch.Generator().manual_seed(3)
    points = torch.randn((2, 37, 64), generator=g).to(dtype).to(device).requires_grad_()
    skip = torch.randn((2, 37, 64), generator=g).to(dtype).to(device)
    with variables.use_store(variables.VariableStore(device, seed=4)) as store:
        def layers():
            with variables.variable_scope("refine"):
                h = tf_util.gated_feed_forward(points, 96, "block", residual=points)
                return tf_util.dense(h, 64, "out", "gelu", skip), tf_util.dense(h, 10, "head", use_bias=False)
        y, z = layers()
        assert sorted(store.keys()) == sorted("refine/%s/%s" % (layer, kind) for layer, kinds in (
            ("block/gate", 2), ("block/up", 2), ("block/down", 2), ("out", 2), ("head", 1)) for kind in ("weights", "biases")[:kinds])
        for name in list(store.keys()):                     # biases that are seen, and the casts made again
            store[name] = store[name] + 0.25
        y, z = layers()
        v = {name: value.to(dtype) for name, value in store.items()}
    x = points.reshape(-1, 64)
    h = F.gated_feed_forward(x, v["refine/block/gate/weights"], v["refine/block/up/weights"], v["refine/block/down/weights"],
                             v["refine/block/gate/biases"], v["refine/block/up/biases"], v["refine/block/down/biases"], residual=x)
    want_y = F.dense(h, v["refine/out/weights"], v["refine/out/biases"], "gelu", skip.reshape(-1, 64))
    want_z = F.dense(h, v["refine/head/weights"])
    assert y.shape == (2, 37, 64) and torch.equal(y.reshape(-1, 64), want_y)
    assert z.shape == (2, 37, 10) and torch.equal(z.reshape(-1, 10), want_z)
    (got,) = torch.autograd.grad([y, z], [points], [torch.ones_like(y), torch.ones_like(z)])
    (want,) = torch.autograd.grad([want_y, want_z], [points], [torch.ones_like(want_y), torch.ones_like(want_z)])
    assert torch.equal(got, want)
    with variables.use_store(store):
        with pytest.raises(ValueError, match="rank 2 or more"):
            tf_util.dense(points.reshape(-1), 10, "head")
        with pytest.raises(ValueError, match="residual has shape"):
            tf_util.dense(points, 10, "head2", residual=skip)


def test_overwritten_results_are_noticed(device):
    """`out` counts as written in place: a backward pass that saved it refuses, and a leaf that requires gradients cannot
    be given."""
    from fpn import feed_forward as F
    x, w = torch.ones((4, 8), device=device), torch.ones((8, 8), device=device)
    leaf = torch.ones((4, 8), device=device, requires_grad=True)
    with pytest.raises(ValueError, match="out requires gradients"):
        F.dense(x, w, out=leaf)
    held = torch.ones((4, 8), device=device)
    y = (leaf * held).sum()
    F.dense(x, w, out=held)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        inside = torch.ones((4, 8), device=device)
        assert (F.dense(x, w, out=inside) == 8).all()


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("cols", [False, True])
@pytest.mark.parametrize("rows,cin,n", [(4096, 544, 4096), (4096, 2048, 2048), (2048, 1312, 1408), (640, 1312, 640), (1088, 1999, 520), (512, 96, 512)])
def test_every_tile_shape(device, t, cols, rows, cin, n):
    """Sizes from which the choice of tile takes each shape, with even and odd numbers of stages and what is left of k: every
    product of a step (with and without gates, and the one that ends in dg and du) relative to its norm.  A result has its
    own rounding, u; dpre (dg, du) were rounded once, independent errors of at most u of each, which a product with independent
    factors passes on as at most u of its norm: 2 u; sums as in test_larger_products."""
    from fpn import feed_forward as F
    dtype, u = TYPES[t]
    g = torch.Generator(device=device).manual_seed(rows + cin)

    def r(*shape, s=1.0):
        return (torch.randn(shape, generator=g, device=device) * s).to(dtype)

    def w(k, m):
        return r(m, k, s=k ** -0.5).t() if cols else r(k, m, s=k ** -0.5)

    def near(got, want, k, halves=1, factor=1, what=""):
        off = float((got.double() - want).norm() / want.norm())
        assert off <= halves * u + factor * 2.0 ** -24 * k ** 0.5, (what, off)
    x, wg, wu, wd, dy, dh = r(rows, cin), w(cin, n), w(cin, n), w(n, cin), r(rows, cin), r(rows, n)
    x6, wg6, wu6, wd6, dy6, dh6 = (v.double() for v in (x, wg, wu, wd, dy, dh))
    gate6, up6 = x6 @ wg6, x6 @ wu6
    sig = torch.sigmoid(gate6)
    value, slope = gate6 * sig, sig * (1 + gate6 * (1 - sig))
    near(F.dense(x, wg), gate6, cin, what="y")
    dx, dw, _ = F.dense_grad(dh, x, wg)
    near(dx, dh6 @ wg6.t(), n, what="dx")
    near(dw, x6.t() @ dh6, rows, what="dw")
    h, gate, up = F.gated(x, wg, wu, keep=True)
    near(h, value * up6, cin, 1, 5, "h")
    assert torch.equal(h, F.gated(x, wg, wu))
    dh6 = dy6 @ wd6.t()
    dg6, du6 = dh6 * up6 * slope, dh6 * value
    dx, dwg, dwu, dbg, dbu = F.gated_grad(dy, x, wg, wu, gate, up, bias=True, w_down=wd)
    near(dx, dg6 @ wg6.t() + du6 @ wu6.t(), 2 * n, 2, 10, "gated dx")
    near(dwg, x6.t() @ dg6, rows, 2, 10, "dw_gate")
    near(dwu, x6.t() @ du6, rows, 2, 10, "dw_up")
    near(dbg, dg6.sum(0), rows, 1, 10, "dbias_gate")
    near(dbu, du6.sum(0), rows, 1, 10, "dbias_up")


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("cols", [False, True])
@pytest.mark.parametrize("rows,cin,n", [(1, 2080, 4104), (3, 2048, 4096), (16, 2048, 2048), (20, 1040, 4096), (31, 96, 512), (50, 1024, 4128),
                                        (5, 64, 8200), (27, 72, 8208), (64, 200, 8192), (512, 1024, 4096)])
def test_few_rows_of_wide_weights(device, t, cols, rows, cin, n):
    """Sizes that take the few-row kernel with each of its shapes (k split over workgroups among them), relative to the
    results' norm as above; the residual may be the output."""
    from fpn import feed_forward as F
    dtype, u = TYPES[t]
    g = torch.Generator(device=device).manual_seed(rows + cin)

    def r(*shape, s=1.0):
        return (torch.randn(shape, generator=g, device=device) * s).to(dtype)
    x, bias, res = r(rows, cin), r(n), r(rows, n)
    wg, wu = (r(n, cin, s=cin ** -0.5).t() if cols else r(cin, n, s=cin ** -0.5) for _ in range(2))
    x6, wg6, wu6, bias6, res6 = (v.double() for v in (x, wg, wu, bias, res))

    def near(got, want, factor):
        assert float((got.double() - want).norm() / want.norm()) <= u + factor * 2.0 ** -24 * cin ** 0.5
    gate = x6 @ wg6 + bias6
    near(F.dense(x, wg, bias), gate, 1)
    near(F.gated(x, wg, wu, bias), gate * torch.sigmoid(gate) * (x6 @ wu6), 5)
    near(F.dense(x, wg, bias, "relu", res, out=res), torch.relu(gate) + res6, 1)
