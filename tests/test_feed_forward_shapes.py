"""Sizes from which the choice of kernel takes each shape of workgroup, with rows and columns off its tile: what each size
takes (on the host, with the paces of a 256-CU device), and every epilogue in every shape against the formulas in float64."""
import ctypes

import pytest
import torch

# rows, cin, cout -> the shape of a dense and of a gated product, 16-bit and float32 types; "deep" ones hold twice the stages,
# "split" ones cut k over workgroups and join the partial sums
SHAPES = [
    ((4099, 72, 2040), "256x256", "256x128", "128x128", "128x128"),
    ((4099, 2056, 2040), "256x256", "128x128", "64x64", "64x64"),
    ((2051, 72, 2040), "256x128", "256x256", "128x128", "128x128"),
    ((1030, 104, 2040), "64x64", "256x128", "64x64", "128x128"),
    ((3001, 520, 1032), "128x128", "256x128", "64x64", "64x64"),
    ((3001, 520, 520), "64x64", "128x128", "64x64", "64x64"),
    ((1030, 1312, 2040), "128x128 deep", "256x128", "64x64", "64x64"),
    ((260, 1312, 4088), "64x64 deep", "128x128 deep", "64x64 split", "64x64"),
    ((130, 1312, 1032), "64x64 deep", "64x64 deep", "64x64 split", "64x64 split"),
    ((130, 1312, 264), "64x64 split", "64x64 split", "64x64 split", "64x64 split"),
    ((130, 72, 264), "64x64", "64x64", "64x64", "64x64"),
    ((61, 1032, 520), "few", "few", "few", "few"),
]
SIZES = [s[0] for s in SHAPES]
TYPES = {"f32": (torch.float32, 2.0 ** -24), "bf16": (torch.bfloat16, 2.0 ** -8), "f16": (torch.float16, 2.0 ** -11)}


class Plan(ctypes.Structure):
    """feed_forward.h's Plan"""
    _fields_ = [("few", ctypes.c_bool), ("wide", ctypes.c_bool), ("bm", ctypes.c_int), ("bn", ctypes.c_int), ("splits", ctypes.c_int),
                ("tiles_per_split", ctypes.c_long), ("partial_bytes", ctypes.c_size_t)]


def shape_of(dtype, m, n, k, gated):
    """fpn::ff::plan_product for a forward product of whole rows, weights (in,out), and what launch_wide makes of the plan."""
    from fpn import _lib
    plan_product = _lib.load()._ZN3fpn2ff12plan_productEililiibbii
    plan_product.restype = Plan
    plan_product.argtypes = [ctypes.c_int, ctypes.c_long, ctypes.c_int, ctypes.c_long, ctypes.c_int, ctypes.c_int, ctypes.c_bool,
                             ctypes.c_bool, ctypes.c_int, ctypes.c_int]
    p = plan_product(dtype, m, n, k, 1, 1, gated, True, 0, 1)
    if p.few:
        return "few"
    assert p.wide
    cols = p.bn // 2 if gated else p.bn
    blocks = -(-m // p.bm) * -(-n // cols) * p.splits
    deep = dtype and p.bm < 256 and p.tiles_per_split >= 40 and blocks <= (1 if p.bm == 128 else 2) * 256
    return "%dx%d" % (p.bm, p.bn) + (" deep" if deep else "") + (" split" if p.splits > 1 else "")


@pytest.mark.parametrize("size,dense16,gated16,dense32,gated32", SHAPES)
def test_each_size_takes_its_shape(size, dense16, gated16, dense32, gated32):
    """If a change of the paces moves a size to another shape, the tests below lose that shape: find another size for it."""
    m, k, n = size
    for dtype in (1, 2):
        assert (shape_of(dtype, m, n, k, False), shape_of(dtype, m, n, k, True)) == (dense16, gated16)
    assert (shape_of(0, m, n, k, False), shape_of(0, m, n, k, True)) == (dense32, gated32)


def test_the_sizes_take_every_shape():
    sixteen = {"256x256", "256x128", "128x128", "128x128 deep", "64x64", "64x64 deep", "64x64 split", "few"}
    assert {s[1] for s in SHAPES} == sixteen == {s[2] for s in SHAPES}
    assert {s[3] for s in SHAPES} == {"128x128", "64x64", "64x64 split", "few"} == {s[4] for s in SHAPES}


def act64(v, act):
    """(value, derivative)"""
    if act == "relu":
        return v.clamp(min=0), (v > 0).double()
    if act == "silu":
        s = torch.sigmoid(v)
        return v * s, s * (1 + v * torch.sigmoid(-v))
    if act == "gelu":
        phi = torch.special.erfc(-v / 2 ** 0.5) / 2
        return v * phi, phi + v * torch.exp(-v * v / 2) * (2 * torch.pi) ** -0.5
    return v, torch.ones_like(v)


def inputs(device, dtype, rows, cin, n, cols):
    g = torch.Generator(device=device).manual_seed(rows + 3 * cin + n)

    def r(*shape, s=1.0):
        return (torch.randn(shape, generator=g, device=device) * s).to(dtype)

    def w(k, m):
        return r(m, k, s=k ** -0.5).t() if cols else r(k, m, s=k ** -0.5)
    return {"x": r(rows, cin), "wg": w(cin, n), "wu": w(cin, n), "wd": w(n, cin), "bg": r(n, s=0.3), "bu": r(n, s=0.3), "res": r(rows, n),
            "dy": r(rows, cin)}


def close(got, want, s, k, u, what):
    """The tolerance of test_gpu_feed_forward.py: the result's own rounding, and 2^-24 (4 + sqrt k) of the root of the sum of
    the squared terms for fp32 sums of k products, six times over for the largest of millions of values; fp16 loses up to
    2^-25 below its normal numbers."""
    assert torch.isfinite(got).all(), what
    tol = u * want.abs() + 6 * 2.0 ** -24 * (4 + k ** 0.5) * s + (2.0 ** -25 if u == 2.0 ** -11 else 0)
    off = (got.double() - want).abs()
    assert (off <= tol).all(), "%s: %.3g of the tolerance" % (what, float((off / tol).max()))


def root(a, b):
    return (a.square() @ b.square()).sqrt()


@pytest.mark.gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("cols", [False, True])
@pytest.mark.parametrize("rows,cin,n", SIZES)
def test_dense_epilogues_of_every_shape(device, t, cols, rows, cin, n):
    """Bias, activation, residual (given, one row for all, and as the output itself) and kept pre-activations."""
    from fpn import feed_forward as F
    dtype, u = TYPES[t]
    a = inputs(device, dtype, rows, cin, n, cols)
    x, w, b, res = a["x"], a["wg"], a["bg"], a["res"]
    x6, w6, b6, res6 = (v.double() for v in (x, w, b, res))
    p = x6 @ w6 + b6
    s = root(x6, w6) + p.abs()
    for act in ("gelu", "relu", None):
        v = act64(p, act)[0]
        y, pre = F.dense(x, w, b, act, res, keep=True)
        close(y, v + res6, 1.2 * s + v.abs() + res6.abs(), cin, u, "y")
        if act:
            close(pre, p, s, cin, 2.0 ** -24, "pre")
        assert torch.equal(y, F.dense(x, w, b, act, res))
        out = res.clone()
        F.dense(x, w, b, act, out, out=out)
        assert torch.equal(out, y)
        wide = torch.full((rows, n + 24), float("nan"), dtype=dtype, device=device)
        wide[:, 8:8 + n] = res
        F.dense(x, w, b, act, wide[:, 8:8 + n], out=wide[:, 8:8 + n])
        assert torch.equal(wide[:, 8:8 + n], y) and wide[:, :8].isnan().all() and wide[:, 8 + n:].isnan().all()
        row = res[:1].expand(rows, n)
        assert torch.equal(F.dense(x, w, b, act, row), F.dense(x, w, b, act, row.contiguous()))
    plain = F.dense(x, w)
    close(plain, x6 @ w6, root(x6, w6) + (x6 @ w6).abs(), cin, u, "plain")


@pytest.mark.gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("cols", [False, True])
@pytest.mark.parametrize("rows,cin,n", SIZES)
def test_gated_epilogues_of_every_shape(device, t, cols, rows, cin, n):
    """Both biases, the activation, the kept sums; and the way back through a down projection, whose product ends in dg, du
    and their column sums (k is cin again, so that it takes the dense product's shape)."""
    from fpn import feed_forward as F
    dtype, u = TYPES[t]
    a = inputs(device, dtype, rows, cin, n, cols)
    x, wg, wu, wd, bg, bu, dy = (a[k] for k in ("x", "wg", "wu", "wd", "bg", "bu", "dy"))
    x6, wg6, wu6, wd6, bg6, bu6, dy6 = (v.double() for v in (x, wg, wu, wd, bg, bu, dy))
    pg, pu = x6 @ wg6 + bg6, x6 @ wu6 + bu6
    sg, su = root(x6, wg6) + pg.abs(), root(x6, wu6) + pu.abs()
    for act in ("gelu", "silu"):
        v, slope = act64(pg, act)
        h, gate, up = F.gated(x, wg, wu, bg, bu, act, keep=True)
        close(h, v * pu, 1.2 * sg * pu.abs() + su * v.abs() + (v * pu).abs(), cin, u, "h")
        close(gate, pg, sg, cin, 2.0 ** -24, "gate")
        close(up, pu, su, cin, 2.0 ** -24, "up")
        assert torch.equal(h, F.gated(x, wg, wu, bg, bu, act))
        dx, dwg, dwu, dbg, dbu = F.gated_grad(dy, x, wg, wu, gate, up, act, bias=True, w_down=wd)
        dh = dy6 @ wd6.t()
        dg, du = dh * pu * slope, dh * v

        def near(got, want, k, halves, what):
            # relative to the norm, as in test_gpu_feed_forward.py: halves roundings of u, and fp32 sums of k terms in each
            # of three factors that the activation's slope and curvature (at most 1.13) pass on
            off = float((got.double() - want).norm() / want.norm())
            assert off <= halves * u + 10 * 2.0 ** -24 * k ** 0.5, (what, off)
        near(dx, dg @ wg6.t() + du @ wu6.t(), 2 * n, 2, "dx")
        near(dwg, x6.t() @ dg, max(rows, cin), 2, "dwg")
        near(dwu, x6.t() @ du, max(rows, cin), 2, "dwu")
        near(dbg, dg.sum(0), max(rows, cin), 1, "dbg")
        near(dbu, du.sum(0), max(rows, cin), 1, "dbu")


@pytest.mark.gpu
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("cols", [False, True])
@pytest.mark.parametrize("rows,cin,n", SIZES)
def test_a_block_rounds_no_more_than_twice(device, t, cols, rows, cin, n):
    """gated_feed_forward and its gradients through autograd, relative to their norms: every result is rounded once, and of the
    operands that one product hands to the next h (to y and dw_down) and dg, du (to dx and the gated weights' gradients) once
    more, each time by at most u of every value - at most u of the norm.  The biases' gradients come from the unrounded
    values.  fp32 sums add 10 2^-24 sqrt k as above."""
    from fpn import feed_forward as F
    dtype, u = TYPES[t]
    a = inputs(device, dtype, rows, cin, n, cols)
    g = torch.Generator(device=device).manual_seed(5)
    a["bd"], a["res"] = ((torch.randn(s, generator=g, device=device) * 0.3).to(dtype) for s in ((cin,), (rows, cin)))
    names = ("x", "wg", "wu", "wd", "bg", "bu", "bd", "res")
    leaves = [a[k].detach().requires_grad_() for k in names]
    y = F.gated_feed_forward(*leaves[:7], "silu", leaves[7])
    got = dict(zip(names, torch.autograd.grad(y, leaves, a["dy"])), y=y.detach())
    x, wg, wu, wd, bg, bu, bd, res = (a[k].double() for k in names)
    dy = a["dy"].double()
    pg, pu = x @ wg + bg, x @ wu + bu
    v, slope = act64(pg, "silu")
    h, dh = v * pu, dy @ wd.t()
    dg, du = dh * pu * slope, dh * v
    want = {"y": h @ wd + bd + res, "wd": h.t() @ dy, "bd": dy.sum(0), "x": dg @ wg.t() + du @ wu.t(), "wg": x.t() @ dg, "wu": x.t() @ du,
            "bg": dg.sum(0), "bu": du.sum(0)}
    assert torch.equal(got["res"], a["dy"])
    for k, w in want.items():
        halves = 1 if k in ("bd", "bg", "bu") else 2
        off = float((got[k].double() - w).norm() / w.norm())
        assert off <= halves * u + 10 * 2.0 ** -24 * max(rows, cin, n) ** 0.5, (k, off)
