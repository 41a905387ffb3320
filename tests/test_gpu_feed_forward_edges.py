"""Values that are not finite, and scratch memory that holds NaN, in each of the feed-forward operators' kernels: what they
reach is what the formula says, value by value, and nothing else."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": (torch.float32, 2.0 ** -24), "bf16": (torch.bfloat16, 2.0 ** -8), "f16": (torch.float16, 2.0 ** -11)}
NAN, INF = float("nan"), float("inf")
# whole 16-byte rows with a rest of k: the few-row and the pipelined kernel (one tile and several); ragged rows: the kernel that
# reads any, and (from 10^8 operations on) copies of the operands
SIZES = [(5, 72, 72), (64, 136, 40), (130, 72, 72), (2051, 72, 2040), (70, 75, 69), (300, 515, 650), (300, 515, 331)]


def tolerance(want, terms, k, u):
    """The result's own rounding and fp32 sums of k products, as in test_gpu_feed_forward.py (fp16: and its subnormal steps)"""
    return u * want.abs() + 6 * 2.0 ** -24 * (4 + k ** 0.5) * (terms + want.abs()) + (2.0 ** -25 if u == 2.0 ** -11 else 0)


def same(got, want, terms, k, u, what):
    """NaN where the formula has NaN, its infinities, and its finite values."""
    got = got.double().cpu()
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        wrong = kind(got) != kind(want)
        assert not wrong.any(), (what, kind.__name__, wrong.nonzero()[:4].tolist())
    finite = torch.isfinite(want)
    off = (got - want).abs()[finite]
    assert (off <= tolerance(want, terms, k, u)[finite]).all(), what


def operands(device, dtype, rows, cin, cout):
    g = torch.Generator().manual_seed(rows + cin + cout)
    x = torch.randn((rows, cin), generator=g).to(dtype)
    w = (torch.randn((cin, cout), generator=g) * cin ** -0.5).to(dtype)
    w[w == 0] = 0.5                                         # (an infinity times 0 is another test's matter)
    return x, w, torch.randn((rows, cout), generator=g).to(dtype)


def magnitudes(a, b):
    """sqrt(a^2 @ b^2) of the finite values"""
    return (a.nan_to_num(0, 0, 0).square() @ b.nan_to_num(0, 0, 0).square()).sqrt()


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows,cin,cout", SIZES)
def test_infinities_and_nan_reach_their_row_and_column(device, t, rows, cin, cout):
    """x: a NaN at the end of the last row, an infinity at the start of another; w: a NaN in the last element."""
    from fpn import feed_forward as F
    dtype, u = TYPES[t]
    x, w, res = operands(device, dtype, rows, cin, cout)
    x[rows - 1, cin - 1], x[3, 0] = NAN, INF
    w[cin - 1, cout - 1] = NAN
    x6, w6 = x.double(), w.double()
    pre = x6 @ w6
    assert torch.isinf(pre[3, :-1]).all() and torch.isnan(pre[-1]).all() and torch.isnan(pre[:, -1]).all()
    inner = pre[:-1, :-1]
    assert torch.isfinite(inner[torch.arange(rows - 1) != 3]).all()
    terms = magnitudes(x6, w6)
    x, w, res = x.to(device), w.to(device), res.to(device)
    for ww in (w, w.t().contiguous().t()):
        for act, f in ((None, lambda v: v), ("relu", torch.relu), ("sigmoid", torch.sigmoid)):
            want = f(pre)
            same(F.dense(x, ww, None, act), want, terms, cin, u, ("dense", act))
            same(F.dense(x, ww, None, act, res), want + res.double().cpu(), terms, cin, u, ("dense + residual", act))
            y, kept = F.dense(x, ww, None, act, keep=True)
            same(y, want, terms, cin, u, ("kept", act))
            if act:
                same(kept, pre, terms, cin, 2.0 ** -24, ("pre", act))
            # (a gated product's two factors: an infinite one times 0 is NaN in the formula, too)
            product = want * pre
            spread = 1.2 * terms * pre.abs().nan_to_num(0, 0, 0) + terms * want.abs().nan_to_num(0, 0, 0)
            same(F.gated(x, ww, ww, activation=act), product, spread, cin, u, ("gated", act))
        for act in ("silu", "gelu", "gelu_tanh"):
            y = F.dense(x, ww, None, act).double().cpu()
            up = torch.isposinf(pre)
            assert torch.isposinf(y[up]).all() and torch.isnan(y[torch.isnan(pre)]).all() and torch.isfinite(y[torch.isfinite(pre)]).all()


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows,cin,cout", SIZES)
@pytest.mark.parametrize("cols", [False, True])
def test_backward_passes_read_no_scratch_that_they_did_not_write(device, monkeypatch, t, rows, cin, cout, cols):
    """With a workspace full of NaN (pad columns of dpre and of copies, partial sums, column sums) every gradient is, bit for
    bit, what it is with a workspace of zeros; and a NaN of dy reaches its row of dx and its column of dw and db."""
    from fpn import feed_forward as F
    dtype, u = TYPES[t]
    x, w, dy = (v.to(device) for v in operands(device, dtype, rows, cin, cout))
    wd = (torch.randn((cout, 24), generator=torch.Generator().manual_seed(1)) * cout ** -0.5).to(dtype).to(device)
    if cols:
        w, wd = w.t().contiguous().t(), wd.t().contiguous().t()
    down = torch.randn((rows, 24), generator=torch.Generator().manual_seed(2)).to(dtype).to(device)

    def gradients(byte, dy):
        monkeypatch.setattr(F, "_workspace", lambda size, like: torch.full((size,), byte, dtype=torch.uint8, device=like.device) if size else None)
        out = {}
        for act in ("silu", None):
            y, pre = F.dense(x, w, None, act, keep=True)
            out["y", act] = (y,)
            out["dense", act] = F.dense_grad(dy, x, w, pre, act, bias=True)
            h, gate, up = F.gated(x, w, w, activation=act, keep=True)
            out["h", act] = (h, gate, up)
            out["gated", act] = F.gated_grad(dy, x, w, w, gate, up, act, bias=True)
            out["down", act] = F.gated_grad(down, x, w, w, gate, up, act, bias=True, w_down=wd)
        return out
    clean, dirty = gradients(0, dy), gradients(255, dy)
    for key, grads in clean.items():
        for a, b in zip(grads, dirty[key]):
            assert torch.isfinite(a).all() and torch.equal(a, b), key
    bad = dy.clone()
    bad[rows - 1, cout - 1] = NAN
    for key, (dx, dw, db) in ((k, v) for k, v in gradients(255, bad).items() if k[0] == "dense"):
        want = clean[key]
        assert torch.isnan(dx[-1]).all() and torch.equal(dx[:-1], want[0][:-1]), key
        assert torch.isnan(dw[:, -1]).all() and torch.equal(dw[:, :-1], want[1][:, :-1]), key
        assert torch.isnan(db[-1]) and torch.equal(db[:-1], want[2][:-1]), key
