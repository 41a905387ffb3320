"""The feed-forward operators' refusals and workspace sizes: all of them are decided on the host, before any launch."""
import ctypes

import pytest
import torch

P, ODD = ctypes.c_void_p(256), ctypes.c_void_p(257)
F32, BF16, F16 = 0, 1, 2
BIG = 1 << 40


def lib():
    from fpn import _lib
    return _lib.load()


def said():
    return lib().fpn_last_error_string().decode()


def dense(**kw):
    a = dict(dtype=BF16, rows=4, cin=8, cout=16, x=P, ldx=8, w=P, ldw=16, tr=0, bias=None, act=0, res=None, ldr=0, y=P, ldy=16,
             pre=None, ldp=0, ws=P, size=BIG)
    a.update(kw)
    return lib().fpn_dense(*a.values(), None)


def dense_grad(**kw):
    a = dict(dtype=BF16, rows=4, cin=8, cout=16, dy=P, lddy=16, x=P, ldx=8, w=P, ldw=16, tr=0, pre=P, ldp=16, act=2, dx=P, lddx=8, dw=P,
             lddw=16, db=P, ws=P, size=BIG)
    a.update(kw)
    return lib().fpn_dense_grad(*a.values(), None)


def gated(**kw):
    a = dict(dtype=BF16, rows=4, cin=8, cout=16, x=P, ldx=8, wg=P, ldg=16, wu=P, ldu=16, tr=0, bg=None, bu=None, act=2, h=P, ldh=16,
             gate=None, up=None, ldp=0, ws=P, size=BIG)
    a.update(kw)
    return lib().fpn_gated(*a.values(), None)


def gated_grad(**kw):
    a = dict(dtype=BF16, rows=4, cin=8, cout=16, cdown=0, dh=P, lddh=16, wd=None, ldd=0, trd=0, x=P, ldx=8, wg=P, ldg=16, wu=P, ldu=16, tr=0, gate=P, up=P, ldp=16,
             act=2, dx=P, lddx=8, dwg=P, dwu=P, lddw=16, dbg=None, dbu=None, ws=P, size=BIG)
    a.update(kw)
    return lib().fpn_gated_grad(*a.values(), None)


@pytest.mark.parametrize("call", [dense, dense_grad, gated, gated_grad])
@pytest.mark.parametrize("bad,code,text", [
    (dict(dtype=3), -1, "dtype"), (dict(dtype=-1), -1, "dtype"), (dict(rows=-1), -1, "rows"), (dict(cin=0), -1, "widths"),
    (dict(cout=0), -1, "widths"), (dict(act=6), -1, "activation"), (dict(act=-1), -1, "activation"),
    (dict(cin=1 << 21), -3, "widths"), (dict(x=None), -1, "x is null"), (dict(x=ODD), -1, "x is not aligned"),
    (dict(ldx=7), -1, "row stride"), (dict(ldx=1 << 21), -3, "row stride"), (dict(ldx=-8), -1, "row stride"),
    (dict(ws=ctypes.c_void_p(264)), -1, "16-byte aligned")])
def test_bad_arguments(call, bad, code, text):
    assert call(**bad) == code
    assert text in said()


@pytest.mark.parametrize("call,bad,text", [
    (dense, dict(w=None), "w is null"), (dense, dict(ldw=15), "w: row stride"), (dense, dict(ldw=0), "w: row stride"),
    (dense, dict(tr=1, ldw=7), "w: row stride"), (dense, dict(y=None), "y is null"), (dense, dict(ldy=0), "y: row stride"),
    (dense, dict(bias=ODD), "bias"), (dense, dict(res=P, ldr=5), "residual"), (dense, dict(pre=P, ldp=3), "pre"),
    (dense, dict(rows=16, cin=4096, cout=4096, ldx=4096, ldw=4096, ldy=4096, size=100), "workspace"),
    (dense, dict(rows=16, cin=4096, cout=4096, ldx=4096, ldw=4096, ldy=4096, ws=None), "workspace"),
    (dense_grad, dict(dy=None), "dy is null"), (dense_grad, dict(lddy=0), "dy: row stride"), (dense_grad, dict(pre=None), "pre is null"),
    (dense_grad, dict(lddx=7), "dx"), (dense_grad, dict(tr=1, lddw=7), "dw"), (dense_grad, dict(db=ODD), "dbias"),
    (dense_grad, dict(size=10), "workspace"),
    (gated, dict(wu=None), "w_up is null"), (gated, dict(ldu=1), "w_up: row stride"), (gated, dict(gate=P, ldp=16), "together"),
    (gated, dict(gate=P, up=P, ldp=15), "gate"), (gated, dict(ldh=2), "h: row stride"), (gated, dict(bu=ODD), "bias_up"),
    (gated_grad, dict(cdown=-1), "cdown"), (gated_grad, dict(cdown=24, lddh=24), "w_down is null"),
    (gated_grad, dict(cdown=24, lddh=24, wd=P, ldd=23), "w_down: row stride"), (gated_grad, dict(cdown=24, wd=P, ldd=24), "dh: row stride"),
    (gated_grad, dict(cdown=24, lddh=24, wd=P, ldd=15, trd=1), "w_down: row stride"),
    (gated_grad, dict(gate=ctypes.c_void_p(258)), "gate is not aligned"),
    (gated_grad, dict(gate=None), "gate is null"), (gated_grad, dict(dwu=None), "together"), (gated_grad, dict(dbu=P), "together"),
    (gated_grad, dict(lddw=3), "dw_gate"), (gated_grad, dict(ws=None), "workspace")])
def test_bad_arguments_of_one(call, bad, text):
    assert call(**bad) == -1
    assert text in said()


def test_no_rows_is_a_valid_call_without_a_launch():
    assert dense(rows=0, x=None, w=None, y=None, ws=None, size=0) == 0
    assert gated(rows=0, x=None, wg=None, wu=None, h=None, ws=None, size=0) == 0


def test_workspace_sizes():
    L = lib()
    assert L.fpn_dense_workspace_bytes(BF16, 8192, 4096, 4096, 1) == 0            # enough tiles: k is not split
    assert L.fpn_dense_workspace_bytes(BF16, 1, 64, 64, 1) == 0                   # a short k is not split either
    assert L.fpn_dense_workspace_bytes(7, 1, 64, 64, 1) == 0 and L.fpn_dense_workspace_bytes(BF16, 1, 0, 64, 1) == 0
    for t, size in ((F32, 4), (BF16, 2), (F16, 2)):
        d = 1000 * 512 * size
        assert L.fpn_dense_grad_workspace_bytes(t, 1000, 64, 512, 2, 1) >= d
        assert L.fpn_gated_grad_workspace_bytes(t, 1000, 64, 512, 0, 1) >= 2 * d
        # partial sums of a split product: whole copies of the result
        need = L.fpn_dense_workspace_bytes(t, 16, 8192, 256, 1)
        assert need % (16 * 256 * 4) == 0
        # ragged operands: room for their copies, rows padded to whole chunks, where there is enough to multiply
        need = L.fpn_dense_workspace_bytes(t, 2000, 1091, 515, 0) - L.fpn_dense_workspace_bytes(t, 2000, 1091, 515, 1)
        assert need >= (2000 * 1092 + 1091 * 516) * size
        assert L.fpn_dense_workspace_bytes(t, 20, 1091, 515, 0) == L.fpn_dense_workspace_bytes(t, 20, 1091, 515, 1)
    # one row more never needs a workspace out of proportion (splits times result stays bounded)
    for rows in (1, 16, 17, 64, 65, 1000, 131072):
        for n in (2, 64, 4096, 8192):
            assert L.fpn_dense_workspace_bytes(BF16, rows, 8192, n, 1) <= 256 << 20


def test_python_refusals_without_a_device():
    from fpn import feed_forward as F
    x, w = torch.zeros(4, 8), torch.zeros(8, 16)
    with pytest.raises(ValueError, match="ROCm device"):
        F.dense(x, w)
    with pytest.raises(ValueError, match="ROCm device"):
        F.gated(x, w, w)
    with pytest.raises(ValueError, match="rank 2"):
        F.dense(x[0], w)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        F.dense(x.double(), w)
    with pytest.raises(TypeError, match="torch.Tensor"):
        F.dense([[1.0]], w)


def test_storage_orders_of_weights():
    from fpn import feed_forward as F
    w = torch.zeros(8, 16)
    assert F._weights(("w",), (w,)) == (0, [16])
    assert F._weights(("w",), (torch.zeros(16, 8).t(),)) == (1, [8])
    both = torch.zeros(8, 40)
    assert F._weights(("g", "u"), (both[:, :16], both[:, 17:33])) == (0, [40, 40])
    assert F._weights(("g", "u"), (torch.zeros(8, 1), torch.zeros(1, 8).t())) [0] in (0, 1)
    with pytest.raises(ValueError, match="both the same"):
        F._weights(("g", "u"), (w, torch.zeros(16, 8).t()))
    for bad in (torch.zeros(1, 16).expand(8, 16), torch.zeros(8, 32)[:, ::2], torch.zeros(8, 1).expand(8, 16)):
        with pytest.raises(ValueError, match="strides"):
            F._weights(("w",), (bad,))


def test_row_strides_and_overlap():
    from fpn import feed_forward as F
    wide = torch.zeros(10, 40)
    assert F._rows("x", wide[:, 3:9]) == 40 and F._rows("x", torch.zeros(1, 6)) == 6
    assert F._rows("x", torch.zeros(1, 6).expand(5, 6), broadcast=True) == 0
    for bad in (torch.zeros(1, 6).expand(5, 6), torch.zeros(6, 5).t(), torch.zeros(20).as_strided((4, 6), (4, 1))):
        with pytest.raises(ValueError):
            F._rows("x", bad)
    assert not F._overlap(wide[:, :8], wide[:, 8:20]) and not F._overlap(wide[:, 30:], wide[:, :30])
    assert F._overlap(wide[:, :8], wide[:, 7:20]) and F._overlap(wide, wide) and F._overlap(wide[2:], wide[:3])
    assert not F._overlap(wide[:3], wide[3:]) and not F._overlap(wide, torch.zeros(4, 4))
    assert F._overlap(wide[:, 30:], wide[1:, :4].as_strided((3, 20), (40, 1), 35))


@pytest.mark.parametrize("call,more", [(dense, {}), (gated, {}), (dense_grad, dict(act=0, dw=None, db=None))])
def test_more_rows_than_one_launch_takes(call, more):
    """Products of sizes would overflow, or a grid have 2^32 threads or more: refused before anything is launched."""
    assert call(rows=(1 << 40) + 1, **more) == -3
    assert "rows" in said()
    assert call(rows=1 << 34, **more) == -3
    assert "workgroups" in said()
