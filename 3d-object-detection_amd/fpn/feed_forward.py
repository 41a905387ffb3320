"""Feed-forward operators: products with bias, activation and residual in the epilogue, and gated blocks, forward and
backward, through libfpn_hip.so (fpn_dense, fpn_dense_grad, fpn_gated, fpn_gated_grad; include/fpn.h).

    dense               y = act(x w + bias) + residual
    gated               h = act(x w_gate + bias_gate) * (x w_up + bias_up)
    gated_feed_forward  y = gated(x) w_down + bias_down + residual

In 16-bit types every result is rounded once, and so are the operands that one product hands to the next, which the matrix
units take in 16 bits: h between gated and the down projection, and dpre (dg, du) before dx and the weights' gradients.  Against
float64 the error of those results is up to about sqrt 2 of one rounding's: relative to the norm 2.3e-3 for the weights'
gradients of a bf16 block of 4096 x 1024 x 4096 (one rounding 1.7e-3), 1.9e-3 for its y; 2.9e-4 for dx and dw of an fp16 step of
1999 x 1091 x 515 (one rounding 2.1e-4).  Kept pre-activations, dh of the block, sums and column sums are fp32.

Which to use in fp32 with bias and ReLU, where both exist: `dense` is the faster for single rows and for many rows of whole
16-byte chunks (us, dense : shared_mlp: 1 x 1027 x 512 6 : 13, 131072 x 128 x 256 89 : 133, 8192 x 512 x 512 40 : 63,
131072 x 512 x 1024 1013 : 1346), `ops.shared_mlp` for widths that are not (1024 x 1027 x 512 26 : 18) and where it pools or
scales.  From two to 64 rows at such widths `dense` takes 15 us where whole ones take 6 to 9 (2 to 64 x 1027 x 512 against 1024):
the kernel for few rows reads whole chunks only.

They stand beside `ops.shared_mlp` (fp32, scale / shift / ReLU, pooling): every tensor of a call is float32, bfloat16
or float16, sums are fp32, weights are (in, out) - or the `.t()` view of weights held (out, in) -, rows may lie apart
(column slices of wider buffers).  Work is enqueued on the current stream of the tensors' device; nothing synchronises.

Gradients, either way:
  * tensors that require gradients: the calls are recorded by autograd;
  * `keep=True` returns what the backward pass needs beside the result, and `dense_grad` / `gated_grad` are that pass.
    This is the form for HIP graphs: recording through autograd while a graph is being captured is refused, since
    autograd would join streams that the capture does not know.
There are no forward-mode derivatives: a tensor that carries a tangent is refused.
"""
import torch
from torch.autograd import forward_ad

from . import _lib

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "sigmoid": 3, "gelu": 4, "gelu_tanh": 5}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _activation(name):
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError("activation must be one of %s, got %r" % (", ".join(repr(a) for a in ACTIVATIONS), name)) from None


def _no_tangent(name, t):
    """Refuses a tensor of forward-mode differentiation: it has a value like any other, and the result would lack a tangent."""
    if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError("%s carries a tangent: the feed-forward operators have no forward-mode derivatives" % name)


def _as_it_is(name, t):
    """Refuses a tensor whose memory does not say all of it."""
    if forward_ad._current_level >= 0:
        _no_tangent(name, t)
    if t.is_neg():
        raise ValueError("%s has a pending negation: call its resolve_neg() first" % name)


def _tensor(name, t, like, shape):
    """The checks that every argument gets: a tensor of the call's type, on its device, of this shape."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch.Tensor, got %s" % (name, type(t).__name__))
    if forward_ad._current_level >= 0 or t.is_neg():
        _as_it_is(name, t)
    if t.dtype is not like.dtype:
        raise ValueError("%s must be %s like x, got %s" % (name, like.dtype, t.dtype))
    if not t.is_cuda:
        raise ValueError("%s must live on a ROCm device (got %s); this package has no CPU path" % (name, t.device))
    if t.get_device() != like.get_device():
        raise ValueError("all tensors must be on the same device (%s is on %s, x on %s)" % (name, t.device, like.device))
    if t.shape != shape:
        raise ValueError("%s has shape %s, expected %s" % (name, tuple(t.shape), tuple(shape)))


def _first(name, x):
    if not isinstance(x, torch.Tensor):
        raise TypeError("%s must be a torch.Tensor, got %s" % (name, type(x).__name__))
    _as_it_is(name, x)
    if x.dim() != 2:
        raise ValueError("%s must have rank 2, got shape %s" % (name, tuple(x.shape)))
    if x.dtype not in _DTYPES:
        raise ValueError("%s must be float32, bfloat16 or float16, got %s" % (name, x.dtype))
    if not x.is_cuda:
        raise ValueError("%s must live on a ROCm device (got %s); this package has no CPU path" % (name, x.device))
    return _DTYPES[x.dtype]


def _rows(name, t, broadcast=False):
    """The row stride of a matrix whose rows are dense (broadcast: one row may stand for all)."""
    rows, cols = t.shape
    ld, unit = t.stride()
    if cols > 1 and unit != 1:
        raise ValueError("%s must have unit column stride, got strides %s" % (name, t.stride()))
    if rows <= 1:
        return cols
    if ld < cols and not (broadcast and ld == 0):
        raise ValueError("%s: rows %d elements apart overlap (%d columns)" % (name, ld, cols))
    return ld


def _orders(w):
    """The storage orders a weight matrix can be read in: {transposed: row stride}."""
    cin, cout = w.shape
    found = {}
    if (cout == 1 or w.stride(1) == 1) and (cin == 1 or w.stride(0) >= cout):
        found[0] = w.stride(0) if cin > 1 else cout
    if (cin == 1 or w.stride(0) == 1) and (cout == 1 or w.stride(1) >= cin):
        found[1] = w.stride(1) if cout > 1 else cin
    return found


def _weights(names, ws):
    """(transposed, row strides) of weights that are all (in, out) matrices or all transposed views of (out, in)."""
    if all(w.is_contiguous() for w in ws):
        return 0, [w.shape[1] for w in ws]
    orders = [_orders(w) for w in ws]
    for order in (0, 1):
        if all(order in o for o in orders):
            return order, [o[order] for o in orders]
    raise ValueError("%s must be dense (in, out) matrices or transposed views of dense (out, in) ones%s, got strides %s"
                     % (" and ".join(names), ", both the same" if len(ws) > 1 else "", ", ".join(str(w.stride()) for w in ws)))


def _vector(name, t, like, n):
    if t is None:
        return
    _tensor(name, t, like, (n,))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)


def _overlap(a, b):
    """Whether two row matrices share an element (column slices of one buffer do not)."""
    if not a.numel() or not b.numel():
        return False
    size = a.element_size()
    first = [t.data_ptr() for t in (a, b)]
    end = [p + ((t.shape[0] - 1) * t.stride(0) + (t.shape[1] - 1) * t.stride(1) + 1) * size for p, t in zip(first, (a, b))]
    if end[0] <= first[1] or end[1] <= first[0]:
        return False
    if a.shape[0] > 1 and b.shape[0] > 1 and a.stride() == b.stride() and a.stride(1) == 1:
        ld = a.stride(0)
        apart, odd = divmod(first[1] - first[0], size)
        at = apart % ld
        if not odd and at >= a.shape[1] and at + b.shape[1] <= ld:
            return False
    return True


def _output(out, x, rows, cols, inputs, may_be=None):
    """`out` or a new tensor, and its row stride."""
    if out is None:
        return torch.empty((rows, cols), dtype=x.dtype, device=x.device), cols
    _tensor("out", out, x, (rows, cols))
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out requires gradients: autograd would not see that it is overwritten")
    ld = _rows("out", out)
    for name, t in inputs:
        t2 = t if t is None or t.dim() == 2 else t.unsqueeze(0)
        if t2 is not None and _overlap(out, t2):
            raise ValueError("out shares memory with %s" % name)
    if may_be is not None and not (out.data_ptr() == may_be.data_ptr() and out.stride() == may_be.stride()) and _overlap(out, may_be):
        raise ValueError("out shares memory with residual without being it")
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)         # (a backward pass that saved it has to notice)
    return out, ld


def _workspace(size, x):
    """A call's own scratch memory, from torch's allocator on the current stream: calls on other streams and in captured
    graphs have theirs."""
    return torch.empty(size, dtype=torch.uint8, device=x.device) if size else None


def _whole(dtype, widths, *operands):
    """Whether every operand (tensor, row stride) starts at and moves by whole 16-byte chunks, and so do the widths."""
    bits = 0
    for n in widths:
        bits |= n
    for t, ld in operands:
        if t is None:
            continue
        bits |= ld
        if t.data_ptr() & 15:
            return 0
    return int(bits & (3 if dtype == 0 else 7) == 0)


def _p(t):
    """Device pointer of a tensor (None -> NULL)."""
    return None if t is None else t.data_ptr()


def _call(x, function, *args):
    index = x.get_device()
    if torch._C._cuda_getDevice() == index:
        status = function(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = function(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status)


def _recorded(*tensors):
    """Whether autograd has to see the call."""
    for t in tensors:
        if t is not None and t.requires_grad:
            break
    else:
        return False
    if not torch.is_grad_enabled():
        return False
    _no_capture()
    return True


def _no_capture():
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a call on tensors that require gradients cannot be captured into a graph: use keep=True and "
                           "dense_grad / gated_grad (or torch.no_grad())")


# ---- dense ---------------------------------------------------------------------------------------------------------

def dense(x, w, bias=None, activation=None, residual=None, out=None, keep=False):
    """y = act(x w + bias) + residual: x (rows, cin), w (cin, cout), bias (cout,), residual and y (rows, cout).

    activation: None, "relu", "silu", "sigmoid", "gelu" (exact) or "gelu_tanh".  `out` receives y (it may be the
    residual itself, but share memory with no other argument).  keep=True returns (y, pre) for `dense_grad`, pre
    being x w + bias in float32 (rounded further it would cost the gradients digits), or None where there is no
    activation."""
    dtype = _first("x", x)
    act = _activation(activation)
    lib = _lib.load()
    rows, cin = x.shape
    if not isinstance(w, torch.Tensor) or w.dim() != 2:
        raise ValueError("w must be a (cin, cout) tensor")
    cout = w.shape[1]
    _tensor("w", w, x, (cin, cout))
    _vector("bias", bias, x, cout)
    if residual is not None:
        _tensor("residual", residual, x, (rows, cout))
    if not keep and _recorded(x, w, bias, residual):
        if out is not None:
            raise ValueError("out cannot be given for tensors that require gradients")
        return _Dense.apply(x, w, bias, activation, residual)
    ldx = _rows("x", x, broadcast=True)
    transposed, (ldw,) = _weights(("w",), (w,))
    ldr = _rows("residual", residual, broadcast=True) if residual is not None else 0
    y, ldy = _output(out, x, rows, cout, (("x", x), ("w", w), ("bias", bias)), residual)
    pre = torch.empty((rows, cout), dtype=torch.float32, device=x.device) if keep and act else None
    size = lib.fpn_dense_workspace_bytes(dtype, rows, cin, cout, _whole(dtype, (cin, cout), (x, ldx), (w, ldw)))
    ws = _workspace(size, x)
    _call(x, lib.fpn_dense, dtype, rows, cin, cout, _p(x), ldx, _p(w), ldw, transposed, _p(bias), act, _p(residual), ldr, _p(y), ldy,
          _p(pre), cout, _p(ws), size)
    return (y, pre) if keep else y


def dense_grad(dy, x, w, pre=None, activation=None, bias=False, need_x=True, need_w=True):
    """The gradients of `dense`: (dx, dw, dbias), each None where it is not asked for (bias=True asks for dbias); dw is
    stored as w is.  `pre` is what keep=True returned.  The residual's gradient is dy."""
    dtype = _first("x", x)
    act = _activation(activation)
    lib = _lib.load()
    rows, cin = x.shape
    if not isinstance(w, torch.Tensor) or w.dim() != 2:
        raise ValueError("w must be a (cin, cout) tensor")
    cout = w.shape[1]
    _tensor("w", w, x, (cin, cout))
    _tensor("dy", dy, x, (rows, cout))
    lddy, ldx = _rows("dy", dy), _rows("x", x, broadcast=True)
    transposed, (ldw,) = _weights(("w",), (w,))
    ldp = cout
    if act:
        if pre is None:
            raise ValueError("pre (from dense(..., keep=True)) is needed where there is an activation")
        ldp = _kept("pre", pre, x, (rows, cout))
    return _dense_backward(dtype, (rows, cin, cout), dy, lddy, x if need_w else None, ldx, w if need_x else None, ldw, transposed,
                           pre if act else None, ldp, act, bias, need_x, need_w)


def _dense_backward(dtype, sizes, dy, lddy, x, ldx, w, ldw, transposed, pre, ldp, act, bias, need_x, need_w):
    """The call of dense_grad: x is there for dw only, w for dx only."""
    lib = _lib.load()
    rows, cin, cout = sizes
    with torch.no_grad():
        dx = torch.empty((rows, cin), dtype=dy.dtype, device=dy.device) if need_x else None
        dw = _weight_gradient(dy, cin, cout, transposed) if need_w else None
        db = torch.empty(cout, dtype=dy.dtype, device=dy.device) if bias else None
    whole = _whole(dtype, (cin, cout), (x, ldx), (w, ldw), (dy, lddy))
    size = lib.fpn_dense_grad_workspace_bytes(dtype, rows, cin, cout, act, whole)
    ws = _workspace(size, dy)
    _call(dy, lib.fpn_dense_grad, dtype, rows, cin, cout, _p(dy), lddy, _p(x), ldx, _p(w), ldw, transposed, _p(pre), ldp, act, _p(dx), cin,
          _p(dw), cin if transposed else cout, _p(db), _p(ws), size)
    return dx, dw, db


def _kept(name, t, x, shape):
    """The row stride of a pre-activation that a forward pass kept."""
    if isinstance(t, torch.Tensor):
        _as_it_is(name, t)
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or not t.is_cuda or t.get_device() != x.get_device() or t.shape != shape:
        raise ValueError("%s must be the float32 %s tensor on %s that keep=True returned" % (name, tuple(shape), x.device))
    return _rows(name, t)


def _weight_gradient(like, cin, cout, transposed):
    """A (cin, cout) matrix in the weights' storage order."""
    if transposed:
        return torch.empty((cout, cin), dtype=like.dtype, device=like.device).t()
    return torch.empty((cin, cout), dtype=like.dtype, device=like.device)


def _dense_rows(t):
    """A gradient as autograd hands it over (it may be an expanded, transposed or negated view), with dense rows."""
    t = t.resolve_neg()
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        return t.contiguous()
    return t


class _Dense(torch.autograd.Function):
    """Keeps what the gradients that will be asked for are formed from, and nothing else."""

    @staticmethod
    def forward(ctx, x, w, bias, activation, residual):
        need_x, need_w, need_b, _, _ = ctx.needs_input_grad
        act = ACTIVATIONS[activation]
        pre = None
        if act and (need_x or need_w or need_b):
            y, pre = dense(x, w, bias, activation, residual, keep=True)
        else:
            y = dense(x, w, bias, activation, residual)
        ctx.save_for_backward(x if need_w else None, w if need_x else None, pre)
        # (dw is stored as w is: a kept w says how)
        order = _weights(("w",), (w,))[0] if need_w and not need_x else 0
        ctx.layout = _DTYPES[x.dtype], (x.shape[0], x.shape[1], w.shape[1]), order, act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _no_capture()
        x, w, pre = ctx.saved_tensors
        need_x, need_w, need_b, _, need_r = ctx.needs_input_grad
        dx = dw = db = None
        if need_x or need_w or need_b:
            dx, dw, db = _dense_gradients(ctx.layout, _dense_rows(dy), x if need_w else None, w if need_x else None, pre, need_b)
        return dx, dw, db, None, dy if need_r else None


def _dense_gradients(layout, dy, x, w, pre, bias):
    """dense_grad on what an autograd function kept: dw where x is given, dx where w is.  (Hooks on saved tensors may have
    brought back copies laid out otherwise.)"""
    dtype, (rows, cin, cout), transposed, act = layout
    _tensor("dy", dy, dy, (rows, cout))
    ldx = ldw = 0
    if x is not None:
        _tensor("x", x, dy, (rows, cin))
        ldx = _rows("x", x, broadcast=True)
    if w is not None:
        _tensor("w", w, dy, (cin, cout))
        transposed, (ldw,) = _weights(("w",), (w,))
    ldp = _kept("pre", pre, dy, (rows, cout)) if act else cout
    return _dense_backward(dtype, (rows, cin, cout), dy, _rows("dy", dy), x, ldx, w, ldw, transposed, pre if act else None, ldp, act, bias,
                           w is not None, x is not None)


# ---- gated ---------------------------------------------------------------------------------------------------------

def _check_gated(x, w_gate, w_up):
    dtype = _first("x", x)
    for name, w in (("w_gate", w_gate), ("w_up", w_up)):
        if not isinstance(w, torch.Tensor) or w.dim() != 2:
            raise ValueError("%s must be a (cin, cout) tensor" % name)
        _tensor(name, w, x, (x.shape[1], w_gate.shape[1]))
    return dtype, x.shape[0], x.shape[1], w_gate.shape[1]


def gated(x, w_gate, w_up, bias_gate=None, bias_up=None, activation="silu", out=None, keep=False):
    """h = act(x w_gate + bias_gate) * (x w_up + bias_up) in one kernel: x (rows, cin), weights (cin, cout) - both the
    same way round, columns of one matrix will do -, biases (cout,), h (rows, cout).

    `out` receives h (it may share memory with no argument).  keep=True returns (h, gate, up) for `gated_grad`, the two
    sums in float32."""
    dtype, rows, cin, cout = _check_gated(x, w_gate, w_up)
    act = _activation(activation)
    lib = _lib.load()
    _vector("bias_gate", bias_gate, x, cout)
    _vector("bias_up", bias_up, x, cout)
    if not keep and _recorded(x, w_gate, w_up, bias_gate, bias_up):
        if out is not None:
            raise ValueError("out cannot be given for tensors that require gradients")
        return _Gated.apply(x, w_gate, w_up, bias_gate, bias_up, activation)
    ldx = _rows("x", x, broadcast=True)
    transposed, (ldg, ldu) = _weights(("w_gate", "w_up"), (w_gate, w_up))
    h, ldh = _output(out, x, rows, cout, (("x", x), ("w_gate", w_gate), ("w_up", w_up), ("bias_gate", bias_gate), ("bias_up", bias_up)))
    gate = up = None
    if keep:
        gate, up = (torch.empty((rows, cout), dtype=torch.float32, device=x.device) for _ in range(2))
    size = lib.fpn_gated_workspace_bytes(dtype, rows, cin, cout, _whole(dtype, (cin, cout), (x, ldx), (w_gate, ldg), (w_up, ldu)))
    ws = _workspace(size, x)
    _call(x, lib.fpn_gated, dtype, rows, cin, cout, _p(x), ldx, _p(w_gate), ldg, _p(w_up), ldu, transposed, _p(bias_gate), _p(bias_up), act,
          _p(h), ldh, _p(gate), _p(up), cout, _p(ws), size)
    return (h, gate, up) if keep else h


def gated_grad(dh, x, w_gate, w_up, gate, up, activation="silu", bias=False, need_x=True, need_w=True, w_down=None):
    """The gradients of `gated`: (dx, dw_gate, dw_up, dbias_gate, dbias_up), each None where it is not asked for
    (bias=True asks for the last two).  `gate` and `up` are what keep=True returned.

    With w_down (cout, cdown) the first argument is the gradient of gated(...) @ w_down: the way back through that product
    is taken on the way, without rounding its result."""
    dtype, rows, cin, cout = _check_gated(x, w_gate, w_up)
    act = _activation(activation)
    lib = _lib.load()
    cdown, ldd, down_transposed = 0, 0, 0
    if w_down is not None:
        if not isinstance(w_down, torch.Tensor) or w_down.dim() != 2:
            raise ValueError("w_down must be a (cout, cdown) tensor")
        cdown = w_down.shape[1]
        _tensor("w_down", w_down, x, (cout, cdown))
        down_transposed, (ldd,) = _weights(("w_down",), (w_down,))
    _tensor("dh", dh, x, (rows, cdown or cout))
    ldp = _kept("gate", gate, x, (rows, cout))
    if _kept("up", up, x, (rows, cout)) != ldp:
        raise ValueError("gate and up must have the same row stride")
    lddh, ldx = _rows("dh", dh), _rows("x", x, broadcast=True)
    transposed, (ldg, ldu) = _weights(("w_gate", "w_up"), (w_gate, w_up))
    return _gated_backward(dtype, (rows, cin, cout, cdown), dh, lddh, w_down, ldd, down_transposed, x if need_w else None, ldx,
                           (w_gate, w_up) if need_x else (None, None), (ldg, ldu), transposed, gate, up, ldp, act, bias, need_x, need_w)


def _gated_backward(dtype, sizes, dh, lddh, w_down, ldd, down_transposed, x, ldx, ws, lds, transposed, gate, up, ldp, act, bias, need_x,
                    need_w):
    """The call of gated_grad: x is there for the weights' gradients only, the weights `ws` for dx only."""
    lib = _lib.load()
    rows, cin, cout, cdown = sizes
    with torch.no_grad():
        dx = torch.empty((rows, cin), dtype=dh.dtype, device=dh.device) if need_x else None
        dwg, dwu = (_weight_gradient(dh, cin, cout, transposed) for _ in range(2)) if need_w else (None, None)
        dbg, dbu = (torch.empty(cout, dtype=dh.dtype, device=dh.device) for _ in range(2)) if bias else (None, None)
    whole = _whole(dtype, (cin, cout, cdown), (x, ldx), (ws[0], lds[0]), (ws[1], lds[1]), (dh, lddh), (w_down, ldd))
    size = lib.fpn_gated_grad_workspace_bytes(dtype, rows, cin, cout, cdown, whole)
    space = _workspace(size, dh)
    _call(dh, lib.fpn_gated_grad, dtype, rows, cin, cout, cdown, _p(dh), lddh, _p(w_down), ldd, down_transposed, _p(x), ldx, _p(ws[0]),
          lds[0], _p(ws[1]), lds[1], transposed, _p(gate), _p(up), ldp, act, _p(dx), cin, _p(dwg), _p(dwu), cin if transposed else cout,
          _p(dbg), _p(dbu), _p(space), size)
    return dx, dwg, dwu, dbg, dbu


class _Gated(torch.autograd.Function):
    """Keeps what the gradients that will be asked for are formed from, and nothing else."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, bias_gate, bias_up, activation):
        need_x, need_g, need_u = ctx.needs_input_grad[:3]
        h, gate, up = gated(x, w_gate, w_up, bias_gate, bias_up, activation, keep=True)
        ctx.save_for_backward(x if need_g or need_u else None, w_gate if need_x else None, w_up if need_x else None, None, gate, up)
        ctx.layout = _gated_layout(x, w_gate, w_up, 0, activation, need_x)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        _no_capture()
        return _gated_gradients(ctx.layout, _dense_rows(dh), ctx.saved_tensors, ctx.needs_input_grad[:5]) + (None,)


def _gated_layout(x, w_gate, w_up, cdown, activation, need_x):
    """(dtype, sizes, storage order of the gated weights, activation) of a recorded call."""
    order = 0 if need_x else _weights(("w_gate", "w_up"), (w_gate, w_up))[0]             # (with need_x they are kept and say it)
    return _DTYPES[x.dtype], (x.shape[0], x.shape[1], w_gate.shape[1], cdown), order, ACTIVATIONS[activation]


def _gated_gradients(layout, dh, saved, needs):
    """gated_grad on what an autograd function kept: the gradients of x, w_gate, w_up, bias_gate and bias_up that are asked
    for."""
    dtype, sizes, transposed, act = layout
    rows, cin, cout, cdown = sizes
    x, w_gate, w_up, w_down, gate, up = saved
    need_x, need_g, need_u, need_bg, need_bu = needs
    need_w = need_g or need_u
    _tensor("dh", dh, dh, (rows, cdown or cout))
    ldx, lds, ldd, down_transposed = 0, (0, 0), 0, 0
    if need_w:
        _tensor("x", x, dh, (rows, cin))
        ldx = _rows("x", x, broadcast=True)
    if need_x:
        _tensor("w_gate", w_gate, dh, (cin, cout))
        _tensor("w_up", w_up, dh, (cin, cout))
        transposed, lds = _weights(("w_gate", "w_up"), (w_gate, w_up))
    if cdown:
        _tensor("w_down", w_down, dh, (cout, cdown))
        down_transposed, (ldd,) = _weights(("w_down",), (w_down,))
    ldp = _kept("gate", gate, dh, (rows, cout))
    if _kept("up", up, dh, (rows, cout)) != ldp:
        raise ValueError("gate and up must have the same row stride")
    dx, dwg, dwu, dbg, dbu = _gated_backward(dtype, sizes, dh, _rows("dh", dh), w_down, ldd, down_transposed, x if need_w else None, ldx,
                                             (w_gate, w_up) if need_x else (None, None), lds, transposed, gate, up, ldp, act,
                                             need_bg or need_bu, need_x, need_w)
    return dx, dwg if need_g else None, dwu if need_u else None, dbg if need_bg else None, dbu if need_bu else None


# ---- the block -----------------------------------------------------------------------------------------------------

def gated_feed_forward(x, w_gate, w_up, w_down, bias_gate=None, bias_up=None, bias_down=None, activation="silu", residual=None,
                       out=None):
    """y = gated(x) w_down + bias_down + residual: `gated` and then `dense` with the residual in its epilogue."""
    if forward_ad._current_level >= 0:                       # (before anything is recorded or launched)
        for name, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down), ("bias_gate", bias_gate),
                        ("bias_up", bias_up), ("bias_down", bias_down), ("residual", residual), ("out", out)):
            _no_tangent(name, t)
    if isinstance(x, torch.Tensor) and isinstance(w_down, torch.Tensor) and \
            _recorded(x, w_gate, w_up, w_down, bias_gate, bias_up, bias_down, residual):
        if out is not None:
            raise ValueError("out cannot be given for tensors that require gradients")
        return _GatedFeedForward.apply(x, w_gate, w_up, w_down, bias_gate, bias_up, bias_down, activation, residual)
    h = gated(x, w_gate, w_up, bias_gate, bias_up, activation)
    return dense(h, w_down, bias_down, None, residual, out)


class _GatedFeedForward(torch.autograd.Function):
    """Keeps what the gradients that will be asked for are formed from, and nothing else."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, bias_gate, bias_up, bias_down, activation, residual):
        need_x, need_g, need_u, need_d, need_bg, need_bu = ctx.needs_input_grad[:6]
        gate = up = None
        through = need_x or need_g or need_u or need_bg or need_bu       # (a gradient goes back through h)
        if through:
            h, gate, up = gated(x, w_gate, w_up, bias_gate, bias_up, activation, keep=True)
        else:
            h = gated(x, w_gate, w_up, bias_gate, bias_up, activation)
        y = dense(h, w_down, bias_down, None, residual)
        ctx.save_for_backward(x if need_g or need_u else None, w_gate if need_x else None, w_up if need_x else None,
                              w_down if through else None, gate, up, h if need_d else None)
        ctx.layout = _gated_layout(x, w_gate, w_up, w_down.shape[1], activation, need_x)
        ctx.down_transposed = _weights(("w_down",), (w_down,))[0]
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _no_capture()
        *saved, h = ctx.saved_tensors
        need_x, need_g, need_u, need_d, need_bg, need_bu, need_bd, _, need_r = ctx.needs_input_grad
        dtype, (rows, _, hidden, cout), _, _ = ctx.layout
        dx = dwg = dwu = dwd = dbg = dbu = dbd = None
        d = _dense_rows(dy)
        if need_d or need_bd:
            layout = dtype, (rows, hidden, cout), ctx.down_transposed, 0
            _, dwd, dbd = _dense_gradients(layout, d, h if need_d else None, None, None, need_bd)
        if need_x or need_g or need_u or need_bg or need_bu:
            dx, dwg, dwu, dbg, dbu = _gated_gradients(ctx.layout, d, saved, (need_x, need_g, need_u, need_bg, need_bu))
        return dx, dwg, dwu, dwd, dbg, dbu, dbd, None, dy if need_r else None
