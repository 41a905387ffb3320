"""What the feed-forward operators keep for their backward passes: no more than the gradients that are asked for need, so
that a tensor which no gradient needs may be written in place meanwhile, and nothing is held for nobody."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

DENSE = ("x", "w", "bias", "residual")
GATED = ("x", "w_gate", "w_up", "bias_gate", "bias_up")
BLOCK = ("x", "w_gate", "w_up", "w_down", "bias_gate", "bias_up", "bias_down", "residual")
SHAPES = {"x": (37, 24), "w": (24, 40), "bias": (40,), "residual": (37, 24), "w_gate": (24, 40), "w_up": (24, 40), "bias_gate": (40,),
          "bias_up": (40,), "w_down": (40, 24), "bias_down": (24,)}


def operands(device, names, dtype=torch.float32, cols=False):
    g = torch.Generator().manual_seed(21)

    def make(name):
        shape = (37, 40) if name == "residual" and names is DENSE else SHAPES[name]
        t = (torch.randn(shape, generator=g) * 0.3).to(dtype).to(device)
        return t.t().contiguous().t() if cols and name.startswith("w") else t
    return {name: make(name) for name in names}


def call(names, a, act):
    from fpn import feed_forward as F
    if names is DENSE:
        return F.dense(a["x"], a["w"], a["bias"], act, a["residual"])
    if names is GATED:
        return F.gated(a["x"], a["w_gate"], a["w_up"], a["bias_gate"], a["bias_up"], act)
    return F.gated_feed_forward(a["x"], a["w_gate"], a["w_up"], a["w_down"], a["bias_gate"], a["bias_up"], a["bias_down"], act, a["residual"])


def reads(names, wanted, act):
    """The arguments whose values the gradients of `wanted` are formed from."""
    used = set()
    if names is DENSE:
        if "x" in wanted:
            used.add("w")
        if "w" in wanted:
            used.add("x")
        return used
    if wanted & {"w_gate", "w_up"}:
        used.add("x")
    if "x" in wanted:
        used |= {"w_gate", "w_up"}
    if names is BLOCK and wanted & {"x", "w_gate", "w_up", "bias_gate", "bias_up"}:
        used.add("w_down")
    return used


def subsets(names):
    if names is BLOCK:
        yield from (set(c) for c in itertools.combinations(names, 1))
        yield from ({"x", "w_down"}, {"w_gate", "residual"}, {"bias_down", "residual"}, {"x", "w_gate", "w_up"}, set(names))
    else:
        for n in range(1, len(names) + 1):
            yield from (set(c) for c in itertools.combinations(names, n))


@pytest.mark.parametrize("cols", [False, True])
@pytest.mark.parametrize("names", [DENSE, GATED, BLOCK], ids=["dense", "gated", "block"])
def test_any_set_of_gradients_with_the_rest_written_in_place(device, names, cols):
    """Each gradient is the one of the call that asks for all, bit for bit, though every argument that no wanted gradient is
    formed from is overwritten between the passes; one that is needed is missed if it was overwritten."""
    for act in ("silu", None):
        a = operands(device, names, cols=cols)
        full = {k: v.detach().clone(memory_format=torch.preserve_format).requires_grad_() for k, v in a.items()}
        y = call(names, full, act)
        dy = torch.linspace(-1, 1, y.numel(), device=device).reshape(y.shape)
        want = dict(zip(names, torch.autograd.grad(y, list(full.values()), dy)))
        for wanted in subsets(names):
            # (results of an operation, so that those which require gradients may be written in place too)
            leaves = {k: v.detach().clone(memory_format=torch.preserve_format).requires_grad_(k in wanted) for k, v in a.items()}
            b = {k: v * 1 for k, v in leaves.items()}
            assert torch.equal(call(names, b, act), y)
            out = call(names, b, act)
            needed = reads(names, wanted, act)
            with torch.no_grad():
                for k in names:
                    if k not in needed:
                        b[k].fill_(float("nan"))
            got = torch.autograd.grad(out, [leaves[k] for k in sorted(wanted)], dy)
            for k, g in zip(sorted(wanted), got):
                assert torch.equal(g, want[k]), (sorted(wanted), k)
            for k in sorted(needed):
                b = {n: v * 1 for n, v in leaves.items()}
                out = call(names, b, act)
                with torch.no_grad():
                    b[k].add_(1)
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    torch.autograd.grad(out, [leaves[n] for n in sorted(wanted)], dy)


def test_pre_activations_are_kept_for_a_gradient_only(device):
    """A call of which only the residual (or the last bias) requires gradients holds its result and nothing else."""
    from fpn import feed_forward as F
    rows, cin, hidden = 4096, 64, 1024
    x, w = torch.randn((rows, cin), device=device), torch.randn((cin, hidden), device=device)
    wd, bd = torch.randn((hidden, cin), device=device), torch.zeros(cin, device=device, requires_grad=True)
    r, rx = (torch.zeros((rows, n), device=device, requires_grad=True) for n in (hidden, cin))
    for f in (lambda: F.dense(x, w, None, "gelu", r), lambda: F.gated_feed_forward(x, w, w, wd, None, None, bd, "silu", rx)):
        f()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = f()
        assert torch.cuda.memory_allocated() - before <= y.numel() * 4 + 1024
        del y


@pytest.mark.parametrize("names", [DENSE, GATED, BLOCK], ids=["dense", "gated", "block"])
def test_saved_tensors_that_come_back_laid_out_otherwise(device, names):
    """Hooks that keep copies (offloading does) bring back weights held (out,in) as (in,out) matrices, and rows apart."""
    def unpack(t):
        wide = torch.full(t.shape[:-1] + (t.shape[-1] + 3,), float("nan"), dtype=t.dtype, device=device)
        wide[..., :t.shape[-1]] = t
        return wide[..., :t.shape[-1]]
    for cols in (False, True):
        for wanted in (set(names), {"x"}, {names[1]}):
            leaves = {k: v.requires_grad_(k in wanted) for k, v in operands(device, names, cols=cols).items()}
            y = call(names, leaves, "gelu")
            dy = torch.linspace(-1, 1, y.numel(), device=device).reshape(y.shape)
            want = torch.autograd.grad(y, [leaves[k] for k in sorted(wanted)], dy)
            for hook in (unpack, torch.Tensor.contiguous):
                with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(memory_format=torch.contiguous_format), hook):
                    y = call(names, leaves, "gelu")
                got = torch.autograd.grad(y, [leaves[k] for k in sorted(wanted)], dy)
                for a, b in zip(got, want):
                    # (another kernel may read other strides: fp32 sums of at most 40 products)
                    assert (a - b).norm() <= 1e-6 * b.norm()


def test_saved_tensors_that_come_back_wrong_are_refused(device):
    from fpn import feed_forward as F
    x, w = torch.ones((6, 8), device=device, requires_grad=True), torch.ones((8, 4), device=device, requires_grad=True)
    for hook in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t[:2]):
        for f in (lambda: F.dense(x, w, activation="silu"), lambda: F.gated(x, w, w), lambda: F.gated_feed_forward(x, w, w, w.t())):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), hook):
                y = f()
            with pytest.raises(ValueError):
                y.sum().backward()
