"""Forward-mode differentiation: the feed-forward operators have no tangents, and a tensor that carries one is refused
(the call would return a result without a tangent, which means a derivative of zero)."""
import pytest
import torch
from torch.autograd import forward_ad


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


def test_every_check_of_a_tensor_refuses_a_tangent():
    from fpn import feed_forward as F
    x, w = torch.ones(4, 8), torch.ones(8, 16)
    with forward_ad.dual_level():
        for call in (lambda t: F._first("x", t), lambda t: F._tensor("x", t, x, (4, 8)), lambda t: F._kept("x", t, x, (4, 8)),
                     lambda t: F.dense(t, w), lambda t: F.gated(t, w, w), lambda t: F.gated_feed_forward(t, w, w, w.t()),
                     lambda t: F.dense_grad(x, t, w), lambda t: F.gated_grad(x, t, w, w, x, x)):
            with pytest.raises(NotImplementedError, match="x carries a tangent"):
                call(dual(x))
        with pytest.raises(ValueError, match="ROCm device"):           # (a tensor without one goes on to the next check)
            F.dense(x, w)


def test_layers_refuse_a_tangent():
    from fpn import tf_util, variables
    with variables.use_store(variables.VariableStore("cpu")), forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="x carries a tangent"):
            tf_util.dense(dual(torch.ones(2, 3, 8)), 4, "layer")


@pytest.mark.gpu
def test_each_argument_with_a_tangent_is_refused(device):
    from fpn import feed_forward as F

    def ones(*shape):
        return torch.ones(shape, device=device)
    x, w, b, r, wd = ones(4, 8), ones(8, 16), ones(16), ones(4, 16), ones(16, 8)
    plain = F.dense(x, w, b, "silu", r)
    _, pre = F.dense(x, w, b, "silu", keep=True)
    _, gate, up = F.gated(x, w, w, keep=True)
    calls = {
        F.dense: dict(x=x, w=w, bias=b, residual=r, out=ones(4, 16)),
        F.dense_grad: dict(dy=r, x=x, w=w, pre=pre),
        F.gated: dict(x=x, w_gate=w, w_up=w, bias_gate=b, bias_up=b, out=ones(4, 16)),
        F.gated_grad: dict(dh=x, x=x, w_gate=w, w_up=w, gate=gate, up=up, w_down=wd),
        F.gated_feed_forward: dict(x=x, w_gate=w, w_up=w, w_down=wd, bias_gate=b, bias_up=b, bias_down=ones(8), residual=x, out=ones(4, 8)),
    }
    more = {F.dense_grad: dict(activation="silu"), F.dense: dict(activation="silu")}
    with forward_ad.dual_level():
        for call, arguments in calls.items():
            call(**arguments, **more.get(call, {}))
            for name in arguments:
                with pytest.raises(NotImplementedError, match="carries a tangent"):
                    call(**{**arguments, name: dual(arguments[name])}, **more.get(call, {}))
                if name == "out":
                    continue
                recorded = {k: v for k, v in arguments.items() if k != "out"}
                recorded[name] = dual(arguments[name].clone().requires_grad_())
                with pytest.raises(NotImplementedError, match="carries a tangent"):
                    call(**recorded, **more.get(call, {}))
        assert torch.equal(F.dense(x, w, b, "silu", r), plain)         # a level without tangents changes nothing
