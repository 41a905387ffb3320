"""tf_util's dense layers on the GPU: training their variables, captures and streams."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def trained(device, dtype, seed=0):
    """A store whose variables are parameters, and points of the layer's type."""
    from fpn import variables
    g = torch.Generator().manual_seed(seed)
    store = variables.VariableStore(device)
    for name, shape in (("head/weights", (24, 16)), ("head/biases", (16,))):
        store[name] = torch.randn(shape, generator=g) * 0.2
        store._vars[name] = torch.nn.Parameter(store[name].clone())
    return store, torch.randn((40, 24), generator=g).to(dtype).to(device), torch.randn((40, 16), generator=g).to(dtype).to(device)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_a_layer_trains_its_variables(device, t):
    """Two steps, the first behind a call without gradients: the float32 variables get the gradients of the operator on
    their casts (the same call on leaves of the layer's type), and the second step runs on the stepped weights."""
    from fpn import feed_forward as F
    from fpn import tf_util, variables
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[t]
    store, x, dy = trained(device, dtype)
    w, b = store["head/weights"], store["head/biases"]
    step = torch.optim.SGD([w, b], lr=0.5)
    with variables.use_store(store):
        with torch.inference_mode():
            tf_util.dense(x, 16, "head", "gelu")
        for _ in range(2):
            step.zero_grad()
            y = tf_util.dense(x, 16, "head", "gelu")
            y.backward(dy)
            wc, bc = (v.detach().to(dtype).requires_grad_() for v in (w, b))
            want = F.dense(x, wc, bc, "gelu")
            assert torch.equal(y, want)
            dw, db = torch.autograd.grad(want, (wc, bc), dy)
            assert torch.equal(w.grad, dw.float()) and torch.equal(b.grad, db.float())
            step.step()


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_a_layer_first_called_in_a_capture(device, t):
    """Its cast belongs to the graph: an eager call before the first replay has its own, and a replay sees the variables as
    they are then."""
    from fpn import tf_util, variables
    dtype = {"bf16": torch.bfloat16, "f16": torch.float16}[t]
    store, x, _ = trained(device, dtype, seed=1)
    store["head/weights"] = store["head/weights"].detach()
    store["head/biases"] = store["head/biases"].detach()
    with variables.use_store(store), torch.no_grad():
        tf_util.dense(x, 16, "head", use_bias=False)         # (kernels loaded; another cast of the weights than the graph's)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            inside = tf_util.dense(x, 16, "head", "silu")
        for r in range(3):
            eager = tf_util.dense(x, 16, "head", "silu")
            want = torch.nn.functional.silu(x.double() @ store["head/weights"].to(dtype).double() + store["head/biases"].to(dtype).double())
            # one rounding of the result, fp32 sums of 24 products
            u = torch.finfo(dtype).eps / 2
            assert ((eager.double() - want).abs() <= u * want.abs() + 1e-5).all()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(inside, eager)
            store["head/weights"].mul_(-0.5)                 # in place, between the replays


def test_a_layer_called_on_two_streams(device):
    """Calls on different streams share nothing that one of them still writes."""
    from fpn import tf_util, variables
    store, x, _ = trained(device, torch.bfloat16, seed=2)
    side = torch.cuda.Stream()
    with variables.use_store(store), torch.no_grad():
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            a = tf_util.dense(x, 16, "head")
        b = tf_util.dense(x, 16, "head")
        torch.cuda.synchronize()
    assert torch.equal(a, b)
