"""tf_util's dense layers: what they take from the variable store and which arguments they refuse, decided on the host."""
import pytest
import torch

from fpn import tf_util, variables


def store_with(weights, biases):
    store = variables.VariableStore("cpu")
    store["layer/weights"], store["layer/biases"] = weights, biases
    return store


def hold(store, name, parameter):
    """A trained parameter in the store itself, as a program that trains the layer holds it."""
    store._vars[name] = parameter


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_layer_sees_its_variables_as_they_are_now(dtype):
    """Updated in place (an optimiser's step, .data, the store's own tensor), by assignment, or replaced."""
    store = store_with(torch.ones(4, 3), torch.zeros(3))
    with variables.use_store(store):
        w, b = tf_util._projection("layer", 4, 3, True, dtype)
        assert w.dtype is dtype and b.dtype is dtype and (w == 1).all() and not b.any()
        with torch.no_grad():
            store["layer/weights"].add_(1)
            store["layer/biases"].fill_(5)
        w, b = tf_util._projection("layer", 4, 3, True, dtype)
        assert (w == 2).all() and (b == 5).all()
        store["layer/weights"].data.fill_(7)                # (leaves the version counter as it was)
        assert (tf_util._projection("layer", 4, 3, True, dtype)[0] == 7).all()
        hold(store, "layer/weights", torch.nn.Parameter(torch.full((4, 3), 3.0)))
        assert (tf_util._projection("layer", 4, 3, True, dtype)[0] == 3).all()
        step = torch.optim.SGD([store["layer/weights"]], lr=1.0)
        store["layer/weights"].grad = torch.ones(4, 3)
        step.step()
        assert (tf_util._projection("layer", 4, 3, True, dtype)[0] == 2).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_a_first_call_without_gradients_does_not_cost_later_ones_theirs(dtype, mode):
    store = store_with(torch.ones(4, 3), torch.zeros(3))
    for name in ("layer/weights", "layer/biases"):
        hold(store, name, torch.nn.Parameter(store[name].clone()))
    with variables.use_store(store):
        with mode():
            tf_util._projection("layer", 4, 3, True, dtype)
        for _ in range(2):                                  # (a second step has a graph of its own)
            w, b = tf_util._projection("layer", 4, 3, True, dtype)
            assert w.requires_grad and b.requires_grad and not w.is_inference()
            (w.float().sum() + b.float().sum()).backward()
        assert (store["layer/weights"].grad == 2).all() and (store["layer/biases"].grad == 2).all()


def test_frozen_variables_after_inference_mode():
    """A cast that inference mode made could not be saved for a backward pass of the points."""
    store = store_with(torch.ones(4, 3), torch.zeros(3))
    with variables.use_store(store):
        with torch.inference_mode():
            tf_util._projection("layer", 4, 3, True, torch.bfloat16)
        w, _ = tf_util._projection("layer", 4, 3, True, torch.bfloat16)
    assert not w.is_inference()


def test_variables_made_inside_inference_mode_are_ordinary_tensors():
    """A layer's first call makes its variables: made in inference mode they could never be saved for a backward pass."""
    store = variables.VariableStore("cpu")
    with variables.use_store(store):
        with torch.inference_mode():
            tf_util._projection("layer", 4, 3, True, torch.float32)
            store["given"] = torch.ones(2)
        for name in ("layer/weights", "layer/biases", "given"):
            assert not store[name].is_inference(), name
        w, _ = tf_util._projection("layer", 4, 3, True, torch.float32)
        (torch.ones(2, 4, requires_grad=True) @ w).sum().backward()


@pytest.mark.parametrize("points,residual", [((4, 8, 5), (8, 4, 3)), ((4, 8, 5), (2, 16, 3)), ((4, 8, 5), (1, 4, 8, 3)), ((32, 5), (4, 8, 3)),
                                             ((4, 8, 5), (4, 8, 2))])
def test_a_residual_of_other_rows_is_refused(points, residual):
    """As many rows, but not the inputs' own: adding them row by row would pair the wrong ones."""
    with variables.use_store(variables.VariableStore("cpu")):
        with pytest.raises(ValueError, match="residual has shape"):
            tf_util.dense(torch.zeros(points), 3, "layer", residual=torch.zeros(residual))
        with pytest.raises(ValueError, match="residual has shape"):
            tf_util.gated_feed_forward(torch.zeros(points), 6, "block", num_outputs=3, residual=torch.zeros(residual))


@pytest.mark.parametrize("points,residual", [((4, 8, 5), (4, 8, 3)), ((4, 8, 5), (32, 3)), ((32, 5), (32, 3))])
def test_a_residual_of_the_same_rows_passes_the_check(points, residual):
    """(a matrix of all rows is the same rows; behind the check comes the refusal of host tensors)"""
    with variables.use_store(variables.VariableStore("cpu")):
        with pytest.raises(ValueError, match="ROCm device"):
            tf_util.dense(torch.zeros(points), 3, "layer", residual=torch.zeros(residual))
