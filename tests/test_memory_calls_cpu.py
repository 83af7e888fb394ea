"""Calls of the policy memory's operators that are refused before anything reaches a GPU."""
import pytest

torch = pytest.importorskip("torch")

from ilrl_amd import memory as M  # noqa: E402


@pytest.mark.parametrize("x,weight,param", [
    (torch.bfloat16, torch.bfloat16, torch.float32), (torch.float16, torch.float16, torch.float32),
    (torch.bfloat16, torch.float32, torch.bfloat16), (torch.float16, torch.float32, torch.float16),
    (torch.bfloat16, None, torch.float16), (torch.float32, None, torch.bfloat16), (torch.float32, None, torch.float64),
    (torch.bfloat16, None, torch.int32), (torch.float32, torch.float32, torch.float64)])
def test_norm_gradient_refuses_a_parameter_type_that_is_not_the_weights(x, weight, param):
    """One type describes the weight and both of its gradients to the kernel: another one's rows would be read past their
    end or as other numbers."""
    a = torch.zeros(3, 8, dtype=x)
    w = torch.zeros(8, dtype=weight) if weight is not None else None
    with pytest.raises(ValueError, match="param_dtype"):
        M.layer_norm_backward(a, a, torch.zeros(3), torch.ones(3), w, param_dtype=param)
