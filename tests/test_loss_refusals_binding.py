"""What the binding of the choice losses refuses by itself (no GPU)."""
import pytest

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("grad", [False, 0, "in place"])
def test_gradient_targets_that_are_no_tensors(dp, grad):
    with pytest.raises(dp.DPError, match="grad must be a tensor"):
        dp._grad_out(torch.zeros(2, 3), grad, False)
