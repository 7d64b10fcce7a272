"""Arguments of the float operators' calls that are refused before a tensor's device is looked at."""
import pytest
import torch


def test_an_error_in_a_truth_value_is_raised():
    """... and not covered by a result."""
    from mamba_int import ops
    x = torch.zeros(1, 3, 8)
    with pytest.raises(RuntimeError, match="ambiguous"):
        ops.selective_scan(x, x, torch.zeros(8, 4), torch.zeros(1, 3, 4), torch.zeros(1, 3, 4), dt_softplus=torch.ones(2))


def test_traced_calls_are_refused():
    """A trace would hold the result as a constant.  (Outside one, the host tensor is what is refused.)"""
    from mamba_int import ops
    x, w = torch.zeros(3, 8), torch.zeros(8)

    def f(v):
        return ops.add_rms_norm(v, w)[0]
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(f, (x,))
    with pytest.raises(ValueError, match="device"):
        f(x)
