"""The decay's gradient of the gated recurrence is a sum over sequences and steps that loses no bits
to their number or order."""
import pytest
import torch

from test_gpu_gated import make, put

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("L", [1, 40, 64, 300, 1500])
def test_sequences_that_cancel(cuda, L):
    """Two sequences with gradients of 2^20 and -2^20 times the same rows leave the third's: their
    sums of a chunk cancel to the last bit, and 64 bits keep the third's beside them.  The result
    is rounded once more than the third's alone (2^-24), its sums in 64 bits are off by 2^-53 for
    each of less than 100 additions of at most 2^20 * 2^7 times it."""
    from mamba_int import ops
    s = make(3, L, 70, torch.float32, L, state=False)
    for k in ("x", "r", "i", "z"):
        s[k][2] = s[k][0]
    s["dy"][0] *= 2.0 ** 20
    s["dy"][2] = -s["dy"][0]
    d = put(s, cuda)

    def gradient(at):
        decay = d["decay"].detach().requires_grad_()
        y = ops.gated_scan(d["x"][at], d["r"][at], d["i"][at], decay, z=d["z"][at])
        return torch.autograd.grad(y, decay, d["dy"][at])[0].double()
    got, alone = gradient(slice(0, 3)), gradient(slice(1, 2))
    # (a channel whose own steps nearly cancel is small against what the others' sums may leave)
    assert ((got - alone).abs() <= 2.0 ** -23 * alone.abs() + 2.0 ** -19 * alone.abs().mean()).all()
