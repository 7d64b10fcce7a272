"""Infinite inputs, states and gradients of the gated recurrence, as the formulas in 64 bits have them."""
import math

import pytest
import torch

import gated_ref as G
from test_gpu_float_nonfinite import same

pytestmark = pytest.mark.gpu

# L: a token; a wave; four waves; a block of sixteen; chunks of the backward pass; chunks of both
LENGTHS = [1, 13, 60, 200, 700, 2000]
FAST = 3.0                                  # with r = 0 a step leaves 5e-6 of a state
MEDIUM = math.log(math.expm1(0.5))          # ... and exp(-2) of it


def make(L, decay, D=9, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return (0.1 + 0.9 * torch.rand(*shape, generator=g)).to(dtype)
    return {"x": rand(2, L, D), "r": torch.zeros(2, L, D, dtype=dtype), "i": rand(2, L, D), "decay": torch.full((D,), decay),
            "h_in": rand(2, D).float()}


def forward(s, cuda, **more):
    from mamba_int import ops
    h = torch.zeros(2, s["x"].shape[2], device=cuda)
    y = ops.gated_scan(**{k: v.to(cuda) for k, v in s.items()}, h_out=h, **more)
    return y, h


@pytest.mark.parametrize("L", LENGTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinite_input(cuda, L, dtype):
    """Infinite from that step on, however small a decay of many steps is."""
    s = make(L, FAST, dtype=dtype, seed=L)
    t = L // 5
    s["x"][1, t, 4] = float("inf")
    s["x"][0, L - 1, 2] = -float("inf")
    want = G.gated(**s)
    assert torch.isinf(want["y"][0][1, t:, 4]).all() and int(torch.isinf(want["y"][0]).sum()) == L - t + 1
    y, h = forward(s, cuda)
    same(y, *want["y"], dtype)
    same(h, *want["h"], torch.float32)


@pytest.mark.parametrize("L", LENGTHS)
def test_large_and_infinite_states(cuda, L):
    """Many steps leave less than the smallest float of a state, each of them exp(-2); without
    inputs the state alone is left."""
    s = make(L, MEDIUM, seed=L)
    s["x"].zero_()
    for c, v in enumerate((1e38, float("inf"), -float("inf"), float("nan"), -1e30, 3e38)):
        s["h_in"][:, c] = v
    want = G.gated(**s)
    y, h = forward(s, cuda)
    # (what is left near the end of the type's range may be flushed to zero)
    same(y, want["y"][0], want["y"][1] + 2.0 ** -110, torch.float32)
    same(h, want["h"][0], want["h"][1] + 2.0 ** -110, torch.float32)


def test_a_prompt_is_its_tokens(cuda):
    from mamba_int import ops
    s = make(300, FAST, seed=7)
    s["x"][0, 3, 1], s["x"][1, 290, 5], s["x"][1, 20, 6] = float("inf"), -float("inf"), float("nan")
    y, h = forward(s, cuda)
    d = {k: v.to(cuda) for k, v in s.items()}
    state = d["h_in"].clone()
    got = torch.cat([ops.gated_scan(d["x"][:, t:t + 1], d["r"][:, t:t + 1], d["i"][:, t:t + 1], d["decay"], h_in=state, h_out=state)
                     for t in range(300)], 1)
    for a, b in ((y, got), (h, state)):
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        assert torch.equal(a.isinf(), b.isinf()) and torch.equal(a[a.isinf()], b[b.isinf()])


@pytest.mark.parametrize("L", LENGTHS)
@pytest.mark.parametrize("what", ["dy", "x", "h_in"])
def test_gradients(cuda, L, what):
    """An infinite gradient is infinite in all steps before it, an infinite state in all behind it."""
    from mamba_int import ops
    s = make(L, FAST, seed=L + 1)
    dy = 0.1 + torch.rand(2, L, 9, generator=torch.Generator().manual_seed(L))
    if what == "dy":
        dy[1, L - 1 - L // 5, 4] = float("inf")
        dy[0, 0, 2] = -float("inf")
    elif what == "x":
        s["x"][1, L // 5, 4] = float("inf")
    else:
        s["h_in"][1, 4] = float("inf")
    want = G.gated(**s, dy=dy)
    leaf = {k: v.to(cuda).requires_grad_() for k, v in s.items()}
    y = ops.gated_scan(**leaf)
    grads = torch.autograd.grad(y, list(leaf.values()), dy.to(cuda))
    same(y.detach(), *want["y"], torch.float32)
    for n, g in zip(leaf, grads):
        same(g, *want["d_" + n], torch.float32)
    if what == "dy":
        assert torch.isinf(grads[0][1, :L - L // 5, 4]).all() and torch.isinf(grads[4][1, 4])


@pytest.mark.parametrize("L", LENGTHS)
@pytest.mark.parametrize("rate", [8.0, 0.0, 1e30])
def test_decays_at_the_ends_of_their_range(cuda, L, rate):
    """A decay of -inf (and what softplus makes 0) keeps the state, one of +inf leaves nothing of
    it but where the gate is closed or the rate is 0, and both have gradients."""
    from mamba_int import ops
    inf = float("inf")
    decay = torch.tensor([-inf, -3.4e38, -1e30, -2e4, inf, 3.4e38, 2.5e38, 1e30, float("nan")])
    s = make(L, 0.0, seed=L)
    s["decay"] = decay
    s["r"][1] = -inf            # closed
    dy = torch.rand(2, L, 9, generator=torch.Generator().manual_seed(L)).to(cuda)
    y, h = forward(s, cuda, rate=rate)
    leaf = {k: v.to(cuda).requires_grad_() for k, v in s.items()}
    grads = dict(zip(leaf, torch.autograd.grad(ops.gated_scan(**leaf, rate=rate), list(leaf.values()), dy)))
    assert torch.isnan(y[..., 8]).all() and not torch.isnan(y[..., :8]).any() and not torch.isnan(h[:, :8]).any()
    x, q = s["x"].double(), torch.sigmoid(s["i"].double())
    kept = torch.zeros(2, 8, dtype=torch.bool)
    kept[:, :4] = True                     # a = 1, so nothing is added
    kept[1] = True
    kept |= rate == 0.0
    first = s["h_in"][:, :8].double()
    want = torch.where(kept.unsqueeze(1), first.unsqueeze(1), (q * x)[..., :8])
    # two roundings of q, its product and h's: 8 U with the hardware's reciprocal and exponential
    assert ((y[..., :8].cpu() - want).abs() <= 2.0 ** -21 * want.abs()).all()
    assert torch.equal(h.cpu()[:, :8], y.cpu()[:, -1, :8])
    g = dy.double().cpu()[..., :8]
    sums = g.flip(1).cumsum(1).flip(1)
    expect = {"x": torch.where(kept.unsqueeze(1), 0.0, g * q[..., :8]), "r": torch.zeros_like(g),
              "i": torch.where(kept.unsqueeze(1), 0.0, g * (q * x * (1 - q))[..., :8]), "decay": torch.zeros(8, dtype=torch.float64),
              "h_in": torch.where(kept, sums[:, 0], 0.0)}
    for n, w in expect.items():
        got = grads[n].double().cpu()[..., :8]
        # sums of up to L gradients; 1 - q is off by two roundings of 1, against 0.26 at least
        assert ((got - w).abs() <= (L + 64) * 2.0 ** -24 * w.abs()).all(), n
