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
