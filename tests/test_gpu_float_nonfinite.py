"""Infinite inputs, steps and states of the selective scan, as the recurrence in 64 bits has them."""
import pytest
import torch

import float_ref as R

pytestmark = pytest.mark.gpu


def same(got, want, err, dtype):
    """NaN and infinities where want has them, the rest within err."""
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    odd = torch.isinf(want)
    assert torch.equal(torch.isinf(got), odd) and torch.equal(got[odd], want[odd])
    on = torch.isfinite(want)
    R.close(got[on].to(dtype), want[on], err[on], dtype)


def positive(B, L, D, N, dtype, seed):
    """Decays that leave a state above 2^-40 over 20 steps; B, C, u and D positive."""
    g = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return (0.1 + 0.9 * torch.rand(*shape, generator=g)).to(dtype)
    return {"u": rand(B, L, D), "dt": rand(B, L, D) - 1.0, "b": rand(B, L, 1, N), "c": rand(B, L, 1, N),
            "a": -(0.1 + 0.9 * torch.rand(D, N, generator=g)), "d_skip": torch.rand(D, generator=g)}


def run(s, cuda, **more):
    from mamba_int import ops
    h = torch.zeros(s["u"].shape[0], *s["a"].shape, device=cuda)
    y = ops.selective_scan(**{k: v.to(cuda) for k, v in s.items()}, h_out=h, **more)
    return y, h


# L: steps one after another, tiles of a whole sequence (many blocks), tiles of its parts
@pytest.mark.parametrize("B,L,D", [(2, 1, 9), (2, 5, 9), (2, 30, 9), (300, 20, 5), (1, 200, 9)])
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 7, 8, 12, 13, 16, 20, 40, 100, 129, 200])
@pytest.mark.parametrize("what", ["u", "dt"])
def test_infinite_input_or_step(cuda, B, L, D, N, what):
    """Infinite from that step on, whatever N: no place of a block beside the states makes a NaN."""
    s = positive(B, L, D, N, torch.float32, 3 * N + L)
    t = L // 3
    s[what][B // 2, t, 4] = float("inf")
    got, h = run(s, cuda)
    y, ey, hw, eh = R.scan(s["u"], s["dt"], s["a"], s["b"], s["c"], s["d_skip"])
    assert torch.isinf(y[B // 2, t:, 4]).all() and torch.isinf(y).sum() == L - t
    same(got, y, ey, torch.float32)
    same(h, hw, eh, torch.float32)


@pytest.mark.parametrize("N", [3, 12, 16, 20])
def test_infinite_input_of_16_bits_with_a_gate(cuda, N):
    for dtype in (torch.bfloat16, torch.float16):
        s = positive(3, 40, 70, N, dtype, N)
        s["z"] = s["u"].clone()
        s["u"][1, 17, 66] = -float("inf")
        got, h = run(s, cuda)
        y, ey, hw, eh = R.scan(s["u"], s["dt"], s["a"], s["b"], s["c"], s["d_skip"], s["z"])
        assert (y[1, 17:, 66] == -float("inf")).all()
        same(got, y, ey, dtype)
        same(h, hw, eh, torch.float32)


@pytest.mark.parametrize("N", [1, 8, 16, 20])
@pytest.mark.parametrize("L", [300, 2000])
def test_large_and_infinite_states_in_a_split_sequence(cuda, L, N):
    """States that decay by 2^-2.9 a step: a part's decay is below the smallest float, that of
    each step is not.  Without inputs the state alone is left."""
    s = positive(1, L, 5, N, torch.float32, L + N)
    s["u"].zero_()
    s["dt"].fill_(2.0)
    s["a"].fill_(-1.0)
    s["h_in"] = torch.full((1, 5, N), 1e38)
    s["h_in"][0, 1] = float("inf")
    s["h_in"][0, 2] = -float("inf")
    s["h_in"][0, 3] = float("nan")
    s["h_in"][0, 4] = -1e30
    got, h = run(s, cuda, dt_softplus=False)
    y, ey, hw, eh = R.scan(s["u"], s["dt"], s["a"], s["b"], s["c"], s["d_skip"], sp=False, h_in=s["h_in"])
    # what is left near the end of the type's range may be flushed to zero
    same(got, y, ey + 2.0 ** -110, torch.float32)
    same(h, hw, eh + 2.0 ** -110, torch.float32)


@pytest.mark.parametrize("B,L,D,N", [(2, 1, 9, 16), (3, 1, 9, 5), (2, 5, 9, 16), (2, 30, 9, 16), (1, 200, 9, 16)])
def test_infinite_input_without_a_skip(cuda, B, L, D, N):
    s = positive(B, L, D, N, torch.float32, L)
    del s["d_skip"]
    t = L // 3
    s["u"][B // 2, t, 4] = float("inf")
    got, h = run(s, cuda)
    y, ey, hw, eh = R.scan(s["u"], s["dt"], s["a"], s["b"], s["c"])
    y[B // 2, t:, 4], ey[B // 2, t, 4] = float("inf"), 0.0     # (the oracle's own skip of 0 times inf)
    same(got, y, ey, torch.float32)
    same(h, hw, eh, torch.float32)


@pytest.mark.parametrize("B,L,D,N", [(2, 1, 9, 16), (2, 1, 9, 5), (2, 5, 9, 16), (2, 30, 9, 16), (1, 200, 9, 16)])
def test_the_fastest_decays(cuda, B, L, D, N):
    """a near the lowest float: a step of 0 keeps the state, any other clears it."""
    s = positive(B, L, D, N, torch.float32, L)
    s["a"].fill_(-3.4e38)
    s["dt"].zero_()
    s["dt"][:, L - 1, 3] = 0.25
    s["h_in"] = torch.ones(B, D, N)
    got, h = run(s, cuda, dt_softplus=False)
    y, ey, hw, eh = R.scan(s["u"], s["dt"], s["a"], s["b"], s["c"], s["d_skip"], sp=False, h_in=s["h_in"])
    assert (hw[:, :3] == 1).all() and (hw[:, 3] < 1).all()
    # (the bound of a decay of 0 is not finite: its exponent's error times 0 is meant)
    same(got, y, torch.where(torch.isfinite(ey), ey, 8 * R.U * y.abs()), torch.float32)
    same(h, hw, torch.where(torch.isfinite(eh), eh, 8 * R.U * hw.abs()), torch.float32)


@pytest.mark.parametrize("B,L,D,N", [(2, 1, 9, 16), (2, 1, 9, 5), (2, 5, 9, 16), (2, 5, 9, 5), (2, 30, 9, 16), (1, 200, 9, 16)])
def test_decays_of_minus_infinity(cuda, B, L, D, N):
    """... are the lowest float's, in a prompt as token by token: a step of 0 keeps the state."""
    s = positive(B, L, D, N, torch.float32, L)
    s["a"].fill_(-float("inf"))
    s["dt"].zero_()
    s["dt"][:, L // 2, 3] = 0.25
    s["h_in"] = torch.ones(B, D, N)
    got, h = run(s, cuda, dt_softplus=False)
    s["a"].fill_(-3.4e38)
    y, ey, hw, eh = R.scan(s["u"], s["dt"], s["a"], s["b"], s["c"], s["d_skip"], sp=False, h_in=s["h_in"])
    same(got, y, torch.where(torch.isfinite(ey), ey, 8 * R.U * y.abs()), torch.float32)
    same(h, hw, torch.where(torch.isfinite(eh), eh, 8 * R.U * hw.abs()), torch.float32)


@pytest.mark.parametrize("B,L,D,N", [(2, 1, 9, 16), (2, 5, 9, 5), (2, 30, 9, 12), (1, 200, 9, 16)])
def test_a_decay_that_is_no_number(cuda, B, L, D, N):
    s = positive(B, L, D, N, torch.float32, L)
    s["a"][4, N - 1] = float("nan")
    s["h_in"] = torch.ones(B, D, N)
    got, h = run(s, cuda)
    bad = torch.zeros(D, dtype=torch.bool, device=cuda)
    bad[4] = True
    assert torch.equal(torch.isnan(got), bad.expand(B, L, D))
    assert torch.isnan(h[:, 4, N - 1]).all() and int(torch.isnan(h).sum()) == B
