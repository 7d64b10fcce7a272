"""Causal convolution against the formula in 64 bits: prompts, tokens, lengths, states, strides."""
import pytest
import torch

import float_ref as R

pytestmark = pytest.mark.gpu


def make(B, L, D, W, dtype, seed, state=True, lens=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, L, D, generator=g).to(dtype)
    w = torch.randn(D, W, generator=g) / W ** 0.5
    bias = 0.3 * torch.randn(D, generator=g)
    st = torch.randn(B, W - 1, D, generator=g).to(dtype) if state else None
    ln = None
    if lens:
        ln = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32)
        ln[0] = L
        ln[-1] = 0
        if B > 2:
            ln[1] = 1
    return x, w, bias, st, ln


def dev(t, cuda):
    return t.to(cuda) if t is not None else None


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("B,L,D,W", [(1, 1, 1, 4), (2, 1, 768, 4), (3, 2, 65, 4), (2, 3, 128, 4), (2, 5, 1003, 3),
                                     (1, 17, 64, 2), (2, 64, 96, 4), (3, 33, 8, 8), (2, 40, 24, 1), (1, 300, 520, 4),
                                     (4, 31, 260, 4), (70, 1, 100, 4)])
@pytest.mark.parametrize("state,lens", [(False, False), (True, False), (True, True)])
def test_conv(cuda, B, L, D, W, dtype, state, lens):
    from mamba_int import ops
    x, w, bias, st, ln = make(B, L, D, W, dtype, B + L + D + W, state, lens)
    y, err, last = R.conv(x, w, bias, True, st, ln)
    out = torch.full((B, W - 1, D), 9.0, dtype=dtype, device=cuda)
    got = ops.causal_conv(x.to(cuda), w.to(cuda), bias=bias.to(cuda), state_in=dev(st, cuda), state_out=out,
                          lens=dev(ln, cuda))
    R.close(got, y, err, dtype)
    assert torch.equal(out.cpu(), last)
    if ln is not None:
        for b in range(B):
            assert (got[b, int(ln[b]):] == 0).all()


def test_no_activation_no_bias_no_state(cuda):
    from mamba_int import ops
    x, w, _, _, _ = make(2, 70, 130, 4, torch.float32, 4, state=False)
    y, err, _ = R.conv(x, w, None, False, None, None)
    R.close(ops.causal_conv(x.to(cuda), w.to(cuda), activation=None), y, err, torch.float32)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("D", [256, 77])
def test_strides_and_offsets(cuda, dtype, D):
    """Half rows of a wider buffer, a slice of the sequence, rows at an odd offset, output into a view."""
    from mamba_int import ops
    x, w, bias, st, _ = make(2, 50, D, 4, dtype, 8)
    wide = torch.empty(2, 60, 2 * D + 1, dtype=dtype, device=cuda)
    for view in (wide[:, :50, :D], wide[:, 10:, D:2 * D], wide[:, 5:55, 1:D + 1]):
        view.copy_(x)
        y, err, last = R.conv(x, w, bias, True, st, None)
        out = torch.zeros(2, 50, 3 * D, dtype=dtype, device=cuda)
        state = st.to(cuda)
        got = ops.causal_conv(view, w.to(cuda), bias=bias.to(cuda), state_in=state, state_out=state,
                              out=out[..., D:2 * D])
        R.close(got, y, err, dtype)
        assert (out[..., :D] == 0).all() and (out[..., 2 * D:] == 0).all()
        assert torch.equal(state.cpu(), last)


@pytest.mark.parametrize("L", [2, 9, 130])
def test_state_in_place_and_steps(cuda, L):
    """A prompt in two parts and then token by token, the state in place, is the prompt at once."""
    from mamba_int import ops
    x, w, bias, _, _ = make(3, L + 6, 200, 4, torch.bfloat16, L, state=False)
    y, err, last = R.conv(x, w, bias, True, None, None)
    xd, wd, bd = x.to(cuda), w.to(cuda), bias.to(cuda)
    st = torch.zeros(3, 3, 200, dtype=torch.bfloat16, device=cuda)
    cut = L // 2
    parts = [xd[:, :cut], xd[:, cut:L]] + [xd[:, t:t + 1] for t in range(L, L + 6)]
    got = torch.cat([ops.causal_conv(p, wd, bias=bd, state_in=st, state_out=st) for p in parts], 1)
    R.close(got, y, err, torch.bfloat16)
    assert torch.equal(st.cpu(), last)


@pytest.mark.parametrize("W", [5, 6, 8])
def test_wide_state_in_place(cuda, W):
    """As many rows of state as a thread walks: only the thread that writes it reads it."""
    from mamba_int import ops
    x, w, bias, st, _ = make(2, 61, 72, W, torch.float32, W)
    y, err, last = R.conv(x, w, bias, True, st, None)
    for _ in range(5):
        state = st.to(cuda)
        R.close(ops.causal_conv(x.to(cuda), w.to(cuda), bias=bias.to(cuda), state_in=state, state_out=state), y, err,
                torch.float32)
        assert torch.equal(state.cpu(), last)


def test_masked_rows_are_not_read_as_values(cuda):
    from mamba_int import ops
    x, w, bias, st, _ = make(3, 20, 64, 4, torch.float32, 2)
    ln = torch.tensor([20, 7, 0], dtype=torch.int32)
    y, err, last = R.conv(x, w, bias, True, st, ln)
    x[1, 7:] = float("nan")
    x[2] = float("inf")
    out = st.to(cuda)
    got = ops.causal_conv(x.to(cuda), w.to(cuda), bias=bias.to(cuda), state_in=out, state_out=out, lens=ln.to(cuda))
    R.close(got, y, err, torch.float32)
    assert torch.equal(out.cpu(), last)
    # lengths outside the rows are clamped to them
    got = ops.causal_conv(x[:1].to(cuda), w.to(cuda), bias=bias.to(cuda), state_in=st[:1].to(cuda),
                          lens=torch.tensor([99], dtype=torch.int32, device=cuda))
    R.close(got, y[:1], err[:1], torch.float32)
    got = ops.causal_conv(x[:1].to(cuda), w.to(cuda), lens=torch.tensor([-3], dtype=torch.int32, device=cuda))
    assert (got == 0).all()


def test_empty(cuda):
    from mamba_int import ops
    w = torch.ones(16, 4, device=cuda)
    st = torch.randn(2, 3, 16, device=cuda)
    out = torch.zeros_like(st)
    y = ops.causal_conv(torch.empty(2, 0, 16, device=cuda), w, state_in=st, state_out=out)
    assert y.shape == (2, 0, 16) and torch.equal(out, st)
    assert ops.causal_conv(torch.empty(0, 5, 16, device=cuda), w).shape == (0, 5, 16)
