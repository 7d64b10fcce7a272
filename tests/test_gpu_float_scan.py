"""Selective scan against the recurrence in 64 bits: prompts, tokens, lengths, states, groups, strides."""
import math

import pytest
import torch

import float_ref as R

pytestmark = pytest.mark.gpu


def make(B, L, D, N, G, dtype, seed, state=True, lens=False, gate=True):
    g = torch.Generator().manual_seed(seed)
    s = {"u": torch.randn(B, L, D, generator=g).to(dtype), "dt": (0.7 * torch.randn(B, L, D, generator=g)).to(dtype),
         "b": torch.randn(B, L, G, N, generator=g).to(dtype), "c": torch.randn(B, L, G, N, generator=g).to(dtype),
         "a": -torch.arange(1, N + 1).float() * torch.exp(0.2 * torch.randn(D, N, generator=g)),
         "d_skip": torch.randn(D, generator=g)}
    step = torch.exp(torch.rand(D, generator=g) * math.log(100) + math.log(1e-3))
    s["dt_bias"] = torch.log(torch.expm1(step))
    s["z"] = torch.randn(B, L, D, generator=g).to(dtype) if gate else None
    s["h_in"] = torch.randn(B, D, N, generator=g) if state else None
    ln = None
    if lens:
        ln = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32)
        ln[0] = L
        ln[-1] = 0
    s["lens"] = ln
    return s


def run(s, cuda, **more):
    from mamba_int import ops
    d = {k: v.to(cuda) if v is not None else None for k, v in s.items()}
    d.update(more)
    h = torch.full((s["u"].shape[0], *s["a"].shape), 7.0, device=cuda)
    d.setdefault("h_out", h)
    return ops.selective_scan(**d), d["h_out"]


def check(s, got, h, dtype):
    y, ey, hw, eh = R.scan(s["u"], s["dt"], s["a"], s["b"], s["c"], s["d_skip"], s["z"], s["dt_bias"], True, s["h_in"],
                           s["lens"])
    R.close(h, hw, eh, torch.float32)
    R.close(got, y, ey, dtype)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("B,L,D,N,G", [
    (1, 1, 1, 1, 1), (2, 1, 64, 16, 1), (3, 1, 100, 16, 1), (5, 1, 70, 64, 2), (2, 1, 33, 5, 1), (2, 1, 8, 256, 1),
    (1, 2, 64, 16, 1), (2, 15, 64, 16, 1), (2, 16, 130, 16, 1), (2, 17, 63, 16, 1), (1, 100, 200, 16, 1),
    (2, 64, 96, 8, 1), (2, 37, 128, 64, 2), (1, 50, 66, 3, 1), (1, 21, 65, 7, 1), (1, 33, 40, 130, 1), (1, 20, 12, 256, 1),
    (2, 33, 96, 12, 3), (1, 18, 192, 32, 4), (2, 70, 1, 16, 1)])
def test_scan(cuda, B, L, D, N, G, dtype):
    s = make(B, L, D, N, G, dtype, B * 31 + L + D + N)
    got, h = run(s, cuda)
    check(s, got, h, dtype)


@pytest.mark.parametrize("B,L,D,N", [(4, 45, 100, 16), (3, 200, 64, 16), (5, 19, 70, 40), (6, 600, 32, 8)])
@pytest.mark.parametrize("gate", [True, False])
def test_lengths(cuda, B, L, D, N, gate):
    """Unequal lengths, an empty sequence among them, and inputs past the ends that are no numbers."""
    s = make(B, L, D, N, 1, torch.float32, L, lens=True, gate=gate)
    want = {k: v.clone() if v is not None else None for k, v in s.items()}
    for b in range(B):
        for k in ("u", "dt", "b", "c", "z"):
            if s[k] is not None:
                s[k][b, int(s["lens"][b]):] = float("nan") if b % 2 else float("inf")
    got, h = run(s, cuda)
    check(want, got, h, torch.float32)
    for b in range(B):
        assert (got[b, int(s["lens"][b]):] == 0).all()


@pytest.mark.parametrize("B,L,D,N", [(1, 3000, 64, 16), (1, 2049, 48, 64), (2, 1500, 20, 16), (1, 5000, 8, 8)])
def test_long(cuda, B, L, D, N):
    """Few channels and many steps (the sequence is split there)."""
    s = make(B, L, D, N, 1, torch.float32, L)
    got, h = run(s, cuda)
    check(s, got, h, torch.float32)
    s["lens"] = torch.full((B,), L // 3, dtype=torch.int32)
    got, h = run(s, cuda)
    check(s, got, h, torch.float32)


def test_long_state_in_place(cuda):
    """The state in place where the sequence is split: its parts read the first state, the
    last one writes the new one."""
    s = make(1, 2000, 200, 16, 1, torch.float32, 8)
    want, h = run(s, cuda)
    check(s, want, h, torch.float32)
    for _ in range(5):
        state = s["h_in"].to(cuda)
        got, _ = run(s, cuda, h_in=state, h_out=state)
        assert torch.equal(got, want) and torch.equal(state, h)


def test_parts_and_steps(cuda):
    """A prompt in parts and then token by token, the state in place, is the prompt at once."""
    from mamba_int import ops
    s = make(2, 90, 130, 16, 1, torch.float32, 1, state=False)
    y, ey, hw, eh = R.scan(s["u"], s["dt"], s["a"], s["b"], s["c"], s["d_skip"], s["z"], s["dt_bias"])
    d = {k: v.to(cuda) if v is not None else None for k, v in s.items()}
    h = torch.zeros(2, 130, 16, device=cuda)
    got = []
    for lo, hi in [(0, 40), (40, 41), (41, 85)] + [(t, t + 1) for t in range(85, 90)]:
        part = {k: d[k][:, lo:hi] for k in ("u", "dt", "b", "c", "z")}
        got.append(ops.selective_scan(part["u"], part["dt"], d["a"], part["b"], part["c"], d_skip=d["d_skip"], z=part["z"],
                                      dt_bias=d["dt_bias"], h_in=h, h_out=h))
    R.close(torch.cat(got, 1), y, ey, torch.float32)
    R.close(h, hw, eh, torch.float32)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("L", [1, 23])
def test_strides(cuda, dtype, L):
    """Slices of x_proj's and in_proj's rows, odd offsets, an output view, [B, L, N] rows."""
    from mamba_int import ops
    B, D, N = 3, 70, 16
    s = make(B, L, D, N, 1, dtype, 9)
    xz = torch.empty(B, L + 3, 2 * D + 1, dtype=dtype, device=cuda)
    xp = torch.empty(B, L, 5 + 2 * N, dtype=dtype, device=cuda)
    z, u, b, c = xz[:, 2:2 + L, D + 1:], xz[:, 2:2 + L, :D], xp[..., 5:5 + N], xp[..., 5 + N:]
    z.copy_(s["z"]); u.copy_(s["u"]); b.copy_(s["b"][:, :, 0]); c.copy_(s["c"][:, :, 0])
    out = torch.zeros(B, L, D + 3, dtype=dtype, device=cuda)
    h = s["h_in"].to(cuda)
    got = ops.selective_scan(u, s["dt"].to(cuda), s["a"].to(cuda), b, c, d_skip=s["d_skip"].to(cuda), z=z,
                             dt_bias=s["dt_bias"].to(cuda), h_in=h, h_out=h, out=out[..., 2:D + 2])
    check(s, got, h, dtype)
    assert (out[..., :2] == 0).all() and (out[..., D + 2:] == 0).all()


def test_without_options(cuda):
    from mamba_int import ops
    s = make(2, 40, 64, 16, 1, torch.float32, 6, state=False, gate=False)
    s["dt"] = s["dt"].abs() * 0.1
    y, ey, _, _ = R.scan(s["u"], s["dt"], s["a"], s["b"], s["c"], sp=False)
    got = ops.selective_scan(*(s[k].to(cuda) for k in ("u", "dt", "a", "b", "c")), dt_softplus=False)
    R.close(got, y, ey, torch.float32)


def test_softplus_keeps_relative_precision(cuda):
    """Small steps are exp(v): their relative precision is what the state keeps."""
    from mamba_int import ops
    v = torch.cat([torch.linspace(-80, 30, 4001), torch.tensor([0.0, -0.0, 1e-30, 88.0, 500.0, -1e30])])
    D = v.numel()
    one = torch.ones(1, 1, D, device=cuda)
    bc = torch.ones(1, 1, 1, device=cuda)
    for L in (1, 3):
        y = ops.selective_scan(one.expand(1, L, D), v.view(1, 1, D).expand(1, L, D).to(cuda), torch.full((D, 1), -1e38, device=cuda),
                               bc.expand(1, L, 1), bc.expand(1, L, 1))
        want = R.softplus(v.double()).expand(1, L, D)
        R.close(y, want, want * R.U * (12 + 2 * v.double().abs().clamp(max=100)), torch.float32)


def test_nan_stays_in_its_channel_and_future(cuda):
    s = make(2, 40, 70, 16, 1, torch.float32, 3)
    clean, _ = run(s, cuda)
    s["u"][1, 22, 30] = float("nan")
    got, h = run(s, cuda)
    bad = torch.zeros(2, 40, 70, dtype=torch.bool, device=cuda)
    bad[1, 22:, 30] = True
    assert torch.equal(torch.isnan(got), bad)
    assert torch.equal(got[~bad], clean[~bad])
    assert torch.isnan(h[1, 30]).all() and int(torch.isnan(h).sum()) == 16


def test_repeats_are_bit_equal(cuda):
    for shape in ((2, 300, 100, 16, 1), (1, 4000, 32, 16, 1), (7, 1, 100, 16, 1)):
        s = make(*shape, torch.bfloat16, 5)
        a, ha = run(s, cuda)
        b, hb = run(s, cuda)
        assert torch.equal(a, b) and torch.equal(ha, hb)


def test_graph_replays(cuda):
    """Captured in a graph (the prompt form and the token form), each replay equals the eager call."""
    from mamba_int import ops
    for L in (1, 700):
        s = {k: v.to(cuda) if v is not None else None for k, v in make(1, L, 96, 16, 1, torch.float32, 2).items()}
        want = ops.selective_scan(**s)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            ops.selective_scan(**s)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.selective_scan(**s)
        for _ in range(3):
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)


def test_empty(cuda):
    from mamba_int import ops
    s = {k: v.to(cuda) if v is not None else None for k, v in make(2, 1, 16, 16, 1, torch.float32, 2).items()}
    none = {k: s[k][:, :0] for k in ("u", "dt", "b", "c", "z")}
    h = torch.zeros_like(s["h_in"])
    y = ops.selective_scan(none["u"], none["dt"], s["a"], none["b"], none["c"], z=none["z"], h_in=s["h_in"], h_out=h)
    assert y.shape == (2, 0, 16) and torch.equal(h, s["h_in"])
    none = {k: s[k][:0] for k in ("u", "dt", "b", "c")}
    assert ops.selective_scan(none["u"], none["dt"], s["a"], none["b"], none["c"]).shape == (0, 1, 16)
