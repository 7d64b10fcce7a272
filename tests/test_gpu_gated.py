"""Gated recurrence against its formulas in 64 bits: prompts, tokens, lengths, states, gates,
strides, and its gradients, also against differences."""
import pytest
import torch

import float_ref as R
import gated_ref as G

pytestmark = pytest.mark.gpu
NAMES = ("x", "r", "i", "decay", "z", "h_in")


def make(B, L, D, dtype, seed, state=True, gate=True, lens=False, slow=False):
    g = torch.Generator().manual_seed(seed)
    s = {"x": torch.randn(B, L, D, generator=g).to(dtype), "r": (1.5 * torch.randn(B, L, D, generator=g)).to(dtype),
         "i": (1.5 * torch.randn(B, L, D, generator=g)).to(dtype), "z": None, "h_in": None, "lens": None}
    # the largest log decay of a step from 0.001 (slow) or 0.02 to 4 (fast channels too)
    top = torch.exp(torch.empty(D).uniform_(-6.9 if slow else -4.0, -2.0 if slow else 1.4, generator=g))
    s["decay"] = torch.log(torch.expm1(top / 8.0))
    if gate:
        s["z"] = torch.randn(B, L, D, generator=g).to(dtype)
    if state:
        s["h_in"] = torch.randn(B, D, generator=g)
    if lens:
        s["lens"] = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32)
        s["lens"][0] = L
        s["lens"][-1] = 0
    s["dy"] = torch.randn(B, L, D, generator=g).to(dtype)
    return s


def put(s, cuda):
    return {k: v.to(cuda) if v is not None else None for k, v in s.items()}


def forward(s, cuda, **more):
    from mamba_int import ops
    d = put(s, cuda)
    d.pop("dy")
    d.update(more)
    d.setdefault("h_out", torch.full((s["x"].shape[0], s["x"].shape[2]), 7.0, device=cuda))
    return ops.gated_scan(**d), d["h_out"]


def backward(s, cuda):
    from mamba_int import ops
    d = put(s, cuda)
    names = [n for n in NAMES if d[n] is not None]
    leaf = {n: d[n].requires_grad_() for n in names}
    y = ops.gated_scan(d["x"], d["r"], d["i"], d["decay"], z=d["z"], h_in=d["h_in"], lens=d["lens"])
    return y.detach(), dict(zip(names, torch.autograd.grad(y, [leaf[n] for n in names], d["dy"])))


def check(s, cuda, train=True):
    want = G.gated(s["x"], s["r"], s["i"], s["decay"], s["z"], h_in=s["h_in"], lens=s["lens"], dy=s["dy"] if train else None)
    y, h = forward(s, cuda)
    R.close(y, *want["y"], s["x"].dtype)
    R.close(h, *want["h"], torch.float32)
    if not train:
        return
    y2, grads = backward(s, cuda)
    assert torch.equal(y, y2)
    for n, v in grads.items():
        R.close(v, *want["d_" + n], s[n].dtype)


SHAPES = [(1, 1, 1), (3, 1, 64), (2, 1, 4100), (70, 1, 33), (2, 2, 65), (1, 7, 130), (2, 15, 64), (2, 16, 128), (3, 17, 127), (1, 31, 256),
          (2, 33, 129), (1, 64, 70), (2, 127, 66), (1, 128, 64), (1, 129, 192), (2, 255, 40), (1, 256, 8), (2, 257, 9), (1, 700, 131),
          (1, 1500, 3)]


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("B,L,D", SHAPES)
def test_gated(cuda, B, L, D, dtype):
    check(make(B, L, D, dtype, B + L + D), cuda)


@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("state", [True, False])
def test_without_options(cuda, gate, state):
    check(make(2, 300, 70, torch.float32, 3, state=state, gate=gate), cuda)


@pytest.mark.parametrize("B,L,D", [(1, 5000, 64), (2, 3000, 33), (1, 20000, 2)])
def test_long_and_slow(cuda, B, L, D):
    """Decays near one: what a step adds is near sqrt(2 n), and the state remembers thousands of steps."""
    check(make(B, L, D, torch.float32, L, slow=True), cuda)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("B,L,D", [(4, 45, 100), (5, 300, 65), (3, 1100, 34), (6, 16, 128), (3, 2, 5)])
def test_lengths(cuda, B, L, D, dtype):
    """Unequal lengths, an empty sequence among them, and inputs past the ends that are no numbers."""
    s = make(B, L, D, dtype, L, lens=True)
    want = {k: v.clone() if v is not None else None for k, v in s.items()}
    for b in range(B):
        for k in ("x", "r", "i", "z", "dy"):
            s[k][b, int(s["lens"][b]):] = float("nan") if b % 2 else float("inf")
    ref = G.gated(want["x"], want["r"], want["i"], want["decay"], want["z"], h_in=want["h_in"], lens=want["lens"], dy=want["dy"])
    y, h = forward(s, cuda)
    R.close(y, *ref["y"], dtype)
    R.close(h, *ref["h"], torch.float32)
    _, grads = backward(s, cuda)
    for n, v in grads.items():
        R.close(v, *ref["d_" + n], s[n].dtype)
        if n in ("x", "r", "i", "z"):
            for b in range(B):
                assert (v[b, int(s["lens"][b]):] == 0).all()


def test_lengths_out_of_range(cuda):
    s = make(2, 20, 64, torch.float32, 1)
    s["lens"] = torch.tensor([-7, 99], dtype=torch.int32)
    check(s, cuda)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("L", [1, 23, 400])
def test_strides(cuda, dtype, L):
    """Gates from halves of one projection's rows at odd offsets, an output view, the state in place."""
    from mamba_int import ops
    B, D = 3, 71
    s = make(B, L, D, dtype, 9)
    ri = torch.zeros(B, L + 3, 2 * D + 1, dtype=dtype, device=cuda)
    r, i = ri[:, 2:2 + L, D + 1:], ri[:, 2:2 + L, :D]
    d = put(s, cuda)
    r.copy_(d["r"]), i.copy_(d["i"])
    want, hw = forward(s, cuda)
    out = torch.zeros(B, L, D + 3, dtype=dtype, device=cuda)
    h = d["h_in"].clone()
    got = ops.gated_scan(d["x"], r, i, d["decay"], z=d["z"], h_in=h, h_out=h, out=out[..., 2:D + 2])
    assert torch.equal(got, want) and torch.equal(h, hw)
    assert (out[..., :2] == 0).all() and (out[..., D + 2:] == 0).all()
    # gradients of views, and of an expanded input: the sum over what it was broadcast to
    base = ri.clone().requires_grad_()
    x1 = d["x"][:1].clone().requires_grad_()
    y = ops.gated_scan(x1.expand(B, L, D), base[:, 2:2 + L, D + 1:], base[:, 2:2 + L, :D], d["decay"], z=d["z"], h_in=d["h_in"])
    gb, gx = torch.autograd.grad(y, (base, x1), d["dy"].transpose(0, 1).contiguous().transpose(0, 1))
    _, grads = backward(dict(s, x=s["x"][:1].expand(B, L, D).contiguous()), cuda)
    assert torch.equal(gb[:, 2:2 + L, D + 1:], grads["r"]) and torch.equal(gb[:, 2:2 + L, :D], grads["i"])
    assert (gb[:, :2] == 0).all() and torch.equal(gx, grads["x"].sum(0, keepdim=True))
    # a gradient of y with one value for all channels, and one of other strides
    x = d["x"].clone().requires_grad_()
    y = ops.gated_scan(x, d["r"], d["i"], d["decay"])
    one = torch.autograd.grad(y, x, d["dy"][..., :1].expand(B, L, D), retain_graph=True)[0]
    assert torch.equal(one, torch.autograd.grad(y, x, d["dy"][..., :1].expand(B, L, D).contiguous(), retain_graph=True)[0])
    turned = d["dy"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(torch.autograd.grad(y, x, turned, retain_graph=True)[0], torch.autograd.grad(y, x, d["dy"])[0])


def test_parts_and_steps(cuda):
    """A prompt in parts and then token by token, the state in place, is the prompt at once."""
    from mamba_int import ops
    s = make(2, 290, 130, torch.float32, 1, state=False)
    want = G.gated(s["x"], s["r"], s["i"], s["decay"], s["z"])
    d = put(s, cuda)
    h = torch.zeros(2, 130, device=cuda)
    got = []
    for lo, hi in [(0, 140), (140, 141), (141, 285)] + [(t, t + 1) for t in range(285, 290)]:
        p = {k: d[k][:, lo:hi] for k in ("x", "r", "i", "z")}
        got.append(ops.gated_scan(p["x"], p["r"], p["i"], d["decay"], z=p["z"], h_in=h, h_out=h))
    R.close(torch.cat(got, 1), *want["y"], torch.float32)
    R.close(h, *want["h"], torch.float32)


def test_closed_and_open_gates(cuda):
    """Gates far out on both sides, and decays from none to all: no 0 / 0 in values or gradients."""
    v = torch.tensor([-1e30, -200.0, -104.0, -88.0, -30.0, -10.0, 0.0, 10.0, 30.0, 88.0, 200.0, 1e30])
    dec = torch.tensor([-120.0, -100.0, -80.0, -30.0, -9.0, -3.0, 0.0, 3.0, 20.0, 25.0])
    r, i, k = torch.meshgrid(v, v, dec, indexing="ij")
    D = r.numel()
    g = torch.Generator().manual_seed(0)
    s = {"x": torch.randn(1, 5, D, generator=g).clamp(-4, 4), "r": r.reshape(1, 1, D).expand(1, 5, D).contiguous(),
         "i": i.reshape(1, 1, D).expand(1, 5, D).contiguous(), "decay": k.reshape(D).contiguous(), "z": None,
         "h_in": torch.randn(1, D, generator=g), "lens": None,
         "dy": torch.randn(1, 5, D, generator=g).clamp(-4, 4)}
    y, h = forward(s, cuda)
    _, grads = backward(s, cuda)
    assert torch.isfinite(y).all() and torch.isfinite(h).all()
    want = G.gated(s["x"], s["r"], s["i"], s["decay"], h_in=s["h_in"], dy=s["dy"])
    # Sigmoids below 2^-126 may be flushed, with log decays n up to 200 * 2^-126: the step's
    # sqrt(2 n) is 2.2e-18 then, x and dy are 4 at most, g 20, p = g q x n / m 9e-17, a sum of
    # five of them 4.4e-16.
    R.close(y, want["y"][0], want["y"][1] + 2.0 ** -50, torch.float32)
    for n, v in grads.items():
        assert torch.isfinite(v).all(), n
        R.close(v, want["d_" + n][0], want["d_" + n][1] + 2.0 ** -50, torch.float32)


def test_nan_stays_in_its_channel_and_future(cuda):
    s = make(2, 300, 70, torch.float32, 3)
    clean, hc = forward(s, cuda)
    _, gc = backward(s, cuda)
    s["x"][1, 122, 30] = float("nan")
    got, h = forward(s, cuda)
    bad = torch.zeros(2, 300, 70, dtype=torch.bool, device=cuda)
    bad[1, 122:, 30] = True
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[~bad], clean[~bad])
    assert torch.isnan(h[1, 30]) and int(torch.isnan(h).sum()) == 1
    _, grads = backward(s, cuda)
    other = torch.ones(2, 300, 70, dtype=torch.bool, device=cuda)
    other[1, :, 30] = False
    for n in ("x", "r", "i", "z"):
        assert torch.equal(grads[n][other], gc[n][other])


@pytest.mark.parametrize("which", NAMES)
def test_one_gradient_alone(cuda, which):
    """Inputs without a gradient are not differentiated, the others' stay the same."""
    from mamba_int import ops
    s = make(2, 150, 40, torch.float32, 5)
    _, all_ = backward(s, cuda)
    d = put(s, cuda)
    d[which].requires_grad_()
    y = ops.gated_scan(d["x"], d["r"], d["i"], d["decay"], z=d["z"], h_in=d["h_in"])
    assert torch.equal(torch.autograd.grad(y, d[which], d["dy"])[0], all_[which])


@pytest.mark.parametrize("which", NAMES)
def test_gradients_against_differences(cuda, which):
    """Along a random direction, by central differences of two steps: their difference bounds
    what the coarser one leaves out by 4/3 of it; the values' own rounding, 2^-24 of what is
    summed for each of at most 40 roundings a value, is divided by the step."""
    from mamba_int import ops
    s = make(2, 60, 20, torch.float32, 6)
    d = put(s, cuda)
    w = d["dy"]
    v = torch.randn(d[which].shape, generator=torch.Generator().manual_seed(1)).to(cuda)

    def value(step):
        e = dict(d, **{which: d[which] + step * v})
        y = ops.gated_scan(e["x"], e["r"], e["i"], e["decay"], z=e["z"], h_in=e["h_in"])
        return (y.double() * w).sum().item(), (y.double() * w).abs().sum().item()

    def difference(step):
        (up, m), (down, _) = value(step), value(-step)
        return (up - down) / (2 * step), 40 * 2.0 ** -24 * m / step

    coarse, fine = difference(2.0 ** -6), difference(2.0 ** -7)
    _, grads = backward(s, cuda)
    got = (grads[which].double() * v).sum().item()
    assert abs(got - fine[0]) <= 4 * abs(coarse[0] - fine[0]) / 3 + 3 * (coarse[1] + fine[1])


def test_repeats_are_bit_equal(cuda):
    for shape in ((2, 300, 100), (1, 4000, 32), (7, 1, 100)):
        s = make(*shape, torch.bfloat16, 5)
        a, ga = backward(s, cuda)
        b, gb = backward(s, cuda)
        assert torch.equal(a, b) and all(torch.equal(ga[n], gb[n]) for n in ga)


def test_graph_replays(cuda):
    """The forward pass, and a whole training step, captured: each replay equals the eager calls."""
    from mamba_int import ops
    for L in (1, 700):
        s = make(1, L, 96, torch.float32, 2)
        d = put(s, cuda)
        names = [n for n in NAMES if d[n] is not None]

        def step():
            leaf = {n: d[n].detach().requires_grad_() for n in names}
            y = ops.gated_scan(leaf["x"], leaf["r"], leaf["i"], leaf["decay"], z=leaf["z"], h_in=leaf["h_in"])
            return (y.detach(), *torch.autograd.grad(y, list(leaf.values()), d["dy"]))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for seed in range(3):
            new = put(make(1, L, 96, torch.float32, 30 + seed), cuda)
            for n in names + ["dy"]:
                d[n].copy_(new[n])
            want = step()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_capture_beside_a_live_graph_of_the_leaves_is_refused(cuda):
    """Its backward pass would make the other graph's stream wait for the capture."""
    from mamba_int import ops
    d = put(make(1, 30, 32, torch.float32, 2, state=False, gate=False), cuda)
    d["decay"].requires_grad_()
    y = ops.gated_scan(d["x"], d["r"], d["i"], d["decay"])
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="decay is a leaf of another graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.gated_scan(d["x"], d["r"], d["i"], d["decay"])
    want = torch.autograd.grad(y, d["decay"], d["dy"])[0]
    del y
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = ops.gated_scan(d["x"], d["r"], d["i"], d["decay"])
        got, = torch.autograd.grad(z, d["decay"], d["dy"])
    for _ in range(2):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_empty(cuda):
    from mamba_int import ops
    d = put(make(2, 1, 16, torch.float32, 2), cuda)
    none = {k: d[k][:, :0].detach().requires_grad_() for k in ("x", "r", "i", "z")}
    h = torch.zeros_like(d["h_in"])
    with torch.no_grad():
        y = ops.gated_scan(none["x"], none["r"], none["i"], d["decay"], z=none["z"], h_in=d["h_in"], h_out=h)
    assert y.shape == (2, 0, 16) and torch.equal(h, d["h_in"])
    d["decay"].requires_grad_(), d["h_in"].requires_grad_()
    y = ops.gated_scan(none["x"], none["r"], none["i"], d["decay"], z=none["z"], h_in=d["h_in"])
    gd, gh, gx = torch.autograd.grad(y.sum(), (d["decay"], d["h_in"], none["x"]))
    assert (gd == 0).all() and (gh == 0).all() and gx.shape == (2, 0, 16)
    y = ops.gated_scan(d["x"][:0], d["r"][:0], d["i"][:0], d["decay"])
    assert y.shape == (0, 1, 16) and (torch.autograd.grad(y.sum(), d["decay"])[0] == 0).all()


def test_refusals(cuda):
    from mamba_int import ops
    d = put(make(2, 6, 16, torch.float32, 2), cuda)
    x, r, i, k = d["x"], d["r"], d["i"], d["decay"]
    for bad, err in ((dict(x=x[0]), ValueError), (dict(r=r.half()), TypeError), (dict(i=i[:, :-1]), ValueError), (dict(decay=k[:-1]), ValueError),
                     (dict(decay=k.double()), TypeError), (dict(h_in=torch.zeros(2, 15, device=cuda)), ValueError),
                     (dict(z=i.transpose(1, 2)), ValueError), (dict(lens=torch.zeros(2, device=cuda)), TypeError), (dict(rate=-1.0), RuntimeError),
                     (dict(rate=float("nan")), RuntimeError), (dict(x=x.cpu()), ValueError), (dict(decay=None), TypeError)):
        with pytest.raises(err):
            ops.gated_scan(**dict(dict(x=x, r=r, i=i, decay=k), **bad))
    k.requires_grad_()
    with pytest.raises(ValueError, match="out and h_out"):
        ops.gated_scan(x, r, i, k, h_out=torch.zeros(2, 16, device=cuda))
    y = ops.gated_scan(x, r, i, k)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(torch.autograd.grad(y.sum(), k, create_graph=True)[0].sum(), k)
    y = ops.gated_scan(x, r, i, k)
    x.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.no_grad():
        assert not ops.gated_scan(x, r, i, k).requires_grad
