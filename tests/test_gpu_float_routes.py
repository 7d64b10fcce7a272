"""Every launch that the float operators choose by size, against the formulas in 64 bits: the
sizes come from the device's CU count, so each rule's branches are really taken.  (Batches
that only have to be large repeat a few sequences, whose results have to repeat too.)"""
import ctypes

import pytest
import torch

import float_ref as R

pytestmark = pytest.mark.gpu


def cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


def repeated(t, B, cuda):
    return None if t is None else t.to(cuda)[torch.arange(B, device=cuda) % t.shape[0]].contiguous()


def check_repeated(got, first):
    """The results of the first sequences, after a check that the others repeat them."""
    assert torch.equal(got, got[:first][torch.arange(got.shape[0], device=got.device) % first])
    return got[:first]


# ------------------------------------------------------------ 4-bit products
def w4_weights(n, k, group, seed, cuda, zeros=True, scale_type=torch.float16):
    from mamba_int import ops
    g = torch.Generator().manual_seed(seed)
    ng = -(-k // group)
    s = {"codes": torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8),
         "scales": ((0.5 + torch.rand(n, ng, generator=g)) / k ** 0.5).to(scale_type),
         "zeros": torch.randint(0, 16, (n, ng), generator=g, dtype=torch.uint8) if zeros else None}
    s["packed"] = ops.pack_w4(s["codes"].to(cuda), s["scales"].to(cuda), group,
                              zeros=s["zeros"].to(cuda) if zeros else None)
    return s


def w4_n(blocks_per_cu, ragged):
    """Weight rows in at least that many row blocks a CU, the last block of them not whole."""
    return 16 * (blocks_per_cu * cus() + 1) + ragged


# rows of x, row blocks a CU, columns, group: one, two and four row blocks a block of up to 16
# rows; two of 32 rows; four of 32 rows by eight and, with few column blocks, by four waves
W4_ROUTES = [(1, 1, 200, 32), (16, 1, 1100, 128), (1, 2, 200, 32), (9, 2, 1100, 64), (3, 4, 129, 64), (16, 4, 1100, 32),
             (1, 4, 2048, 256), (20, 1, 300, 64), (32, 2, 1100, 32), (64, 1, 1100, 128), (40, 2, 300, 32), (64, 4, 768, 64),
             (33, 2, 1100, 64), (64, 2, 2048, 128), (65, 4, 1030, 32)]


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("m,blocks,k,group", W4_ROUTES)
def test_w4(cuda, m, blocks, k, group, dtype):
    from mamba_int import ops
    n = w4_n(blocks, 5) if blocks > 1 else 333
    s = w4_weights(n, k, group, m + k, cuda, zeros=group != 128)
    g = torch.Generator().manual_seed(m)
    x, bias = torch.randn(m, k, generator=g).to(dtype), torch.randn(n, generator=g)
    y, err = R.w4(x, s["codes"], s["scales"], s["zeros"], group, bias)
    p, sc, z = s["packed"]
    R.close(ops.w4_matvec(x.to(cuda), p, sc, n, group, zeros=z, bias=bias.to(cuda)), y, err, dtype)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("m,blocks,k,group", W4_ROUTES)
def test_w4_keeps_the_bits_of_x(cuda, m, blocks, k, group, dtype):
    """Rows with one value, so each result is one product: x (q - zero) is exact in 16 bits' types;
    a float32 x is three parts of 8 bits, whose products with q - zero are exact and whose sum is
    rounded once (the sum of the two lower ones fits 24 bits).  The scale's product is rounded, and
    the result to its type.  A part left out would be 2^-16 of the result."""
    from mamba_int import ops
    n = w4_n(blocks, 5) if blocks > 1 else 333
    s = w4_weights(n, k, group, 3 * m + k, cuda, zeros=group != 128)
    p, sc, z = s["packed"]
    g = torch.Generator().manual_seed(m + 1)
    for turn in range(3):
        cols = torch.randperm(k, generator=g)[torch.arange(m) % k]
        if turn == 0:
            cols[0] = k - 1
        v = ((1 + torch.rand(m, generator=g)) * torch.exp2(torch.randint(-3, 4, (m,), generator=g).float())).to(dtype)
        x = torch.zeros(m, k, dtype=dtype)
        x[torch.arange(m), cols] = v
        w = s["codes"][:, cols].double() - (s["zeros"][:, cols // group].double() if z is not None else 8.0)
        y = (v.double() * w * s["scales"][:, cols // group].double()).t()
        R.close(ops.w4_matvec(x.to(cuda), p, sc, n, group, zeros=z), y, 2.5 * R.U * y.abs(), dtype)


# ------------------------------------------------------------ convolution
@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("steps,W,D", [(8, 4, 1003), (16, 4, 768), (16, 3, 1003), (32, 4, 1003), (32, 2, 768), (16, 7, 520)])
def test_conv_threads_of_many_rows(cuda, steps, W, D, dtype):
    """Threads that walk 8, 16 and 32 rows, with unequal lengths and the state in place."""
    from mamba_int import ops
    V = 16 // torch.empty(0, dtype=dtype).element_size()
    L = 5 * steps + 3
    B = -(-1024 * cus() // (-(-D // V) * -(-L // steps)))
    assert B * -(-D // V) * -(-L // (2 * steps)) < 1024 * cus() or steps == 32
    g = torch.Generator().manual_seed(steps + W + D)
    first = 4
    x = torch.randn(first, L, D, generator=g).to(dtype)
    w, bias = torch.randn(D, W, generator=g) / W ** 0.5, 0.3 * torch.randn(D, generator=g)
    st = torch.randn(first, W - 1, D, generator=g).to(dtype)
    lens = torch.tensor([L, 0, L // 2, 1], dtype=torch.int32)
    y, err, last = R.conv(x, w, bias, True, st, lens)
    state = repeated(st, B, cuda)
    got = ops.causal_conv(repeated(x, B, cuda), w.to(cuda), bias=bias.to(cuda), state_in=state, state_out=state,
                          lens=repeated(lens, B, cuda))
    R.close(check_repeated(got, first), y, err, dtype)
    assert torch.equal(check_repeated(state, first).cpu(), last)


# ------------------------------------------------------------ scan
def scan_inputs(B, L, D, N, G, dtype, seed, state=True, lens=None, gate=True):
    from test_gpu_float_scan import make
    s = make(B, L, D, N, G, dtype, seed, state=state, gate=gate)
    s["lens"] = torch.tensor(lens, dtype=torch.int32) if lens is not None else None
    return s


def parts(B, L, D, N, G=1):
    from mamba_int import _lib
    bytes_ = ctypes.c_size_t()
    assert _lib.raw("mi_selective_scan_workspace_size", B, L, D, N, G, ctypes.byref(bytes_)) == 0
    return bytes_.value // (4 * B * (N + 1) * D)


def run_scan(s, B, cuda, in_place=True):
    from mamba_int import ops
    per_sequence = ("u", "dt", "b", "c", "z", "h_in", "lens")
    d = {k: repeated(v, B, cuda) if k in per_sequence else v.to(cuda) for k, v in s.items()}
    if not in_place or d["h_in"] is None:
        d["h_out"] = torch.full((B, *s["a"].shape), 7.0, device=cuda)
    else:
        d["h_out"] = d["h_in"]
    return ops.selective_scan(**d), d["h_out"]


def check_scan(s, got, h, dtype):
    y, ey, hw, eh = R.scan(s["u"], s["dt"], s["a"], s["b"], s["c"], s["d_skip"], s["z"], s["dt_bias"], True, s["h_in"],
                           s["lens"])
    R.close(h, hw, eh, torch.float32)
    R.close(got, y, ey, dtype)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("N,D,G", [(16, 448, 1), (4, 130, 1), (8, 130, 2), (5, 70, 1), (24, 130, 1), (64, 130, 2), (40, 70, 1),
                                   (100, 70, 1), (200, 70, 1)])
def test_scan_whole_sequences_of_many_tiles(cuda, N, D, G, dtype):
    """More blocks than half the CUs: a sequence is one part, of many tiles, the last one not whole."""
    L, blocks = 203, G * -(-D // G // 64)
    B = cus() // (2 * blocks) + 2
    assert parts(B, L, D, N, G) == 0
    s = scan_inputs(4, L, D, N, G, dtype, N + D, lens=[L, 0, 100, 17])
    got, h = run_scan(s, B, cuda)
    check_scan(s, check_repeated(got, 4), check_repeated(h, 4), dtype)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("L,D,N,G", [(700, 70, 24, 1), (520, 64, 32, 1), (600, 40, 17, 1), (400, 33, 100, 1), (300, 20, 128, 1),
                                     (300, 20, 200, 1), (260, 10, 256, 1), (300, 64, 96, 2), (90, 64, 16, 1), (40, 20, 12, 1)])
def test_scan_split_sequences(cuda, L, D, N, G, dtype):
    """Few blocks: sequences in parts, for every number of states a wave and tile length; lengths
    that end before, in and after a part; the state in place."""
    assert parts(3, L, D, N, G) >= 3
    s = scan_inputs(3, L, D, N, G, dtype, N + D, lens=[L, 0, 2 * L // 3 + 1])
    got, h = run_scan(s, 3, cuda)
    check_scan(s, got, h, dtype)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("L", [1, 2, 5, 8, 9])
@pytest.mark.parametrize("N,state", [(16, True), (16, False), (5, True), (5, False), (64, True), (200, False), (3, True)])
def test_scan_lengths_of_few_steps(cuda, L, N, state, dtype):
    """An odd batch with empty, whole and partly filled sequences, step by step and at the first length
    that goes by tiles; with and without a state, in place and not."""
    lens = [L, 0, (L + 1) // 2, L, 0, 1, min(2, L)]
    s = scan_inputs(7, L, 70, N, 1, dtype, N + L, state=state, lens=lens)
    for in_place in (True, False):
        got, h = run_scan(s, 7, cuda, in_place)
        check_scan(s, got, h, dtype)
        for b in range(7):
            assert (got[b, lens[b]:] == 0).all()
        if state:
            assert torch.equal(h[1].cpu(), s["h_in"][1])


# ------------------------------------------------------------ graphs
def test_graph_replays(cuda):
    """Captured, each replay equals the eager call, with eager work in between."""
    from mamba_int import ops
    x, r, w = torch.randn(37, 776, device=cuda), torch.randn(37, 776, device=cuda), torch.ones(776, device=cuda)
    c, cw = torch.randn(3, 70, 200, device=cuda), torch.randn(200, 4, device=cuda)
    state = torch.randn(3, 3, 200, device=cuda)
    s = w4_weights(333, 776, 64, 5, cuda)
    p, sc, z = s["packed"]
    calls = [lambda: ops.add_rms_norm(x, w, residual=r)[0], lambda: ops.add_rms_norm_quant(x, w, residual=r)[0],
             lambda: ops.causal_conv(c, cw, state_in=state), lambda: ops.causal_conv(c[:, :1], cw, state_in=state),
             lambda: ops.w4_matvec(x, p, sc, 333, 64, zeros=z), lambda: ops.w4_matvec(x[:2], p, sc, 333, 64, zeros=z)]
    want = [f() for f in calls]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for f in calls:
            f()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [f() for f in calls]
    for turn in range(3):
        for y in got:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for y, e, f in zip(got, want, calls):
            assert torch.equal(y, e) and torch.equal(f(), e)
