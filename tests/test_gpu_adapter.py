"""Low-rank adapters against their formula in 64 bits: types, ranks, odd sizes, sequences and
single rows, requests without an adapter, lengths, strides, in place, 8-bit rows, graphs.

The bound: a product of k terms in any order of 32-bit sums is off by (k + 8) U of the sum of
their magnitudes (tests/float_ref.py), which goes through the second product; that adds (rank
+ 8) U of its own, the two scales 2 U, the sum with y one."""
import pytest
import torch

import float_ref as R

pytestmark = pytest.mark.gpu


def make(B, L, K, N, rank, bank, x_type, w_type, seed, y_type=None, lens=False, none=0.3, scales=True):
    g = torch.Generator().manual_seed(seed)
    s = {"x_scale": None, "lens": None, "scales": None}
    if x_type == torch.int8:
        s["x"] = torch.randint(-127, 128, (B, L, K), generator=g).to(torch.int8)
        s["x_scale"] = torch.rand(B, L, generator=g) / 50
    else:
        s["x"] = torch.randn(B, L, K, generator=g).to(x_type)
    s["y"] = torch.randn(B, L, N, generator=g).to(y_type or (torch.float32 if x_type == torch.int8 else x_type))
    s["a"], s["b"] = torch.randn(bank, rank, K, generator=g).to(w_type), torch.randn(bank, N, rank, generator=g).to(w_type)
    ids = torch.randint(0, bank, (B,), generator=g)
    s["ids"] = torch.where(torch.rand(B, generator=g) < none, -1, ids).int()
    if scales:
        s["scales"] = torch.randn(bank, generator=g)
    if lens:
        s["lens"] = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32)
        s["lens"][0] = L
        s["lens"][-1] = 0
    return s


def oracle(s):
    y = s["y"].double()
    err = torch.zeros_like(y)
    bank, rank, K = s["a"].shape
    for b in range(y.shape[0]):
        j = int(s["ids"][b])
        n = y.shape[1] if s["lens"] is None else min(max(int(s["lens"][b]), 0), y.shape[1])
        if not 0 <= j < bank or n == 0:
            continue
        x, a, w = s["x"][b, :n].double(), s["a"][j].double(), s["b"][j].double()
        f = s["scales"][j].double() if s["scales"] is not None else torch.ones((), dtype=torch.float64)
        f = f * (s["x_scale"][b, :n, None].double() if s["x_scale"] is not None else 1.0)
        t, mt = f * (x @ a.t()), f.abs() * (x.abs() @ a.abs().t())
        et = (K + 10) * R.U * mt
        d, md = t @ w.t(), t.abs() @ w.abs().t()
        y[b, :n] += d
        err[b, :n] = et @ w.abs().t() + (rank + 8) * R.U * md + R.U * (d.abs() + y[b, :n].abs())
    return y, err


def run(s, cuda, **more):
    from mamba_int import ops
    d = {k: v.to(cuda) if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    d.update(more)
    return ops.adapter_add(**d)


def check(s, got):
    R.close(got, *oracle(s), s["y"].dtype)


SHAPES = [(1, 1, 1, 1, 1, 1), (8, 1, 64, 64, 8, 4), (5, 1, 100, 70, 5, 3), (3, 1, 2048, 768, 16, 9), (2, 3, 33, 17, 3, 2),
          (2, 16, 64, 128, 16, 2), (3, 17, 130, 65, 12, 5), (1, 64, 256, 192, 32, 1), (2, 65, 96, 200, 64, 3), (2, 31, 200, 1108, 7, 4),
          (1, 130, 1000, 129, 128, 2), (1, 40, 72, 96, 33, 2), (4, 8, 4100, 48, 4, 4), (70, 1, 40, 300, 2, 128),
          (2, 20, 72, 100, 80, 2), (3, 9, 31, 15, 17, 2), (1, 300, 520, 260, 24, 2)]


@pytest.mark.parametrize("x_type", R.TYPES + [torch.int8])
@pytest.mark.parametrize("w_type", R.TYPES)
@pytest.mark.parametrize("B,L,K,N,rank,bank", SHAPES)
def test_adapters(cuda, B, L, K, N, rank, bank, x_type, w_type):
    s = make(B, L, K, N, rank, bank, x_type, w_type, B + L + K)
    check(s, run(s, cuda))


@pytest.mark.parametrize("y_type", [torch.bfloat16, torch.float16])
def test_bytes_beside_short_floats(cuda, y_type):
    s = make(3, 40, 128, 80, 9, 3, torch.int8, torch.bfloat16, 1, y_type=y_type)
    check(s, run(s, cuda))


@pytest.mark.parametrize("x_type", [torch.float32, torch.bfloat16, torch.int8])
@pytest.mark.parametrize("L", [3, 50, 200])
def test_lengths(cuda, x_type, L):
    """Rows past a sequence's length are y's, whatever x holds there, and rows without an adapter."""
    s = make(6, L, 100, 72, 6, 3, x_type, torch.float16, L, lens=True)
    s["ids"] = torch.tensor([0, 1, 2, -1, 7, 1], dtype=torch.int32)
    want = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    for b in range(6):
        n = int(s["lens"][b]) if b not in (3, 4) else 0
        if s["x"].is_floating_point():
            s["x"][b, n:] = float("nan")
        else:
            s["x_scale"][b, n:] = float("nan")
    got = run(s, cuda)
    check(want, got)
    for b in range(6):
        n = int(s["lens"][b]) if b not in (3, 4) else 0
        assert torch.equal(got[b, n:].cpu(), s["y"][b, n:])
    y = s["y"].to(cuda)
    assert run(s, cuda, y=y, out=y) is y and torch.equal(y, got)


def test_lengths_out_of_range(cuda):
    s = make(3, 20, 64, 64, 4, 2, torch.float32, torch.float32, 2, none=0.0)
    s["lens"] = torch.tensor([-5, 999, 20], dtype=torch.int32)
    s["ids"] = torch.tensor([1, 1, -2 ** 31], dtype=torch.int32)
    check(s, run(s, cuda))


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("L", [1, 45])
def test_strides_and_in_place(cuda, dtype, L):
    """Views of wider rows at odd offsets, in and out, and y in place."""
    B, K, N = 3, 75, 90
    s = make(B, L, K, N, 6, 3, dtype, torch.bfloat16, 3)
    x = torch.zeros(B, L + 2, K + 5, dtype=dtype, device=cuda)[:, 1:L + 1, 3:K + 3]
    y = torch.zeros(B, L + 1, 2 * N + 1, dtype=dtype, device=cuda)
    o = torch.zeros(B, L, N + 3, dtype=dtype, device=cuda)
    x.copy_(s["x"])
    y[:, :L, N + 1:].copy_(s["y"])
    want = run(s, cuda)
    check(s, want)
    assert torch.equal(run(s, cuda, x=x, y=y[:, :L, N + 1:], out=o[..., 1:N + 1]), want)
    assert (o[..., 0] == 0).all() and (o[..., N + 1:] == 0).all()
    run(s, cuda, x=x, y=y[:, :L, N + 1:], out=y[:, :L, N + 1:])
    assert torch.equal(y[:, :L, N + 1:], want) and (y[..., :N + 1] == 0).all() and (y[:, L:] == 0).all()


def test_flat_rows(cuda):
    """[B, K] and [B, N] are sequences of one token."""
    s = make(7, 1, 60, 33, 4, 3, torch.int8, torch.float32, 4)
    want = run(s, cuda)
    flat = dict(s, x=s["x"][:, 0], y=s["y"][:, 0], x_scale=s["x_scale"][:, 0].contiguous())
    assert torch.equal(run(flat, cuda), want[:, 0])
    y = torch.zeros(7, 80, device=cuda)
    y[:, 5:38] = flat["y"].to(cuda)
    run(flat, cuda, y=y[:, 5:38], out=y[:, 5:38])
    assert torch.equal(y[:, 5:38], want[:, 0]) and (y[:, :5] == 0).all() and (y[:, 38:] == 0).all()


def test_one_adapter_for_all_and_rows_alike(cuda):
    """The same adapter twice, and a row of x for every token: each token's result is one row's."""
    s = make(4, 30, 64, 64, 8, 1, torch.float32, torch.bfloat16, 5, none=0.0)
    s["x"], s["y"] = s["x"][:1, :1].expand(4, 30, 64).contiguous(), s["y"][:1, :1].expand(4, 30, 64).contiguous()
    got = run(s, cuda)
    check(s, got)
    assert (got == got[0, 0]).all()
    d = {k: v.to(cuda) if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    from mamba_int import ops
    wide = ops.adapter_add(**dict(d, x=d["x"][:1, :1].expand(4, 30, 64), y=d["y"][:1, :1].expand(4, 30, 64)))
    assert torch.equal(wide, got)


def test_empty(cuda):
    s = make(3, 5, 16, 12, 4, 2, torch.float32, torch.float32, 6)
    assert run(dict(s, x=s["x"][:0], y=s["y"][:0], ids=s["ids"][:0]), cuda).shape == (0, 5, 12)
    assert run(dict(s, x=s["x"][:, :0], y=s["y"][:, :0]), cuda).shape == (3, 0, 12)
    for a, b, sc in ((s["a"][:0], s["b"][:0], s["scales"][:0]), (s["a"][:, :0], s["b"][:, :, :0], s["scales"])):
        assert torch.equal(run(dict(s, a=a.contiguous(), b=b.contiguous(), scales=sc), cuda).cpu(), s["y"])


def test_no_ranks_and_no_columns(cuda):
    """Nothing to add: y in a new tensor, for rows and for tiles."""
    for L in (2, 50):
        s = make(3, L, 16, 12, 4, 2, torch.float16, torch.float16, 6, none=0.0)
        none = dict(s, a=s["a"][:, :0].contiguous(), b=s["b"][:, :, :0].contiguous())
        assert torch.equal(run(none, cuda).cpu(), s["y"])
        none = dict(s, a=s["a"][:, :, :0].contiguous(), x=s["x"][..., :0].contiguous())
        assert torch.equal(run(none, cuda).cpu(), s["y"])


def test_nan_stays_in_its_row(cuda):
    for L in (1, 40):
        s = make(3, L, 64, 64, 8, 2, torch.float32, torch.float32, 7, none=0.0)
        clean = run(s, cuda)
        s["x"][1, L // 2, 5] = float("nan")
        got = run(s, cuda)
        bad = torch.zeros(3, L, dtype=torch.bool, device=cuda)
        bad[1, L // 2] = True
        assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], clean[~bad])


def test_repeats_and_graph_replays(cuda):
    from mamba_int import ops
    for B, L in ((6, 1), (2, 300)):
        s = make(B, L, 512, 320, 16, 4, torch.bfloat16, torch.bfloat16, 8)
        d = {k: v.to(cuda) if isinstance(v, torch.Tensor) else v for k, v in s.items()}
        want = ops.adapter_add(**d)
        assert torch.equal(ops.adapter_add(**d), want)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = ops.adapter_add(**d)
        for shift in range(3):
            d["ids"].copy_((s["ids"] + shift) % 4)
            graph.replay()
            want = ops.adapter_add(**d)
            torch.cuda.synchronize()
            assert torch.equal(got, want)


def test_refusals(cuda):
    from mamba_int import ops
    d = {k: v.to(cuda) if isinstance(v, torch.Tensor) else v
         for k, v in make(3, 5, 16, 12, 4, 2, torch.float32, torch.float32, 6).items()}
    for bad, err in ((dict(x=d["x"].half()), TypeError), (dict(ids=d["ids"].long()), TypeError), (dict(b=d["b"].half()), TypeError),
                     (dict(b=d["b"][:, :-1].contiguous()), ValueError), (dict(ids=d["ids"][:2]), ValueError),
                     (dict(x_scale=torch.ones(3, 5, device=cuda)), ValueError), (dict(x=d["x"].to(torch.int8)), ValueError),
                     (dict(x=d["x"][0]), ValueError), (dict(a=d["a"].transpose(1, 2)), ValueError), (dict(ids=None), TypeError),
                     (dict(out=d["y"].transpose(0, 1)), ValueError), (dict(lens=d["ids"][:1]), ValueError)):
        with pytest.raises(err):
            ops.adapter_add(**dict(d, **bad))
    base = torch.zeros(60, device=cuda)
    y, out = base.as_strided((3, 5, 4), (4, 12, 1)), base.as_strided((3, 5, 4), (20, 4, 1))
    with pytest.raises(ValueError, match="overlaps"):
        ops.adapter_add(**dict(d, y=y, b=d["b"][:, :4].contiguous(), out=out))
    wide = torch.zeros(2, 200, 8, device=cuda)
    with pytest.raises(ops._lib.MIError, match="rank"):
        ops.adapter_add(torch.zeros(1, 4, device=cuda), torch.zeros(1, 8, device=cuda), wide, torch.zeros(2, 4, 200, device=cuda), d["ids"][:1])
