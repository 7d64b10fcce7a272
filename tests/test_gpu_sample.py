"""Token sampling against its definition: types, sizes, filters alone and together, ties,
masked and infinite logits, parameters of every row, strides, graphs.

Tokens have to be equal.  The kernel's masses are e rounded to a unit of at least 2^-46 of
the largest (vocab <= 2^16 here) and to 2^-52 of itself, so a border between two tokens is
off by at most vocab * 2^-45 of the kept mass, 2^-29: a row whose u or top_p lies nearer
than that to a border is not judged (the oracle says how near; under 1 in 1000 rows)."""
import numpy as np
import pytest
import torch

import sample_ref as R

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16, torch.int32]


def make(B, V, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    l = spread * torch.randn(B, V, generator=g) - torch.log1p(torch.arange(V).float())[torch.randperm(V, generator=g)]
    if dtype == torch.int32:
        return torch.round(l * 1024).to(dtype), 1.0 / 1024, torch.rand(B, generator=g)
    return l.to(dtype), 1.0, torch.rand(B, generator=g)


def at(v, b):
    return v[b].item() if isinstance(v, torch.Tensor) else np.float32(v).item() if isinstance(v, float) else v


def check(logits, u, got, logprob, scale=1.0, **par):
    ids, lp = got.cpu(), logprob.cpu()
    rows = logits.double().numpy()
    judged = 0
    for b in range(rows.shape[0]):
        token, p, border = R.draw(rows[b], at(u, b), scale=scale, **{n: at(v, b) for n, v in par.items()})
        if border < 2.0 ** -29 and 0 < at(u, b) < 1 and len(set(rows[b])) > 8:
            continue
        judged += 1
        assert ids[b].item() == token, (b, ids[b].item(), token, border)
        want = np.log(p) if token >= 0 else -np.inf
        # the logarithm of a sum off by 2^-29, rounded to 32 bits
        assert lp[b].item() == want or abs(lp[b].item() - want) <= 2.0 ** -28 + 2.0 ** -24 * abs(want), (b, lp[b].item(), want)
    assert judged >= 0.9 * rows.shape[0]


def run(cuda, logits, u, **par):
    from mamba_int import ops
    par = {n: v.to(cuda) if isinstance(v, torch.Tensor) else v for n, v in par.items()}
    return ops.sample_tokens(logits.to(cuda), u.to(cuda), logprob=True, **par)


FILTERS = [dict(), dict(temperature=0.7, top_k=50, top_p=0.9), dict(top_p=0.95), dict(temperature=1.3, min_p=0.02),
           dict(top_k=1), dict(top_k=7, min_p=0.1), dict(temperature=0.0), dict(top_p=0.5, min_p=0.001, top_k=400),
           dict(temperature=3.0, top_p=0.999)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,V", [(3, 1), (3, 2), (5, 63), (5, 64), (4, 65), (9, 1000), (4, 1024), (3, 1025), (2, 4097), (6, 32000),
                                 (2, 50257)])
def test_filters(cuda, B, V, dtype):
    logits, scale, u = make(B, V, dtype, B + V)
    for par in FILTERS:
        got, lp = run(cuda, logits, u, scale=scale, **par)
        check(logits, u, got, lp, scale=scale, **par)


@pytest.mark.parametrize("dtype", TYPES)
def test_parameters_of_every_row(cuda, dtype):
    B, V = 40, 3001
    logits, scale, u = make(B, V, dtype, 4)
    g = torch.Generator().manual_seed(5)
    par = dict(temperature=torch.where(torch.rand(B, generator=g) < 0.2, 0.0, 0.3 + torch.rand(B, generator=g)),
               top_k=torch.randint(-1, 60, (B,), generator=g).int(), top_p=0.2 + torch.rand(B, generator=g),
               min_p=0.2 * torch.rand(B, generator=g) - 0.05)
    got, lp = run(cuda, logits, u, scale=scale, **par)
    check(logits, u, got, lp, scale=scale, **par)
    # a row's token does not depend on its neighbours, nor on how a parameter is given
    one = [run(cuda, logits[b:b + 1], u[b:b + 1], scale=scale, **{n: v[b].item() for n, v in par.items()})[0].item()
           for b in range(B)]
    assert one == got.tolist()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [10, 1000, 1500, 40000])
def test_equal_logits(cuda, V, dtype):
    """Ties go to the lower token: sums of equal masses are exact, so borders are as well."""
    logits = torch.full((8, V), 3, dtype=dtype)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.999, 1 - 2.0 ** -24, 0.3, 0.7])
    for par in (dict(), dict(top_k=V // 2), dict(top_p=0.5), dict(top_k=V // 2, top_p=0.5), dict(top_k=V - 1, min_p=1.0)):
        got, lp = run(cuda, logits, u, **par)
        check(logits, u, got, lp, **par)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("values", [2, 3, 40])
def test_many_ties(cuda, dtype, values):
    """A few values, each of thousands of tokens: cuts inside a value, in every bin."""
    g = torch.Generator().manual_seed(values)
    V = 30000
    logits = (torch.randint(0, values, (6, V), generator=g).float() * (0.01 if values > 3 else 0.7)).to(dtype)
    u = torch.rand(6, generator=g)
    for k in (1, 5, 999, 5000, 14999, 15000, 15001, 20000, V - 1):
        for p in (1.0, 0.3, 0.77):
            got, lp = run(cuda, logits, u, top_k=k, top_p=p)
            check(logits, u, got, lp, top_k=k, top_p=p)


def test_one_bin_of_unlike_values(cuda):
    """Thousands of float32 logits next to each other, none alike, and two far ones."""
    g = torch.Generator().manual_seed(1)
    V = 9000
    logits = 1.0 + 1e-3 * torch.rand(5, V, generator=g)
    logits[:, 17], logits[:, 4000] = 1.5, 1.2
    u = torch.rand(5, generator=g)
    for par in (dict(top_k=4321), dict(top_p=0.6), dict(top_k=6000, top_p=0.6), dict(top_k=2), dict(top_k=3)):
        got, lp = run(cuda, logits, u, **par)
        check(logits, u, got, lp, **par)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_masked_and_infinite(cuda, dtype):
    g = torch.Generator().manual_seed(2)
    low, inf, nan = torch.finfo(dtype).min, float("inf"), float("nan")
    logits = torch.randn(9, 777, generator=g).to(dtype)
    hole = torch.rand(9, 777, generator=g) < 0.9
    for b, v in enumerate((-inf, low, nan)):
        logits[b][hole[b]] = v
    logits[3], logits[4], logits[5] = -inf, low, nan
    logits[6, 100], logits[6, 300] = inf, inf
    logits[7] = -inf
    logits[7, 500] = low
    logits[8, ::2], logits[8, 1::2] = 0.0, -0.0
    u = torch.tensor([0.3, 0.6, 0.9, 0.5, 0.5, 0.5, 0.75, 0.5, 0.4])
    for par in (dict(), dict(top_k=20), dict(top_p=0.8), dict(temperature=0.0), dict(top_k=30, top_p=0.7, min_p=0.01),
                dict(temperature=1e-38), dict(temperature=inf)):
        got, lp = run(cuda, logits, u, **par)
        check(logits, u, got, lp, **par)
    assert got[3].item() == -1 and got[5].item() == -1 and lp[3].item() == -inf


def test_numbers_out_of_range(cuda):
    """u outside [0, 1), and filters of NaN."""
    logits, _, _ = make(6, 500, torch.float32, 3)
    u = torch.tensor([1.0, 5.0, float("inf"), float("nan"), -1.0, 0.0])
    got, lp = run(cuda, logits, u, top_k=10)
    check(logits, u.clamp(max=1.0), got, lp, top_k=10)
    nan = torch.full((6,), float("nan"), device=cuda)
    u = torch.rand(6)
    plain, _ = run(cuda, logits, u)
    assert torch.equal(run(cuda, logits, u, top_p=nan, min_p=nan)[0], plain)
    assert torch.equal(run(cuda, logits, u, temperature=nan)[0], logits.argmax(1).to(cuda))


def test_every_token_has_its_share(cuda):
    """A fine grid of u draws each token as often as its probability says."""
    n, V = 4096, 40
    logits = torch.randn(1, V, generator=torch.Generator().manual_seed(7))
    u = (torch.arange(n) + 0.5) / n
    got, _ = run(cuda, logits.expand(n, V), u, temperature=0.9)
    share = torch.bincount(got.cpu(), minlength=V) / n
    assert ((share - torch.softmax(logits[0].double() / 0.9, 0)).abs() <= 1.0 / n + 1e-6).all()
    assert (got[1:] >= got[:-1]).all()


def test_strides_and_outputs(cuda):
    from mamba_int import ops
    logits, _, u = make(5, 700, torch.float16, 8)
    wide = torch.zeros(5, 900, dtype=torch.float16, device=cuda)
    wide[:, 3:703] = logits.to(cuda)
    want = ops.sample_tokens(logits.to(cuda), u.to(cuda), top_p=0.9)
    out = torch.empty(5, dtype=torch.int64, device=cuda)
    assert ops.sample_tokens(wide[:, 3:703], u.to(cuda), top_p=0.9, out=out) is out and torch.equal(out, want)
    one = ops.sample_tokens(wide[:1, 3:703].expand(5, 700), u.to(cuda), top_p=0.9)
    assert one[0] == want[0]
    assert ops.sample_tokens(logits[:0].to(cuda), u[:0].to(cuda)).shape == (0,)


def test_graph_replays(cuda):
    """Captured with its parameters as tensors, replayed with others."""
    from mamba_int import ops
    B, V = 6, 5000
    logits, scale, u = make(B, V, torch.int32, 9)
    logits, u = logits.to(cuda), u.to(cuda)
    k = torch.full((B,), 30, dtype=torch.int32, device=cuda)
    p = torch.full((B,), 0.9, device=cuda)
    ops.sample_tokens(logits, u, top_k=k, top_p=p, scale=scale)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, lp = ops.sample_tokens(logits, u, top_k=k, top_p=p, scale=scale, logprob=True)
    for seed in range(4):
        logits.copy_(make(B, V, torch.int32, 20 + seed)[0])
        k.fill_(10 * seed)
        p.fill_(1.0 - 0.1 * seed)
        graph.replay()
        want, wlp = ops.sample_tokens(logits, u, top_k=k, top_p=p, scale=scale, logprob=True)
        torch.cuda.synchronize()
        assert torch.equal(ids, want) and torch.equal(lp, wlp)


def test_refusals(cuda):
    from mamba_int import ops
    x, u = torch.randn(3, 8, device=cuda), torch.rand(3, device=cuda)
    for bad, err in ((dict(temperature=torch.ones(2, device=cuda)), ValueError), (dict(top_k=torch.ones(3, device=cuda)), TypeError),
                     (dict(top_p=torch.ones(3)), ValueError), (dict(temperature="a"), TypeError), (dict(top_k=1.5), TypeError),
                     (dict(out=torch.empty(3, device=cuda)), TypeError)):
        with pytest.raises(err):
            ops.sample_tokens(x, u, **bad)
    with pytest.raises(ValueError):
        ops.sample_tokens(x, u[:2])
    with pytest.raises(ValueError, match="forward only"):
        ops.sample_tokens(x.requires_grad_(), u)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_row_alone_and_among_many(cuda, dtype):
    """Few rows are shared by several blocks, many are not: a row's token is the same."""
    logits, _, u = make(5, 40000, dtype, 11, spread=0.7)
    many = logits.repeat(120, 1)
    for par in (dict(), dict(top_p=0.9), dict(top_k=300, top_p=0.8), dict(top_k=20000), dict(top_p=0.5, min_p=0.01), dict(min_p=0.3)):
        got, lp = run(cuda, logits, u, **par)
        check(logits, u, got, lp, **par)
        all_, lps = run(cuda, many, u.repeat(120), **par)
        assert torch.equal(all_, got.repeat(120)) and torch.equal(lps, lp.repeat(120))
