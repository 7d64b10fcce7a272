"""Token sampling where a row is shared by several blocks (few rows of more than 8192 tokens), beside
the same where it is not: rows of every kind in one call, masked and infinite logits, numbers out of
range, replays on a used workspace."""
import numpy as np
import pytest
import torch

import sample_ref as R
from test_gpu_sample import TYPES, at, check, make, run
from test_host_sample import mixed as mixed_rows

pytestmark = pytest.mark.gpu
FLOATS = [torch.float32, torch.bfloat16, torch.float16]
VOCABS = [777, 9001, 40000]
LOWEST = -2 ** 31


def mixed(B, seed):
    return {n: torch.from_numpy(v) for n, v in mixed_rows(B, seed)[0].items()}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", VOCABS)
def test_rows_of_every_kind(cuda, V, dtype):
    B = 36
    logits, scale, u = make(B, V, dtype, V)
    par = mixed(B, 1)
    got, lp = run(cuda, logits, u, scale=scale, **par)
    check(logits, u, got, lp, scale=scale, **par)
    # a row's token does not depend on its neighbours, nor on how a parameter is given
    one = [run(cuda, logits[b:b + 1], u[b:b + 1], scale=scale, **{n: v[b].item() for n, v in par.items() if v[b] == v[b]})[0].item()
           for b in range(B) if par["temperature"][b] == par["temperature"][b]]
    assert one == [t for b, t in enumerate(got.tolist()) if par["temperature"][b] == par["temperature"][b]]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("V", VOCABS)
def test_masked_and_infinite(cuda, V, dtype):
    """Whole slices that hold nothing to draw, too."""
    g = torch.Generator().manual_seed(2)
    low, inf, nan = torch.finfo(dtype).min, float("inf"), float("nan")
    logits = torch.randn(13, V, generator=g).to(dtype)
    hole = torch.rand(13, V, generator=g) < 0.9
    for b, v in enumerate((-inf, low, nan)):
        logits[b][hole[b]] = v
        logits[3 + b, : V - 300] = v
        logits[6 + b, 300:] = v
    logits[9], logits[10] = -inf, nan
    logits[11, 100], logits[11, V - 5] = inf, inf
    logits[12] = -inf
    logits[12, V // 2] = low
    u = torch.rand(13, generator=g)
    for par in (dict(), dict(top_k=20), dict(top_p=0.8), dict(temperature=0.0), dict(top_k=600, top_p=0.7, min_p=0.01),
                dict(top_p=0.9, min_p=0.01), dict(temperature=1e-38), dict(temperature=inf)):
        got, lp = run(cuda, logits, u, **par)
        check(logits, u, got, lp, **par)
        assert got[9].item() == -1 and got[10].item() == -1 and lp[9].item() == -inf


@pytest.mark.parametrize("V", VOCABS)
def test_numbers_out_of_range(cuda, V):
    """u outside [0, 1), and filters of NaN."""
    logits, _, _ = make(6, V, torch.float32, 3)
    u = torch.tensor([1.0, 5.0, float("inf"), float("nan"), -1.0, 0.0])
    for par in (dict(top_k=10), dict(top_k=900), dict(top_p=0.9), dict()):
        got, lp = run(cuda, logits, u, **par)
        check(logits, u.clamp(max=1.0), got, lp, **par)
    nan = torch.full((6,), float("nan"), device=cuda)
    u = torch.rand(6)
    plain, _ = run(cuda, logits, u)
    assert torch.equal(run(cuda, logits, u, top_p=nan, min_p=nan)[0], plain)
    assert torch.equal(run(cuda, logits, u, temperature=nan)[0], logits.argmax(1).to(cuda))


@pytest.mark.parametrize("V", [5000, 20000])
def test_lowest_integers(cuda, V):
    """int32 logits from the lowest one up, nearly alike, cut near the order's end; and half of them
    the lowest, half 0, alike at an infinite temperature."""
    g = torch.Generator().manual_seed(V)
    logits = (LOWEST + torch.randint(0, 5_000_000, (4, V), generator=g)).to(torch.int32)
    u = torch.tensor([0.0, 0.31, 0.77, 0.9999])
    for below in (1, 2, 10, 260, 2500, 4900):
        for par in (dict(top_k=V - below), dict(top_p=np.float32(1 - (below + 0.5) / V).item())):
            got, lp = run(cuda, logits, u, scale=1e-12, **par)
            check(logits, u, got, lp, scale=1e-12, **par)
    logits = torch.where(torch.rand(4, V, generator=g) < 0.5, 0, LOWEST).to(torch.int32)
    for par in (dict(top_k=V * 3 // 4), dict(top_p=0.9), dict(top_k=V - 50, top_p=0.95)):
        got, lp = run(cuda, logits, u, temperature=float("inf"), **par)
        check(logits, u, got, lp, temperature=float("inf"), **par)


@pytest.mark.parametrize("dtype", [torch.float32, torch.int32])
@pytest.mark.parametrize("V", VOCABS)
def test_replays_on_a_used_workspace(cuda, V, dtype):
    """Captured once; every replay has other logits, and another kind of filter in each row."""
    from mamba_int import ops
    B = 14
    logits, scale, u = make(B, V, dtype, 9)
    logits, u = logits.to(cuda), u.to(cuda)
    par = {n: v.to(cuda) for n, v in mixed(B, 0).items()}
    ops.sample_tokens(logits, u, scale=scale, **par)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, lp = ops.sample_tokens(logits, u, scale=scale, logprob=True, **par)
    for seed in range(6):
        new, _, un = make(B, V, dtype, 20 + seed)
        if dtype == torch.float32 and seed % 2:
            new[seed] = -float("inf")
        logits.copy_(new), u.copy_(un)
        for n, v in mixed(B, seed).items():
            par[n].copy_(v)
        graph.replay()
        want, wlp = ops.sample_tokens(logits, u, scale=scale, logprob=True, **par)
        torch.cuda.synchronize()
        assert torch.equal(ids, want) and torch.equal(lp, wlp)
        rows = {n: v.clone() for n, v in mixed(B, seed).items()}
        check(new, un, ids, lp, scale=scale, **rows)


def test_two_graphs_and_a_stream(cuda):
    """Two captured calls and an eager one have workspaces of their own: replayed at the same time
    on streams, each draws its own tokens."""
    from mamba_int import ops
    B, V = 8, 40000
    side = [torch.cuda.Stream() for _ in range(2)]
    graphs, got, want, inputs = [], [], [], []
    for i in range(2):
        logits, _, u = make(B, V, torch.float32, 50 + i)
        logits, u = logits.to(cuda), u.to(cuda)
        inputs.append((logits, u))      # (a graph reads them at every replay)
        want.append(ops.sample_tokens(logits, u, top_p=0.9 - 0.2 * i))
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            got.append(ops.sample_tokens(logits, u, top_p=0.9 - 0.2 * i))
    logits, _, u = make(B, V, torch.float32, 60)
    logits, u = logits.to(cuda), u.to(cuda)
    third = ops.sample_tokens(logits, u, top_k=500)
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(side[i]):
                got[i].zero_()
                graphs[i].replay()
        now = ops.sample_tokens(logits, u, top_k=500)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(now, third)


def test_many_slices(cuda):
    """Vocabularies past 64 slices of 8192 tokens, with slices that grow."""
    for V in (524288, 1 << 20, (1 << 22) + 3):
        logits, _, u = make(2, V, torch.float32, V % 1000, spread=3.0)
        for par in (dict(top_k=50, top_p=0.9), dict(top_p=0.9), dict(min_p=0.05)):
            got, lp = run(cuda, logits, u, **par)
            for b in range(2):
                token, p, border = R.draw(logits[b].double().numpy(), at(u, b), **{n: at(v, b) for n, v in par.items()})
                # masses are in units of 2^-39 and finer, so V of them are off by V * 2^-40 of the
                # largest's, a cut and the draw by twice that each
                if border < V * 2.0 ** -38:
                    continue
                assert got[b].item() == token, (V, par, b)
                assert abs(lp[b].item() - np.log(p)) <= V * 2.0 ** -39 + 2.0 ** -28 - 2.0 ** -24 * np.log(p), (V, par, b)
