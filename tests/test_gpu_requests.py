"""Requests of one batch together: a model with a selective and a gated layer, prompts of unequal
lengths, each with its own adapter and its own sampling parameters."""
import numpy as np
import pytest
import torch

import float_ref as R
import gated_ref as G
import sample_ref as S
from test_gpu_float_model import bitlinear, near

pytestmark = pytest.mark.gpu


def small(seed=0, gated=(1,)):
    from mamba_int.params import ModelDims
    from mamba_int.selective import SelectiveRunner, random_params
    return SelectiveRunner(random_params(ModelDims(d_model=128, n_layer=2, vocab_size=300, d_state=16, dt_rank=16), seed, gated=gated))


def bank(run, n, rank, ids, cuda, seed=5):
    from mamba_int.selective import Adapters
    g = torch.Generator().manual_seed(seed)
    d, D = run.dims.d_model, run.dims.d_inner

    def pair(k, m):
        return (torch.randn(n, rank, k, generator=g) / k ** 0.5).to(cuda).bfloat16(), \
            (torch.randn(n, m, rank, generator=g) / rank ** 0.5).to(cuda).bfloat16()
    # one projection without an adapter
    return Adapters([pair(d, 2 * D), pair(d, 2 * D)], [pair(D, d), None], torch.tensor(ids, dtype=torch.int32, device=cuda),
                    (0.5 + torch.rand(n, generator=g)).to(cuda))


def low_rank(x, ab, ad):
    out = torch.zeros(*x.shape[:-1], ab[1].shape[1], dtype=torch.float64)
    for b, j in enumerate(ad.ids.tolist()):
        if 0 <= j < ab[0].shape[0]:
            out[b] = float(ad.scales[j]) * (x[b] @ ab[0][j].cpu().double().t() @ ab[1][j].cpu().double().t())
    return out


def plain(run, ids, lens, ad):
    """The last rows' hidden values in 64 bits."""
    from mamba_int.selective import GATED_RATE, GatedLayer
    P, dims = run.params, run.dims
    B, L = ids.shape
    D, N, Rk = dims.d_inner, dims.d_state, dims.dt_rank
    r, x = P.emb.cpu().double()[ids.cpu()], None

    def rms(v, w):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5) * w.cpu().double()
    for i, ly in enumerate(P.layers):
        if x is not None:
            r = r + x
        v = rms(r, ly.norm).view(B * L, -1)
        uz = bitlinear(v, ly.w_in).view(B, L, 2 * D)
        top = v.abs().amax(-1, keepdim=True)
        q = (torch.round(v * 127 / top) * top / 127).view(B, L, -1)      # the rows that the adapter reads
        uz = uz + low_rank(q, ad.w_in[i], ad)
        u, _, _ = R.conv(uz[..., :D], ly.conv_w.cpu(), ly.conv_b.cpu(), True, None, lens)
        if isinstance(ly, GatedLayer):
            ri = bitlinear(u.view(B * L, D), ly.w_gates).view(B, L, 2 * D)
            y = G.gated(u, ri[..., :D], ri[..., D:], ly.decay.cpu(), uz[..., D:], rate=GATED_RATE, lens=lens)["y"][0]
        else:
            xp = bitlinear(u.view(B * L, D), ly.w_x)
            dt = bitlinear(xp[:, :Rk], ly.w_dt).view(B, L, D)
            xp = xp.view(B, L, -1)
            y, _, _, _ = R.scan(u, dt, ly.a.cpu(), xp[..., Rk:Rk + N].unsqueeze(2), xp[..., Rk + N:].unsqueeze(2), ly.d.cpu(),
                                uz[..., D:], ly.dt_bias.cpu(), True, None, lens)
        x = bitlinear(y.view(B * L, D), ly.w_out).view(B, L, -1)
        if ad.w_out[i] is not None:
            x = x + low_rank(y, ad.w_out[i], ad)
    return rms((r + x)[torch.arange(B), lens.long() - 1], P.norm_f)


def head(run, cuda):
    """The head's weights, from its products with the unit vectors."""
    from mamba_int import ops
    from mamba_int.selective import HEAD_GROUP
    packed, scales, zeros = run.params.head
    eye = torch.eye(run.dims.d_model, device=cuda)
    return ops.w4_matvec(eye, packed, scales, run.dims.vocab_size, HEAD_GROUP, zeros=zeros).double().cpu()


def test_prompts_with_adapters_against_the_plain_model(cuda):
    run = small()
    ids = torch.randint(0, 300, (4, 21), generator=torch.Generator().manual_seed(1)).to(cuda)
    lens = torch.tensor([21, 9, 1, 14], dtype=torch.int32)
    ad = bank(run, 3, 4, [2, 0, -1, 2], cuda)
    got = run.forward(ids, run.new_state(4), lens.to(cuda), ad)
    near(got, plain(run, ids, lens, ad) @ head(run, cuda))
    # an adapter moves its own sequences alone
    bare = run.forward(ids, run.new_state(4), lens.to(cuda))
    assert torch.equal(got[2], bare[2])
    assert all(float((got[b] - bare[b]).norm() / bare[b].norm()) > 0.05 for b in (0, 1, 3))


def test_parts_and_tokens_are_the_prompt(cuda):
    run = small(3, gated=(0, 1))
    ids = torch.randint(0, 300, (3, 40), generator=torch.Generator().manual_seed(2)).to(cuda)
    ad = bank(run, 2, 8, [1, 0, 7], cuda)
    whole = run.new_state(3)
    want = run.forward(ids, whole, adapters=ad)
    state = run.new_state(3)
    run.forward(ids[:, :17], state, adapters=ad)
    run.forward(ids[:, 17:35], state, adapters=ad)
    for t in range(35, 40):
        got = run.forward(ids[:, t:t + 1], state, adapters=ad)
    near(got, want)
    for a, b in zip(state.h + state.conv, whole.h + whole.conv):
        near(a, b)


def test_generation_draws_each_requests_tokens(cuda):
    """The drawn tokens are those of the definition on the logits of every step; one seed, one text."""
    from mamba_int.sampling import Sampling
    run = small(1)
    ids = torch.randint(0, 300, (4, 12), generator=torch.Generator().manual_seed(3)).to(cuda)
    lens = torch.tensor([12, 5, 8, 1], dtype=torch.int32, device=cuda)
    ad = bank(run, 3, 4, [2, 0, -1, 1], cuda)
    par = dict(temperature=torch.tensor([0.0, 0.7, 1.0, 1.5], device=cuda), top_k=torch.tensor([0, 20, 0, 5], dtype=torch.int32, device=cuda),
               top_p=torch.tensor([1.0, 0.9, 0.8, 1.0], device=cuda), min_p=0.01)

    def generator():
        g = torch.Generator(device=cuda)
        g.manual_seed(9)
        return g
    new = run.generate(ids, 6, lens, sampling=Sampling(generator=generator(), **par), adapters=ad)
    assert new.shape == (4, 6)
    assert torch.equal(new, run.generate(ids, 6, lens, sampling=Sampling(generator=generator(), **par), adapters=ad))
    g, state = generator(), run.new_state(4)
    logits = run.forward(ids, state, lens, ad)
    for i in range(6):
        u = torch.rand(4, device=cuda, generator=g)
        for b in range(4):
            token, _, border = S.draw(logits[b].double().cpu().numpy(), u[b].item(), par["temperature"][b].item(), par["top_k"][b].item(),
                                      par["top_p"][b].item(), np.float32(0.01).item())
            assert border < 2.0 ** -29 or new[b, i].item() == token
        logits = run.forward(new[:, i:i + 1], state, adapters=ad)


def test_integer_model_draws_from_its_logits(cuda):
    from mamba_int.sampling import Sampling
    from mamba_integer_model import MambaIntegerModel
    model = MambaIntegerModel({"d_model": 128, "n_layer": 2, "vocab_size": 500, "ssm_cfg": {"d_state": 16, "dt_rank": 16}})
    ids = torch.randint(0, 500, (3, 9), generator=torch.Generator().manual_seed(4)).to(cuda)
    greedy = model.generate(ids, 5)
    assert torch.equal(model.generate(ids, 5, sampling=Sampling(temperature=0.0)), greedy)
    assert torch.equal(model.generate(ids, 5, sampling=Sampling(top_k=1)), greedy)
    g = torch.Generator(device=cuda)
    g.manual_seed(1)
    new = model.generate(ids, 5, sampling=Sampling(temperature=2.0, top_k=50, generator=g))
    assert new.shape == greedy.shape and torch.equal(new[:, :9], ids)
    g.manual_seed(1)
    u = torch.rand(3, device=cuda, generator=g)
    logits = model.forward_int(ids)[:, -1]
    for b in range(3):
        token, _, border = S.draw(logits[b].cpu().numpy(), u[b].item(), 2.0, 50, scale=model.logit_scale)
        assert border < 2.0 ** -29 or new[b, 9].item() == token
    assert model.generate(ids, 0, sampling=Sampling()).shape == (3, 9)


def test_a_decode_step_of_requests_in_a_graph(cuda):
    """Forward, adapters and draw captured together, with other adapters and random numbers at each replay."""
    from mamba_int import ops
    run = small(2)
    ad = bank(run, 3, 4, [0, 1, -1, 2], cuda)
    tok, u = torch.zeros(4, 1, dtype=torch.int64, device=cuda), torch.rand(4, device=cuda)
    state, twin = run.new_state(4), run.new_state(4)

    def step(st):
        logits = run.forward(tok, st, adapters=ad)
        return ops.sample_tokens(logits, u, temperature=0.8, top_k=30, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(run.new_state(4))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(state)
    for i in range(4):
        tok.fill_(17 * i + 3)
        u.copy_(torch.rand(4, generator=torch.Generator().manual_seed(i)))
        ad.ids.copy_((ad.ids + 1) % 4 - 1)
        graph.replay()
        want = step(twin)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in zip(state.h + state.conv, twin.h + twin.conv):
            assert torch.equal(a, b)
