"""The float selective model: its path over a padded batch, in parts and token by token,
and its head, against a plain statement of the same layer."""
import math

import pytest
import torch

import float_ref as R

pytestmark = pytest.mark.gpu


def small(cuda, seed=0):
    from mamba_int.params import ModelDims
    from mamba_int.selective import SelectiveRunner, random_params
    return SelectiveRunner(random_params(ModelDims(d_model=128, n_layer=2, vocab_size=300, d_state=16, dt_rank=16), seed))


def unpack(p, k):
    """Ternary weights of packed words: weight 4 j + i of a word in bits 8 i + 2 j."""
    b = p.packed.cpu().long().view(p.n, -1, 4)
    q = torch.arange(16)
    code = (b[..., q & 3] >> (2 * (q >> 2))) & 3
    return torch.where(code >= 2, code - 4, code).reshape(p.n, -1)[:, :k].double()


def bitlinear(x, p):
    """BitLinear in 64 bits: activations in 8 bits by rows."""
    top = x.abs().amax(-1, keepdim=True).clamp(min=1e-8)
    q = torch.round(x * 127 / top).clamp(-127, 127)
    return (q @ unpack(p, x.shape[1]).t()) * (p.scale * top / 127)


def plain(run, ids, lens):
    P, d = run.params, run.dims
    B, L = ids.shape
    D, N, Rk = d.d_inner, d.d_state, d.dt_rank
    r, x = P.emb.cpu().double()[ids.cpu()], None

    def rms(v, w):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5) * w.cpu().double()
    for ly in P.layers:
        if x is not None:
            r = r + x
        uz = bitlinear(rms(r, ly.norm).view(B * L, -1), ly.w_in).view(B, L, 2 * D)
        u, _, _ = R.conv(uz[..., :D], ly.conv_w.cpu(), ly.conv_b.cpu(), True, None, lens)
        xp = bitlinear(u.view(B * L, D), ly.w_x)
        dt = bitlinear(xp[:, :Rk], ly.w_dt).view(B, L, D)
        xp = xp.view(B, L, -1)
        y, _, _, _ = R.scan(u, dt, ly.a.cpu(), xp[..., Rk:Rk + N].unsqueeze(2), xp[..., Rk + N:].unsqueeze(2), ly.d.cpu(),
                            uz[..., D:], ly.dt_bias.cpu(), True, None, lens)
        x = bitlinear(y.view(B * L, D), ly.w_out).view(B, L, -1)
    last = (lens.long() if lens is not None else torch.full((B,), L)) - 1
    rows = (torch.arange(B), last)
    y = rms((r + x)[rows], P.norm_f)
    packed, scales, zeros = (t.cpu() for t in P.head)
    w = torch.zeros(d.vocab_size, d.d_model, dtype=torch.float64)
    words = packed.view(torch.int32).long().view(packed.shape[0], packed.shape[1], 256)
    for n in range(d.vocab_size):
        for k in range(d.d_model):
            i, c = k % 128, k % 8
            word = int(words[n // 16, k // 128, 4 * (16 * (i % 32 // 8) + n % 16) + i // 32])
            q = (word >> (4 * (c // 2) + 16 * (c % 2))) & 15
            w[n, k] = (q - int(zeros[n // 16, k // 64, n % 16])) * float(scales[n // 16, k // 64, n % 16])
    return y @ w.t()


def near(got, want):
    # a value of 8 bits that rounds to its other neighbour moves a projection's output by
    # 1 / 127 of its row's largest product: a few of them in a hundred leave a relative
    # 1e-3 in a layer
    d = (got.double().cpu() - want.double().cpu()).norm() / want.double().norm().cpu()
    assert float(d) < 0.02, float(d)


def test_padded_prompts_against_the_plain_model(cuda):
    run = small(cuda)
    ids = torch.randint(0, 300, (3, 21), generator=torch.Generator().manual_seed(1)).to(cuda)
    near(run.forward(ids, run.new_state(3)), plain(run, ids, None))
    lens = torch.tensor([21, 9, 1], dtype=torch.int32)
    near(run.forward(ids, run.new_state(3), lens.to(cuda)), plain(run, ids, lens))


def test_parts_and_tokens_are_the_prompt(cuda):
    run = small(cuda, 3)
    ids = torch.randint(0, 300, (2, 40), generator=torch.Generator().manual_seed(2)).to(cuda)
    whole = run.new_state(2)
    want = run.forward(ids, whole)
    state = run.new_state(2)
    run.forward(ids[:, :17], state)
    run.forward(ids[:, 17:35], state)
    for t in range(35, 40):
        got = run.forward(ids[:, t:t + 1], state)
    near(got, want)
    for a, b in zip(state.h + state.conv, whole.h + whole.conv):
        near(a, b)


def test_generate_follows_the_logits(cuda):
    run = small(cuda, 5)
    ids = torch.randint(0, 300, (2, 12), generator=torch.Generator().manual_seed(4)).to(cuda)
    new = run.generate(ids, 5)
    assert new.shape == (2, 5) and run.generate(ids, 0).shape == (2, 0)
    logits = run.forward(ids, run.new_state(2))
    assert torch.equal(new[:, :1], logits.argmax(-1, keepdim=True))


def test_quantized_head(cuda):
    """A group's codes hold its weights within half a step of its range in 15."""
    from mamba_int import ops
    from mamba_int.selective import quantize_w4
    w = torch.randn(50, 200, generator=torch.Generator().manual_seed(6)).to(cuda)
    packed, scales, zeros = quantize_w4(w, 64)
    back = ops.w4_matvec(torch.eye(200, device=cuda), packed, scales, 50, 64, zeros=zeros).t()
    step = torch.cat([w, w.new_zeros(50, 56)], 1).view(50, 4, 64)
    step = ((step.amax(-1).clamp(min=0) - step.amin(-1).clamp(max=0)) / 15).repeat_interleave(64, 1)[:, :200]
    assert ((back - w).abs() <= step * 1.01 + 1e-6).all()
