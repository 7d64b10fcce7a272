"""Sampled generation of the integer model through the decode graph: the tokens of the eager steps."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def build(seed=0, d_model=128):
    from mamba_integer_model import MambaIntegerModel
    torch.manual_seed(seed)
    return MambaIntegerModel({"d_model": d_model, "n_layer": 2, "vocab_size": 500, "ssm_cfg": {"d_state": 16, "dt_rank": 16}})


def sampling(cuda, B, seed):
    from mamba_int.sampling import Sampling
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return Sampling(temperature=torch.linspace(0.0, 2.0, B, device=cuda), top_k=50, top_p=0.95, generator=g)


@pytest.mark.parametrize("B", [1, 3, 70])
def test_the_graphs_tokens_are_the_eager_ones(cuda, B, monkeypatch):
    model = build(B)
    ids = torch.randint(0, 500, (B, 9), generator=torch.Generator().manual_seed(B)).to(cuda)
    want = [model.generate(ids, n, use_graph=False, sampling=sampling(cuda, B, n)) for n in (1, 2, 12)]
    greedy = model.generate(ids, 12, use_graph=False)

    def no_step(*_):
        raise AssertionError("an eager step in a generation by graphs")
    monkeypatch.setattr(model.runner(cuda), "decode_step", no_step)
    for _ in range(2):
        for n, w in zip((1, 2, 12), want):
            assert torch.equal(model.generate(ids, n, sampling=sampling(cuda, B, n)), w)
            assert torch.equal(model.generate(ids, 12), greedy)
    assert len(set(want[2][-1, 9:].tolist())) > 1


def test_the_state_goes_on(cuda):
    """The state that a drawn generation leaves is the eager one's."""
    model = build(7)
    run = model.runner(cuda)
    ids = torch.randint(0, 500, (3, 5), generator=torch.Generator().manual_seed(1)).to(cuda)
    out = []
    for use_graph in (False, True):
        logits, state = run.prefill(ids)
        s = sampling(cuda, 3, 4)
        first = run.decode_loop(logits, state, 6, use_graph=use_graph, sampling=s, scale=model.logit_scale)
        more = run.decode_step(first[:, -1].contiguous(), state)
        out.append((first, more, *state.conv, *state.h))
    assert all(torch.equal(a, b) for a, b in zip(*out))
