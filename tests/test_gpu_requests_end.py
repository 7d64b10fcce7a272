"""Generation where a sequence has nothing to draw."""
import pytest
import torch

from test_gpu_requests import small

pytestmark = pytest.mark.gpu


class Ending:
    """A Sampling that finds nothing to draw for one sequence at one step."""
    def __init__(self, row, step, **more):
        from mamba_int.sampling import Sampling
        self.inner, self.row, self.at, self.step = Sampling(**more), row, step, 0

    def draw(self, logits, scale=1.0):
        ids = self.inner.draw(logits, scale)
        if self.step == self.at:
            ids[self.row] = -1
        self.step += 1
        return ids


@pytest.mark.parametrize("step", [0, 2])
def test_a_sequence_without_a_token_ends(cuda, step):
    """-1 is no index of the embedding: the sequence has -1 from there on, the others are as before."""
    from mamba_int.sampling import Sampling
    run = small(4)
    ids = torch.randint(0, 300, (3, 7), generator=torch.Generator().manual_seed(5)).to(cuda)
    want = run.generate(ids, 6, sampling=Sampling(temperature=0.0))
    new = run.generate(ids, 6, sampling=Ending(1, step, temperature=0.0))
    assert torch.equal(new[[0, 2]], want[[0, 2]]) and torch.equal(new[1, :step], want[1, :step])
    assert (new[1, step:] == -1).all()


def test_logits_that_are_no_numbers(cuda):
    from mamba_int.sampling import Sampling
    run = small(5)
    run.params.emb[17] = float("nan")
    ids = torch.randint(0, 17, (3, 7), generator=torch.Generator().manual_seed(5)).to(cuda)
    ids[2, 6] = 17
    new = run.generate(ids, 5, sampling=Sampling(top_k=1))
    assert (new[2] == -1).all()
    assert torch.equal(new[:2], run.generate(ids[:2], 5, sampling=Sampling(top_k=1)))
