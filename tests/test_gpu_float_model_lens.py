"""Lengths of the float selective model's prompts: none, and more than the rows hold."""
import pytest
import torch

from test_gpu_float_model import small

pytestmark = pytest.mark.gpu


def prompts(cuda):
    return torch.randint(0, 300, (3, 9), generator=torch.Generator().manual_seed(8)).to(cuda)


def lens(cuda, *v):
    return torch.tensor(v, dtype=torch.int32, device=cuda)


def test_a_sequence_of_no_tokens_has_logits_of_zero(cuda):
    """... and keeps its state; not the logits of another sequence's row."""
    run, ids = small(cuda), prompts(cuda)
    want = run.forward(ids, run.new_state(3), lens(cuda, 4, 1, 9))
    state = run.new_state(3)
    for h in state.h + state.conv:
        h[1] = 0.5
    got = run.forward(ids, state, lens(cuda, 4, 0, 9))
    assert torch.equal(got[[0, 2]], want[[0, 2]])
    assert (got[1] == 0).all()
    for h in state.h + state.conv:
        assert (h[1] == 0.5).all()


def test_lengths_outside_the_rows_are_taken_as_within(cuda):
    run, ids = small(cuda), prompts(cuda)
    want = run.forward(ids, run.new_state(3), lens(cuda, 9, 0, 9))
    assert torch.equal(run.forward(ids, run.new_state(3), lens(cuda, 10, -3, 2 ** 31 - 1)), want)


def test_prompts_without_tokens_are_refused(cuda):
    run = small(cuda)
    with pytest.raises(ValueError, match="one token"):
        run.forward(torch.zeros((2, 0), dtype=torch.int64, device=cuda), run.new_state(2))
