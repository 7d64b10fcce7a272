"""Adapters of many tokens against their formula in 64 bits: the grids where a block takes 64 tokens of
the first product, and several turns of tokens in the second."""
import pytest
import torch

import float_ref as R
from test_gpu_adapter import make, oracle, run

pytestmark = pytest.mark.gpu


def check(s, cuda):
    """In a new tensor against the formula, and in place to the bit."""
    got = run(s, cuda)
    R.close(got, *oracle(s), s["y"].dtype)
    y = s["y"].to(cuda)
    assert run(s, cuda, y=y, out=y) is y and torch.equal(y, got)


# 64 tokens of the first product from 256 of them on (CUs of the card); 64 of the second where that leaves 1024 blocks
@pytest.mark.parametrize("x_type", R.TYPES + [torch.int8])
@pytest.mark.parametrize("w_type", R.TYPES)
@pytest.mark.parametrize("rank", [5, 20, 50, 100])
def test_many_tokens(cuda, rank, x_type, w_type):
    s = make(8, 2048, 97, 801, rank, 3, x_type, w_type, rank)
    s["lens"] = torch.tensor([2048, 2047, 0, 1, 64, 65, 1000, 2033], dtype=torch.int32)
    s["ids"][0] = 1
    check(s, cuda)


@pytest.mark.parametrize("x_type", R.TYPES + [torch.int8])
@pytest.mark.parametrize("K,N,rank", [(256, 1024, 16), (264, 1100, 64), (65, 777, 33)])
def test_tokens_past_whole_tiles(cuda, K, N, rank, x_type):
    check(make(5, 4100, K, N, rank, 4, x_type, torch.bfloat16, K), cuda)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("L", [64 * 65535, 64 * 65535 + 1, (1 << 22) - 1])
def test_the_longest_sequences(cuda, L, dtype):
    """From 64 * 65535 tokens on a block of the second product takes 128."""
    check(make(1, L, 2, 1, 1, 1, dtype, torch.float32, 3, none=0.0), cuda)
