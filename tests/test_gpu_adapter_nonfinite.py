"""Infinite values in the adapters' inputs give what the formula in 64 bits gives, for rows and for
tiles of tokens alike."""
import pytest
import torch

import float_ref as R
from test_gpu_adapter import make, oracle, run
from test_gpu_float_nonfinite import same

pytestmark = pytest.mark.gpu
INF = float("inf")


def check(s, cuda, infinite=True):
    want, err = oracle(s)
    odd = ~torch.isfinite(want)
    assert odd.any() == infinite and not odd.all()
    got = run(s, cuda)
    same(got, want, err, s["y"].dtype)
    y = s["y"].to(cuda)
    run(s, cuda, y=y, out=y)
    assert torch.equal(y.nan_to_num(7.0), got.nan_to_num(7.0)) and torch.equal(torch.isnan(y), torch.isnan(got))


@pytest.mark.parametrize("x_type", R.TYPES)
@pytest.mark.parametrize("w_type", R.TYPES)
@pytest.mark.parametrize("L,rank", [(1, 1), (7, 1), (8, 1), (40, 1), (40, 20), (130, 40), (33, 100)])
def test_infinite_rows(cuda, L, rank, x_type, w_type):
    """One rank: the row is infinite in every column.  More: the ranks' infinities meet in sums."""
    s = make(3, L, 75, 150, rank, 2, x_type, w_type, L + rank, none=0.0)
    s["x"][1, L // 2, 3] = INF
    s["x"][2, L - 1, 74] = -INF
    s["x"][0, 0, 10] = s["x"][0, 0, 70] = INF
    if L > 1:
        s["x"][0, 1, 20], s["x"][0, 1, 21] = INF, -INF
    s["x"][2, 0, 5] = float("nan")
    if L == 1:
        s["x"][1] = 1.0      # (a row without)
    check(s, cuda)


@pytest.mark.parametrize("w_type", R.TYPES)
@pytest.mark.parametrize("x_type", R.TYPES + [torch.int8])
@pytest.mark.parametrize("L,rank", [(3, 4), (50, 1), (50, 4), (50, 60)])
def test_infinite_adapters_and_scales(cuda, L, rank, x_type, w_type):
    s = make(6, L, 64, 90, rank, 6, x_type, w_type, L, none=0.0)
    s["ids"] = torch.arange(6, dtype=torch.int32)
    s["a"][1, rank - 1, 7] = INF
    s["b"][2, 60, 0] = -INF
    s["scales"][3] = INF
    s["b"][4, 11, rank // 2], s["scales"][4] = float("nan"), 1.0
    s["scales"][5] = -INF
    check(s, cuda)


@pytest.mark.parametrize("L", [2, 30])
def test_infinite_scales_of_rows(cuda, L):
    s = make(2, L, 64, 90, 1, 2, torch.int8, torch.bfloat16, L, none=0.0)
    s["x_scale"][1, L - 1], s["x_scale"][0, 0] = INF, -INF
    check(s, cuda)


@pytest.mark.parametrize("dtype", R.TYPES)
def test_infinite_base_rows(cuda, dtype):
    """y's infinities stay, in rows and in columns past whole vectors."""
    s = make(2, 30, 64, 93, 6, 2, dtype, torch.bfloat16, 4, none=0.0)
    s["y"][0, 3, 92], s["y"][1, 29, 1], s["y"][1, 7, 40] = INF, -INF, float("nan")
    check(s, cuda)
