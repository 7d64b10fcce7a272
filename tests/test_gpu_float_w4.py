"""Products with 4-bit weights against the formula in 64 bits."""
import pytest
import torch

import float_ref as R

pytestmark = pytest.mark.gpu


def make(m, n, k, group, dtype, seed, zeros=True, bias=True, scale_type=torch.float16):
    g = torch.Generator().manual_seed(seed)
    ng = -(-k // group)
    return {"x": torch.randn(m, k, generator=g).to(dtype),
            "codes": torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8),
            "scales": ((0.5 + torch.rand(n, ng, generator=g)) / k ** 0.5).to(scale_type),
            "zeros": torch.randint(0, 16, (n, ng), generator=g, dtype=torch.uint8) if zeros else None,
            "bias": torch.randn(n, generator=g) if bias else None}


def run(s, group, cuda, x=None):
    from mamba_int import ops
    z = s["zeros"].to(cuda) if s["zeros"] is not None else None
    packed, scales, zeros = ops.pack_w4(s["codes"].to(cuda), s["scales"].to(cuda), group, zeros=z)
    b = s["bias"].to(cuda) if s["bias"] is not None else None
    return ops.w4_matvec(s["x"].to(cuda) if x is None else x, packed, scales, s["codes"].shape[0], group, zeros=zeros,
                         bias=b)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("m,n,k,group", [
    (1, 1, 1, 32), (1, 16, 128, 128), (1, 17, 129, 32), (1, 300, 768, 64), (2, 33, 1000, 128), (3, 64, 96, 32),
    (4, 48, 200, 64), (5, 1108, 1000, 64), (8, 100, 2048, 128), (16, 130, 256, 32), (17, 80, 384, 128), (31, 65, 511, 64),
    (64, 96, 640, 32), (65, 40, 300, 128), (130, 33, 257, 64), (1, 40, 4096, 256), (2, 24, 1030, 1152),
    (33, 512, 1536, 128), (1, 5000, 512, 128)])
def test_matvec(cuda, m, n, k, group, dtype):
    s = make(m, n, k, group, dtype, m + n + k)
    y, err = R.w4(s["x"], s["codes"], s["scales"], s["zeros"], group, s["bias"])
    R.close(run(s, group, cuda), y, err, dtype)


@pytest.mark.parametrize("zeros,bias,scale_type", [(False, False, torch.float16), (True, False, torch.float32),
                                                   (False, True, torch.bfloat16)])
@pytest.mark.parametrize("m", [1, 6, 40])
def test_options(cuda, m, zeros, bias, scale_type):
    s = make(m, 200, 700, 64, torch.float32, 7, zeros, bias, scale_type)
    y, err = R.w4(s["x"], s["codes"], s["scales"], s["zeros"], 64, s["bias"])
    R.close(run(s, 64, cuda), y, err, torch.float32)


@pytest.mark.parametrize("m", [1, 3, 20])
@pytest.mark.parametrize("dtype", R.TYPES)
def test_strided_rows_of_x(cuda, m, dtype):
    """Rows inside a wider buffer whose other columns are no numbers, at an odd offset."""
    s = make(m, 70, 333, 32, dtype, 5)
    y, err = R.w4(s["x"], s["codes"], s["scales"], s["zeros"], 32, s["bias"])
    for off, width in ((0, 512), (3, 341), (8, 344)):
        wide = torch.full((m, width), float("nan"), dtype=dtype, device=cuda)
        x = wide[:, off:off + 333]
        x.copy_(s["x"])
        R.close(run(s, 32, cuda, x), y, err, dtype)


def test_pack_layout(cuda):
    """The layout of include/mamba_int.h, word by word."""
    from mamba_int import ops
    g = torch.Generator().manual_seed(1)
    n, k, group = 21, 300, 64
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = torch.rand(n, 5, generator=g).half()
    zeros = torch.randint(0, 16, (n, 5), generator=g, dtype=torch.uint8)
    packed, so, zo = ops.pack_w4(codes.to(cuda), scales.to(cuda), group, zeros=zeros.to(cuda))
    words = packed.cpu().view(torch.int32).view(2, 3, 256).tolist()
    for row in range(32):
        for col in range(384):
            blk = words[row // 16][col // 128]
            i = col % 128
            c = i % 8
            w = blk[4 * (16 * (i % 32 // 8) + row % 16) + i // 32]
            got = (w >> (4 * (c // 2) + 16 * (c % 2))) & 15
            assert got == (int(codes[row, col]) if row < n and col < k else 0)
    full = torch.zeros(32, 6)
    full[:n, :5] = scales.float()
    assert torch.equal(so.cpu().float(), full.view(2, 16, 6).transpose(1, 2))
    full[:n, :5] = zeros.float()
    assert torch.equal(zo.cpu().float(), full.view(2, 16, 6).transpose(1, 2))


def test_a_row_of_no_numbers_stays_alone(cuda):
    s = make(6, 50, 256, 32, torch.float32, 4)
    want = run(s, 32, cuda)
    s["x"][2, 17] = float("nan")
    s["x"][4, 200] = float("inf")
    got = run(s, 32, cuda)
    assert torch.isnan(got[2]).all() and not torch.isfinite(got[4]).any()
    keep = [0, 1, 3, 5]
    assert torch.equal(got[keep], want[keep])


def test_wide_range_of_float_rows(cuda):
    """float32 rows keep 32 bits: values 2^40 apart within a row, and ones near the type's ends."""
    s = make(4, 64, 256, 128, torch.float32, 9, bias=False)
    s["x"] *= torch.exp2(torch.randint(-20, 21, (4, 256)).float())
    s["x"][1] *= 2.0 ** -60
    s["x"][2] *= 2.0 ** 90
    y, err = R.w4(s["x"], s["codes"], s["scales"], s["zeros"], 128, None)
    R.close(run(s, 128, cuda), y, err, torch.float32)


def test_empty(cuda):
    s = make(1, 33, 64, 32, torch.float32, 3)
    assert run(s, 32, cuda, torch.empty(0, 64, device=cuda)).shape == (0, 33)
