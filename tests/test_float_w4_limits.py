"""Sizes of the 4-bit products that do not fit 32 bits (groups: refused before a tensor is looked at)."""
import pytest
import torch


@pytest.mark.parametrize("group", [2 ** 31, 2 ** 32 + 32, 2 ** 32 + 128, 2 ** 40, 2 ** 63 - 128, -2 ** 32 + 128])
def test_groups_past_32_bits_are_refused(group):
    """Cut to 32 bits, 2^32 + 128 would be a group of 128: more scales than were passed."""
    from mamba_int import ops
    codes = torch.zeros(4, 256, dtype=torch.uint8)
    with pytest.raises(ValueError, match="group="):
        ops.pack_w4(codes, torch.zeros(4, 1), group)
    with pytest.raises(ValueError, match="group="):
        ops.w4_matvec(torch.zeros(1, 256), None, torch.zeros(1, 1, 16), 4, group)


@pytest.mark.gpu
def test_codes_past_32_bits_are_refused(cuda):
    from mamba_int import ops
    codes = torch.empty((1, 2 ** 32 + 128), dtype=torch.uint8, device=cuda)
    with pytest.raises(ValueError, match="codes"):
        ops.pack_w4(codes, torch.zeros((1, 5), device=cuda), 2 ** 30)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [2 ** 31 - 128, 2 ** 30])
def test_groups_far_above_k(cuda, group):
    """One scale and zero point a row, as with a group that just holds it."""
    from mamba_int import ops
    g = torch.Generator().manual_seed(7)
    n, k = 70, 2048
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8).to(cuda)
    scales = (0.5 + torch.rand(n, 1, generator=g)).to(cuda)
    zeros = torch.randint(0, 16, (n, 1), generator=g, dtype=torch.uint8).to(cuda)
    x = torch.randn(3, k, generator=g).to(cuda)
    got, want = ([*ops.pack_w4(codes, scales, by, zeros=zeros)] for by in (group, k))
    for i in range(3):
        assert torch.equal(got[i], want[i])
    a, b = (ops.w4_matvec(x, *p[:2], n, by, zeros=p[2]) for p, by in ((got, group), (want, k)))
    assert torch.equal(a, b)
