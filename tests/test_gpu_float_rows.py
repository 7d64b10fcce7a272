"""Which views the float operators take as rows, and what they refuse on the device."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_row_strides(cuda):
    """Adjacent elements, outputs that do not overlap."""
    from mamba_int import ops
    x = torch.randn(3, 4, 10, device=cuda)
    w = torch.ones(10, 1, device=cuda)

    def conv(v, **k):
        return ops.causal_conv(v, w[:v.shape[2]], activation=None, **k)
    for v in (x, x[..., :4], x[:, 1:3], x[:1], x[:, :1], x[:, :1].expand(3, 4, 10), x[:1].expand(3, 4, 10)):
        assert torch.equal(conv(v), v)
        out = torch.zeros(3, 4, 12, device=cuda)[:v.shape[0], :v.shape[1], 1:1 + v.shape[2]]
        assert conv(v, out=out) is out and torch.equal(out, v)
    for bad in (x.transpose(1, 2), x[..., ::2]):
        with pytest.raises(ValueError, match="adjacent"):
            conv(bad)
    for bad in (x[:, :1].expand(3, 4, 10), x[:1].expand(3, 4, 10), x.as_strided((3, 4, 10), (10, 10, 1))):
        with pytest.raises(ValueError, match="overlap"):
            conv(x, out=bad)
    with pytest.raises(ValueError, match="out must be"):
        conv(x, out=x[:2].clone())
    with pytest.raises(TypeError, match="out must be"):
        conv(x, out=x.half())


def test_gradients_are_refused(cuda):
    from mamba_int import ops
    x = torch.randn(3, 8, device=cuda, requires_grad=True)
    w = torch.ones(8, device=cuda)
    with pytest.raises(ValueError, match="forward only"):
        ops.add_rms_norm(x, w)
    with torch.no_grad():
        ops.add_rms_norm(x, w)
    ops.add_rms_norm(x.detach(), w)


def test_shapes_types_and_library_errors(cuda):
    from mamba_int import _lib, ops
    x, w = torch.randn(3, 8, device=cuda), torch.ones(8, device=cuda)
    with pytest.raises(ValueError, match="weight must be"):
        ops.add_rms_norm(x, w[:7])
    with pytest.raises(TypeError, match="weight must be float32, got float16"):
        ops.add_rms_norm(x, w.half())
    with pytest.raises(ValueError, match="residual must be"):
        ops.add_rms_norm(x, w, residual=x[:2])
    with pytest.raises(_lib.MIError, match="eps"):
        ops.add_rms_norm(x, w, eps=-1.0)
    with pytest.raises(_lib.MIError, match="width"):
        ops.causal_conv(x[None], torch.ones(8, 9, device=cuda))
    with pytest.raises(ValueError, match="state_in must be"):
        ops.causal_conv(x[None], torch.ones(8, 4, device=cuda), state_in=torch.zeros(1, 4, 8, device=cuda))
    with pytest.raises(TypeError, match="lens must be int32"):
        ops.causal_conv(x[None], torch.ones(8, 4, device=cuda), lens=torch.zeros(1, dtype=torch.int64, device=cuda))
    bc = torch.randn(1, 3, 2, 4, device=cuda)
    with pytest.raises(ValueError, match="groups of a row"):
        ops.selective_scan(x[None], x[None], -torch.ones(8, 4, device=cuda), bc.transpose(2, 3).contiguous().transpose(2, 3), bc)
    with pytest.raises(_lib.MIError, match="nstate"):
        ops.selective_scan(x[None], x[None], -torch.ones(8, 257, device=cuda), *[torch.ones(1, 3, 257, device=cuda)] * 2)
    packed, scales, _ = ops.pack_w4(torch.zeros(20, 64, dtype=torch.uint8, device=cuda), torch.ones(20, 2, device=cuda), 32)
    with pytest.raises(ValueError, match="packed must be"):
        ops.w4_matvec(torch.ones(1, 200, device=cuda), packed, scales, 20, 32)
    with pytest.raises(ValueError, match="scales must be"):
        ops.w4_matvec(torch.ones(1, 64, device=cuda), packed, scales[:1], 20, 32)
