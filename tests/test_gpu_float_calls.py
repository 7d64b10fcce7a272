"""What the float operators' calls refuse beside shapes and types, on the device."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def every_call(cuda):
    """name -> a small call, its first tensor's name."""
    from mamba_int import ops
    x, w = torch.randn(3, 16, device=cuda), torch.ones(16, device=cuda)
    a, bc = -torch.ones(16, 4, device=cuda), torch.randn(1, 3, 4, device=cuda)
    codes, scales = torch.zeros(4, 16, dtype=torch.uint8, device=cuda), torch.ones(4, 1, device=cuda)
    packed, s, _ = ops.pack_w4(codes, scales, 32)
    return {"norm": lambda: ops.add_rms_norm(x, w), "quant": lambda: ops.add_rms_norm_quant(x, w),
            "conv": lambda: ops.causal_conv(x[None], torch.ones(16, 4, device=cuda)),
            "scan": lambda: ops.selective_scan(x[None], x[None], a, bc, bc),
            "w4": lambda: ops.w4_matvec(x, packed, s, 4, 32), "pack": lambda: ops.pack_w4(codes, scales, 32)}


@pytest.mark.parametrize("name", ["norm", "quant", "conv", "scan", "w4", "pack"])
def test_tensors_of_another_device_than_the_streams(cuda, name, monkeypatch):
    """The call would run on the current device's stream, not behind what made its tensors."""
    from mamba_int import ops
    call = every_call(cuda)[name]
    call()
    stream, device = ops._here()
    assert device == cuda.index and stream == torch.cuda.current_stream().cuda_stream
    monkeypatch.setattr(ops, "_here", lambda: (stream, device + 1))
    with pytest.raises(ValueError, match="current device"):
        call()


def test_tangents_are_refused(cuda):
    """A dual tensor's result would have none, without an error."""
    from mamba_int import ops
    x, w = torch.randn(3, 16, device=cuda), torch.ones(16, device=cuda)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.add_rms_norm(dual, w), lambda: ops.add_rms_norm(x, w, residual=dual),
                     lambda: ops.causal_conv(dual[None], torch.ones(16, 4, device=cuda))):
            with pytest.raises(ValueError, match="forward only"):
                call()
        with torch.autograd.forward_ad._set_fwd_grad_enabled(False):
            ops.add_rms_norm(dual, w)
    ops.add_rms_norm(x, w)


def test_negated_views_are_refused(cuda):
    """Their memory holds the values before the negation."""
    from mamba_int import ops
    x, w = torch.randn(3, 16, device=cuda), torch.ones(16, device=cuda)
    neg = torch._neg_view(x)
    with pytest.raises(ValueError, match="resolve_neg"):
        ops.add_rms_norm(neg, w)
    assert torch.equal(ops.add_rms_norm(neg.resolve_neg(), w)[0], ops.add_rms_norm(-x, w)[0])


def test_written_tensors_count_a_version(cuda):
    """A backward pass that saved a buffer which a call has overwritten since is an error."""
    from mamba_int import ops
    x, w = torch.randn(3, 16, device=cuda), torch.ones(16, device=cuda)
    a, bc = -torch.ones(16, 4, device=cuda), torch.randn(1, 3, 4, device=cuda)
    packed, s, _ = ops.pack_w4(torch.zeros(4, 16, dtype=torch.uint8, device=cuda), torch.ones(4, 1, device=cuda), 32)
    out, res, state, h = (torch.empty(*v, device=cuda) for v in ((3, 16), (3, 16), (1, 3, 16), (1, 16, 4)))
    y = torch.empty(3, 4, device=cuda)
    calls = [((out, res), lambda: ops.add_rms_norm(x, w, residual=x, residual_out=res, out=out)),
             ((res,), lambda: ops.add_rms_norm_quant(x, w, residual=x, residual_out=res)),
             ((out, state), lambda: ops.causal_conv(x[None], torch.ones(16, 4, device=cuda), state_out=state, out=out[None])),
             ((out, h), lambda: ops.selective_scan(x[None], x[None], a, bc, bc, h_out=h, out=out[None])),
             ((y,), lambda: ops.w4_matvec(x, packed, s, 4, 32, out=y))]
    for buffers, call in calls:
        before, inputs = [b._version for b in buffers], (x._version, w._version)
        call()
        assert all(b._version > v for b, v in zip(buffers, before)) and inputs == (x._version, w._version)
    with torch.inference_mode():
        buf = torch.empty(3, 16, device=cuda)
        ops.add_rms_norm(x, w, out=buf)
    p = torch.ones(1, 16, 4, device=cuda, requires_grad=True)
    loss = (p * h).sum()
    ops.selective_scan(x[None], x[None], a, bc, bc, h_in=h, h_out=h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
