"""Residual addition + RMS norm with float and 8-bit outputs against the formula in 64 bits."""
import pytest
import torch

import float_ref as R

pytestmark = pytest.mark.gpu
EPS = 1e-5


def make(rows, dim, xt, rt, seed, wide=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, wide * dim, generator=g).to(xt)[:, :dim]
    r = (3 * torch.randn(rows, dim, generator=g)).to(rt) if rt is not None else None
    w = 1 + 0.2 * torch.randn(dim, generator=g)
    return x, r, w


def check_quant(q, scale, y, dim):
    m = y.abs().amax(-1).clamp(min=1e-8)
    assert ((scale.cpu().double() - m / 127).abs() <= 60 * R.U * m / 127).all()
    qd = q.cpu().double()
    assert (qd[:, dim:] == 0).all()
    # nearest of 255 levels: half a level, and what 32 bits move a value of up to 127 of them
    assert ((qd[:, :dim] - y / (m / 127)[:, None]).abs() <= 0.5 + 127 * 120 * R.U).all()


@pytest.mark.parametrize("xt,rt", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                   (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                   (torch.float16, torch.float32), (torch.float32, None), (torch.bfloat16, None)])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (8, 768), (5, 1000), (2, 1001), (33, 64), (4, 2048), (3, 2050),
                                      (2, 4096), (2, 8192), (1, 8193), (2, 16384), (257, 384)])
def test_norm(cuda, rows, dim, xt, rt):
    from mamba_int import ops
    x, r, w = make(rows, dim, xt, rt, rows * 7 + dim)
    s, y, ey = R.norm(x, r, w, EPS)
    xd, wd, rd = x.to(cuda), w.to(cuda), r.to(cuda) if r is not None else None
    got, res = ops.add_rms_norm(xd, wd, residual=rd, eps=EPS)
    R.close(got, y, ey, xt)
    q, scale, res2 = ops.add_rms_norm_quant(xd, wd, residual=rd, eps=EPS)
    check_quant(q, scale, y, dim)
    assert q.shape[1] % 64 == 0
    if r is None:
        assert res is None and res2 is None
    else:
        want = (x.float() + r.float()).to(rt)
        assert torch.equal(res.cpu(), want) and torch.equal(res2.cpu(), want)
        assert torch.equal(rd.cpu(), r)


@pytest.mark.parametrize("dim", [768, 1003])
def test_strided_rows_and_in_place(cuda, dim):
    from mamba_int import ops
    x, r, w = make(9, dim, torch.bfloat16, torch.float32, 3, wide=2)
    assert not x.is_contiguous()
    s, y, ey = R.norm(x, r, w, EPS)
    xd = torch.empty(9, 2 * dim, dtype=torch.bfloat16, device=cuda)[:, :dim]
    xd.copy_(x)
    rd = r.to(cuda)
    got, res = ops.add_rms_norm(xd, w.to(cuda), residual=rd, eps=EPS, residual_out=rd, out=xd)
    assert res is rd and got is xd
    R.close(got, y, ey, torch.bfloat16)
    assert torch.equal(rd.cpu(), x.float() + r)
    # rows at an odd element offset (no vector alignment)
    big = torch.empty(9 * (dim + 1) + 1, dtype=torch.bfloat16, device=cuda)
    xo = big[1:].view(9, dim + 1)[:, :dim]
    xo.copy_(x)
    R.close(ops.add_rms_norm(xo, w.to(cuda), residual=r.to(cuda), eps=EPS)[0], y, ey, torch.bfloat16)


def test_quantizer_is_act_quants(cuda):
    """The 8-bit rows are those that BitLinear's quantizer makes of the float norm, bit for bit."""
    from mamba_int import ops
    x, r, w = make(37, 776, torch.float32, torch.float32, 5)
    x, r, w = x.to(cuda), r.to(cuda), w.to(cuda)
    y, _ = ops.add_rms_norm(x, w, residual=r, eps=EPS)
    q, s, _ = ops.add_rms_norm_quant(x, w, residual=r, eps=EPS)
    q2, s2 = ops.act_quant(y)
    assert torch.equal(q[:, :776], q2) and torch.equal(s, s2)


def test_extreme_rows(cuda):
    from mamba_int import ops
    w = torch.ones(768, device=cuda)
    x = torch.randn(6, 768, device=cuda)
    x[0] = 0.0                     # an all-zero row: eps alone in the root
    x[1, 5] = float("nan")
    x[2, 700] = float("inf")
    x[3] *= 1e-20                  # squares below the smallest float
    x[4] *= 1e15
    y, _ = ops.add_rms_norm(x, w, eps=EPS)
    q, scale, _ = ops.add_rms_norm_quant(x, w, eps=EPS)
    assert (y[0] == 0).all() and (q[0] == 0).all() and abs(scale[0].item() - 1e-8 / 127) < 1e-16
    assert torch.isnan(y[1]).all() and torch.isnan(scale[1])
    assert torch.isnan(y[2, 700]) and torch.isnan(scale[2])
    for i in (3, 4, 5):
        s, want, err = R.norm(x[i:i + 1].cpu(), None, w.cpu(), EPS)
        R.close(y[i:i + 1], want, err + 1e-40, torch.float32)
        check_quant(q[i:i + 1], scale[i:i + 1], want, 768)


def test_empty_and_stream(cuda):
    from mamba_int import ops
    w = torch.ones(64, device=cuda)
    y, res = ops.add_rms_norm(torch.empty(0, 64, device=cuda), w, residual=torch.empty(0, 64, device=cuda))
    assert y.shape == (0, 64) and res.shape == (0, 64)
    side = torch.cuda.Stream()
    x = torch.randn(64, 64, device=cuda)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, _ = ops.add_rms_norm(x, w)
    side.synchronize()
    s, want, err = R.norm(x.cpu(), None, w.cpu(), 1e-5)
    R.close(y, want, err, torch.float32)
