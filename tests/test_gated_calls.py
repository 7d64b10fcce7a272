"""Refusals of the gated recurrence and of adapters (no GPU: nothing is enqueued), and the
recurrence's oracle against autograd and differences."""
import ctypes
import math

import pytest
import torch

import gated_ref as G

A = ctypes.c_void_p(0x100000)     # never dereferenced: every call below fails validation
X = ctypes.c_void_p(0x100004)     # not 16-byte aligned
F = ctypes.c_float


def scan(x=A, ld=8, decay=A, rate=8.0, ldz=0, y=A, ldy=8, t=0, B=1, L=4, D=8, ws=None, wsb=0):
    return ("mi_gated_scan", x, ld, 0, A, 8, 0, A, 8, 0, decay, F(rate), None, ldz, 0, None, None, None, y, ldy, 0, None, t, B, L,
            D, ws, wsb, None)


def back(dy=A, ldy=8, saved=A, rate=8.0, dz=None, t=0, B=1, L=4, D=8, ws=A, wsb=1 << 20, decay=A):
    return ("mi_gated_scan_backward", dy, ldy, 0, A, 8, 0, A, 8, 0, A, 8, 0, decay, F(rate), None, 0, 0, None, saved, A, A, A, dz,
            A, A, t, B, L, D, ws, wsb, None)


def adapter(x=A, xt=0, ldx=8, xs=None, a=A, wt=0, ids=A, y=A, ldy=8, out=X, ldo=8, t=0, B=1, L=4, K=8, N=8, R=4, bank=2, ws=A,
            wsb=1 << 20):
    return ("mi_adapter_add", x, xt, ldx, 0, xs, a, A, wt, None, ids, None, y, ldy, 0, out, ldo, 0, t, B, L, K, N, R, bank, ws, wsb,
            None)


@pytest.mark.parametrize("call,status,needle", [
    (scan(B=-1), 2, "negative"), (scan(B=65536), 2, "65535"), (scan(D=(1 << 24) + 1), 2, "2^24"), (scan(L=(1 << 30) + 1), 2, "2^30"),
    (scan(t=3), 4, "type"), (scan(rate=-1.0), 4, "rate"), (scan(rate=math.nan), 4, "rate"), (scan(ld=-1), 2, "stride"),
    (scan(ldz=-1), 2, "stride"), (scan(ldy=7), 2, "ldy"), (scan(x=None), 1, "required"), (scan(decay=None), 1, "required"),
    (scan(y=None), 1, "required"),
    (back(L=-1), 2, "negative"), (back(t=4), 4, "type"), (back(rate=math.inf), 4, "rate"), (back(ldy=-1), 2, "stride"),
    (back(dz=A), 4, "dz"), (back(dy=None), 1, "required"), (back(saved=None), 1, "required"), (back(decay=None), 1, "required"),
    (back(ws=None), 4, "workspace"), (back(wsb=1), 4, "workspace"), (back(ws=X), 3, "aligned"),
    (adapter(B=-1), 2, "negative"), (adapter(K=(1 << 23) + 1), 2, "8388608"), (adapter(N=(1 << 23) + 1, ldo=1 << 24), 2, "8388608"),
    (adapter(R=129), 2, "rank=129"), (adapter(bank=-1), 2, "bank"), (adapter(B=1 << 12, L=1 << 10), 2, "batch * len"),
    (adapter(t=3), 4, "type"), (adapter(wt=4), 4, "type"), (adapter(xt=1), 4, "type"), (adapter(xt=4), 4, "x_scale"),
    (adapter(xs=A), 4, "x_scale"), (adapter(ldx=-1), 2, "stride"), (adapter(ldo=7), 2, "ldo"), (adapter(ids=None), 1, "required"),
    (adapter(y=None), 1, "required"), (adapter(x=None), 1, "required"), (adapter(a=None), 1, "required"),
    (adapter(out=A, ldy=9), 4, "strides"), (adapter(ws=None), 4, "workspace"), (adapter(wsb=8), 4, "workspace"),
    (adapter(ws=X), 3, "aligned")])
def test_argument_validation(call, status, needle):
    from mamba_int import _lib
    assert _lib.raw(*call) == status and needle in _lib.last_error(), _lib.last_error()


def test_zero_sizes_are_noops():
    from mamba_int import _lib
    for call in (scan(B=0, x=None, decay=None, y=None), scan(D=0, x=None, decay=None, y=None, ld=0, ldy=0), back(D=0, decay=None),
                 adapter(B=0, x=None, ids=None), adapter(N=0, y=None), adapter(out=A, R=0, x=None, ws=None)):
        assert _lib.raw(*call) == 0, _lib.last_error()


def test_sizes():
    from mamba_int import _lib
    n = [ctypes.c_size_t(9) for _ in range(3)]
    p = [ctypes.byref(v) for v in n]
    assert _lib.raw("mi_gated_scan_sizes", 2, 0, 8, *p) == 0 and n[2].value == 0
    assert _lib.raw("mi_gated_scan_sizes", 2, 1, 8, *p) == 0 and n[2].value >= 64
    assert _lib.raw("mi_gated_scan_sizes", -2, 1, 8, *p) == 2
    assert _lib.raw("mi_gated_scan_sizes", 2, 1, 8, None, p[1], p[2]) == 1
    assert _lib.raw("mi_adapter_workspace_size", 2, 3, 5, p[0]) == 0 and n[0].value >= 120
    assert _lib.raw("mi_adapter_workspace_size", 2, 3, 200, p[0]) == 2
    assert _lib.raw("mi_adapter_workspace_size", 2, 3, 5, None) == 1


def test_host_tensors_and_wrong_shapes_are_refused():
    from mamba_int import ops
    x, k = torch.zeros(2, 3, 8), torch.zeros(8)
    with pytest.raises(ValueError, match="device"):
        ops.gated_scan(x, x, x, k)
    with pytest.raises(ValueError, match="batch, len, dim"):
        ops.gated_scan(x[0], x, x, k)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.gated_scan(x.double(), x, x, k)
    with pytest.raises(ValueError, match="device"):
        ops.gated_scan(x.requires_grad_(), x, x, k)
    a, b, ids = torch.zeros(2, 4, 8), torch.zeros(2, 8, 4), torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 3, 8)
    with pytest.raises(ValueError, match="device"):
        ops.adapter_add(x, x, a, b, ids)
    with pytest.raises(ValueError, match="bank, rank, k"):
        ops.adapter_add(x, x, a[0], b, ids)
    with pytest.raises(ValueError, match="dimensions"):
        ops.adapter_add(x, x[0], a, b, ids)
    with pytest.raises(TypeError, match="torch.Tensor"):
        ops.adapter_add(x, x, a, None, ids)


@pytest.mark.parametrize("gate,state,lens", [(True, True, True), (False, False, False)])
def test_oracle(gate, state, lens):
    """Values against the recurrence step by step, gradients against autograd's and central differences."""
    g = torch.Generator().manual_seed(3)
    B, L, D = 3, 6, 4
    v = {n: torch.randn(B, L, D, generator=g, dtype=torch.float64) for n in ("x", "r", "i")}
    v["decay"] = torch.randn(D, generator=g, dtype=torch.float64)
    if gate:
        v["z"] = torch.randn(B, L, D, generator=g, dtype=torch.float64)
    if state:
        v["h_in"] = torch.randn(B, D, generator=g, dtype=torch.float64)
    n = torch.tensor([L, 3, 0]) if lens else torch.tensor([L] * B)
    dy = torch.randn(B, L, D, generator=g, dtype=torch.float64)

    def f(v):
        out = []
        for b in range(B):
            h = v["h_in"][b] if state else torch.zeros(D, dtype=torch.float64)
            for t in range(L):
                if t >= n[b]:
                    out.append(torch.zeros(D, dtype=torch.float64))
                    continue
                a = torch.exp(-8.0 * torch.log1p(torch.exp(v["decay"])) * torch.sigmoid(v["r"][b, t]))
                h = a * h + torch.sqrt(1 - a * a) * torch.sigmoid(v["i"][b, t]) * v["x"][b, t]
                out.append(h * v["z"][b, t] * torch.sigmoid(v["z"][b, t]) if gate else h)
        return torch.stack(out).view(B, L, D)

    leaf = {k: t.clone().requires_grad_() for k, t in v.items()}
    y = f(leaf)
    grads = dict(zip(leaf, torch.autograd.grad(y, list(leaf.values()), dy)))
    got = G.gated(v["x"], v["r"], v["i"], v["decay"], v.get("z"), h_in=v.get("h_in"), lens=n if lens else None, dy=dy)
    assert (got["y"][0] - y).abs().max() < 1e-12
    for k, w in grads.items():
        assert (got["d_" + k][0] - w).abs().max() < 1e-11, k
        assert (got["d_" + k][1] >= 0).all() and got["d_" + k][1].max() < 1e-4
        d = torch.randn(v[k].shape, generator=g, dtype=torch.float64)
        up, down = f(dict(v, **{k: v[k] + 1e-5 * d})), f(dict(v, **{k: v[k] - 1e-5 * d}))
        assert abs(float(((up - down) * dy).sum() / 2e-5) - float((w * d).sum())) < 1e-7
