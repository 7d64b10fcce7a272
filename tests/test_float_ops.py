"""Refusals of the float operators (no GPU: nothing is enqueued), and the 64-bit oracle of
their tests against brute force."""
import ctypes
import math

import pytest
import torch

import float_ref as R

A = ctypes.c_void_p(0x100000)     # never dereferenced: every call below fails validation
X = ctypes.c_void_p(0x100004)     # not 16-byte aligned
Z = ctypes.c_float(1e-5)


def norm(x=A, xt=0, ldx=8, res=None, rt=0, ldr=8, w=A, eps=Z, y=A, ldy=8, q=None, ldq=0, scale=None, ro=None, ldro=8, T=2,
         d=8):
    return ("mi_add_rms_norm", x, xt, ldx, res, rt, ldr, w, eps, y, ldy, q, ldq, scale, ro, ldro, T, d, None)


def conv(x=A, ldx=8, bsx=0, t=0, w=A, bias=None, width=4, silu=1, si=None, so=None, lens=None, y=A, ldy=8, bsy=0, B=1, L=4,
         D=8):
    return ("mi_causal_conv", x, ldx, bsx, t, w, bias, width, silu, si, so, lens, y, ldy, bsy, B, L, D, None)


def scan(u=A, ld=8, a=A, ldz=0, hin=None, lens=None, y=A, ldy=8, t=0, B=1, L=4, D=8, N=16, G=1, ws=None, wsb=0):
    return ("mi_selective_scan", u, ld, 0, A, 8, 0, a, A, 16, 0, A, 16, 0, None, None, ldz, 0, None, 1, hin, None, lens, y,
            ldy, 0, t, B, L, D, N, G, ws, wsb, None)


def w4(x=A, ldx=128, t=0, p=A, s=A, st=2, z=None, bias=None, y=A, ldy=16, m=1, n=16, k=128, g=128):
    return ("mi_w4_matvec", x, ldx, t, p, s, st, z, bias, y, ldy, m, n, k, g, None)


def pack(c=A, s=A, st=2, z=None, p=A, so=A, zo=None, n=16, k=128, g=128):
    return ("mi_pack_w4", c, s, st, z, p, so, zo, n, k, g, None)


@pytest.mark.parametrize("call,status,needle", [
    (norm(T=-1), 2, "tokens"), (norm(d=0), 2, "dim=0"), (norm(d=16385), 2, "16384"), (norm(xt=3), 4, "type"),
    (norm(xt=0, rt=1), 4, "residual"), (norm(xt=1, rt=2), 4, "residual"), (norm(eps=ctypes.c_float(-1)), 4, "eps"),
    (norm(eps=ctypes.c_float(math.nan)), 4, "eps"), (norm(ldy=7), 2, "stride"), (norm(ldx=-1), 2, "stride"),
    (norm(ro=A, ldro=7), 2, "stride"), (norm(q=A, ldq=7, scale=A), 2, "ldq"), (norm(q=A, ldq=8), 1, "scale"),
    (norm(y=None), 1, "required"), (norm(x=None), 1, "required"), (norm(T=1 << 22), 2, "tokens"),
    (conv(B=-1), 2, "negative"), (conv(width=0), 4, "width"), (conv(width=9), 4, "width"), (conv(t=5), 4, "type"),
    (conv(ldy=7), 2, "ldy"), (conv(bsx=-8), 2, "stride"), (conv(x=None), 1, "required"), (conv(w=None), 1, "required"),
    (conv(B=1 << 20, D=1 << 11, ldx=1 << 11, ldy=1 << 11), 2, "2^31"),
    (conv(L=(1 << 30) + 1), 2, "2^30"), (scan(L=(1 << 30) + 1), 2, "2^30"), (scan(D=1 << 18, G=1 << 18, N=256, ld=1 << 18, ldy=1 << 18), 2, "groups"),
    (w4(k=(1 << 30) + 1), 2, "2^30"), (pack(n=(1 << 28) + 1), 2, "2^28"), (scan(ld=1 << 26, L=64), 2, "row stride"),
    (scan(L=-1), 2, "negative"), (scan(N=0), 2, "nstate"), (scan(N=257), 2, "nstate"), (scan(G=3), 2, "groups"),
    (scan(G=0), 2, "groups"), (scan(t=-1), 4, "type"), (scan(ldy=4), 2, "ldy"), (scan(ldz=-1), 2, "stride"),
    (scan(B=1 << 23, D=8), 2, "2^25"), (scan(a=None), 1, "required"), (scan(u=None), 1, "required"),
    (w4(k=0), 2, "k=0"), (w4(g=48), 4, "group"), (w4(g=192), 4, "group"), (w4(g=0), 4, "group"), (w4(g=-128), 4, "group"),
    (w4(t=7), 4, "type"), (w4(st=1), 4, "scales"), (w4(ldy=15), 2, "ldy"), (w4(p=X), 3, "aligned"), (w4(p=None), 1, "required"),
    (w4(y=None), 1, "required"), (w4(m=1 << 20, n=1 << 11, ldy=1 << 11), 2, "2^31"), (w4(n=(1 << 28) + 1, ldy=1 << 30), 2, "2^28"),
    (w4(m=32 * 65535 + 1), 2, "65535"),
    (pack(n=-1), 2, "negative"), (pack(g=16), 4, "group"), (pack(st=1), 4, "scales"), (pack(c=None), 1, "required"),
    (pack(z=A), 1, "zeros"), (pack(p=X), 3, "aligned"),
])
def test_argument_validation(call, status, needle):
    from mamba_int import _lib
    st = _lib.raw(*call)
    assert st == status, (_lib.last_error(), st)
    assert needle in _lib.last_error()


def test_zero_sizes_are_noops():
    from mamba_int import _lib
    for call in (norm(T=0, x=None, w=None, y=None), conv(B=0, x=None, w=None, y=None), scan(B=0, u=None, a=None, y=None),
                 w4(m=0, x=None, y=None), w4(n=0, p=None), pack(n=0, c=None)):
        assert _lib.raw(*call) == 0, _lib.last_error()


def test_workspace_size():
    from mamba_int import _lib
    n = ctypes.c_size_t(99)
    assert _lib.raw("mi_selective_scan_workspace_size", 1, 1, 64, 16, 1, ctypes.byref(n)) == 0 and n.value == 0
    assert _lib.raw("mi_selective_scan_workspace_size", 1, 1, 64, 0, 1, ctypes.byref(n)) == 2
    assert _lib.raw("mi_selective_scan_workspace_size", 1, 1, 64, 16, 1, None) == 1
    # a call that needs a workspace is refused without one
    assert _lib.raw("mi_selective_scan_workspace_size", 1, 65536, 64, 16, 1, ctypes.byref(n)) == 0
    if n.value:
        assert _lib.raw(*scan(L=65536, D=64, ldy=64, ld=64)) == 4
        assert "workspace" in _lib.last_error()
        assert _lib.raw(*scan(L=65536, D=64, ldy=64, ld=64, ws=A, wsb=n.value - 1)) == 4


def test_host_tensors_and_wrong_types_are_refused():
    from mamba_int import ops
    x, w = torch.zeros(2, 8), torch.zeros(8)
    with pytest.raises(ValueError, match="device"):
        ops.add_rms_norm(x, w)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.add_rms_norm(x.double(), w)
    with pytest.raises(ValueError, match="tokens, dim"):
        ops.add_rms_norm_quant(x[0], w)
    with pytest.raises(TypeError, match="residual"):
        ops.add_rms_norm(x, w, residual=x.half())
    with pytest.raises(ValueError, match="unit"):
        ops.add_rms_norm_quant(x, w, unit=0)
    with pytest.raises(ValueError, match="batch, len, dim"):
        ops.causal_conv(x, torch.zeros(8, 4))
    with pytest.raises(ValueError, match="activation"):
        ops.causal_conv(x[None], torch.zeros(8, 4), activation="gelu")
    with pytest.raises(ValueError, match="weight"):
        ops.causal_conv(x[None], w)
    with pytest.raises(ValueError, match="device"):
        ops.causal_conv(x[None], torch.zeros(8, 4))
    with pytest.raises(ValueError, match="dim, states"):
        ops.selective_scan(x[None], x[None], w, x[None], x[None])
    with pytest.raises(ValueError, match="b must be"):
        ops.selective_scan(x[None], x[None], torch.zeros(8, 4), torch.zeros(1, 2, 1, 5), torch.zeros(1, 2, 4))
    with pytest.raises(TypeError, match="torch.Tensor"):
        ops.causal_conv([1.0], torch.zeros(8, 4))
    with pytest.raises(TypeError, match="scales"):
        ops.w4_matvec(x, None, w.double(), 4, 32)
    with pytest.raises(ValueError, match="group"):
        ops.w4_matvec(x, None, w, 4, 48)
    with pytest.raises(ValueError, match="device"):
        ops.pack_w4(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2), 32)


def test_oracle_against_brute_force():
    g = torch.Generator().manual_seed(0)
    u, dt, z = (torch.randn(2, 5, 6, generator=g, dtype=torch.float64) for _ in range(3))
    b, c = (torch.randn(2, 5, 2, 3, generator=g, dtype=torch.float64) for _ in range(2))
    a = -torch.rand(6, 3, generator=g, dtype=torch.float64)
    skip, bias = torch.randn(6, generator=g).double(), torch.randn(6, generator=g).double()
    h0 = torch.randn(2, 6, 3, generator=g).double()
    lens = torch.tensor([5, 3])
    y, _, h, _ = R.scan(u, dt, a, b, c, skip, z, bias, True, h0, lens)
    for i in range(2):
        for ch in range(6):
            st = [float(v) for v in h0[i, ch]]
            for t in range(5):
                if t >= lens[i]:
                    assert y[i, t, ch] == 0
                    continue
                d = math.log1p(math.exp(float(dt[i, t, ch] + bias[ch])))
                out = float(skip[ch] * u[i, t, ch])
                for n in range(3):
                    st[n] = math.exp(d * float(a[ch, n])) * st[n] + d * float(u[i, t, ch] * b[i, t, ch // 3, n])
                    out += float(c[i, t, ch // 3, n]) * st[n]
                zz = float(z[i, t, ch])
                assert abs(float(y[i, t, ch]) - out * zz / (1 + math.exp(-zz))) < 1e-12
            assert all(abs(float(h[i, ch, n]) - st[n]) < 1e-12 for n in range(3))
    x = torch.randn(1, 4, 3, generator=g)
    w = torch.randn(3, 2, generator=g)
    st = torch.randn(1, 1, 3, generator=g)
    y, _, last = R.conv(x, w, None, False, st, None)
    for t in range(4):
        for ch in range(3):
            prev = st[0, 0, ch] if t == 0 else x[0, t - 1, ch]
            assert abs(float(y[0, t, ch]) - (float(w[ch, 0]) * float(prev) + float(w[ch, 1]) * float(x[0, t, ch]))) < 1e-12
    assert torch.equal(last[:, 0], x[:, 3])
    codes = torch.randint(0, 16, (3, 70), generator=g, dtype=torch.uint8)
    sc, ze = torch.rand(3, 3, generator=g), torch.randint(0, 16, (3, 3), generator=g, dtype=torch.uint8)
    xr = torch.randn(2, 70, generator=g)
    y, _ = R.w4(xr, codes, sc, ze, 32, None)
    want = sum(float(xr[1, k]) * (int(codes[2, k]) - int(ze[2, k // 32])) * float(sc[2, k // 32]) for k in range(70))
    assert abs(float(y[1, 2]) - want) < 1e-9
