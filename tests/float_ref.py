"""The float operators from their formulas in 64 bits on the CPU, with a bound of
the error that 32-bit arithmetic may leave (tests/test_gpu_float_*.py).

U is the unit roundoff of float32 (2^-24); UNIT that of each output type.  A
bound counts roundings: each operation adds U of its result, hardware
exponentials, logarithms and reciprocals two of them, and exp(p) carries its
argument's error |p| U on top."""
import torch

U = 2.0 ** -24
UNIT = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -14}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def close(got, want, err, dtype):
    """got (dtype) is want within err and one rounding to dtype (half a subnormal's step near 0)."""
    assert got.dtype == dtype and tuple(got.shape) == tuple(want.shape)
    got = got.double().cpu()
    far = (got - want).abs()
    tol = err + UNIT[dtype] * (want.abs() + err) + TINY[dtype] * UNIT[dtype]
    bad = ~(far <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, the worst by "
                           f"{float((far / tol)[bad].max()):.3g} of its tolerance, first at {bad.nonzero()[0].tolist()}")


def silu(v):
    """(v * sigmoid(v), the error of evaluating it in 32 bits): e = exp(-v) carries (2|v| + 3) U,
    1 / (1 + e) at most that times e / (1 + e), and 4 U more; values below 2^-120 may be flushed."""
    s = torch.sigmoid(v)
    y = v * s
    return y, y.abs() * U * (6 + (2 * v.abs() + 3) * (1 - s)) + 2.0 ** -118


def norm(x, residual, w, eps):
    """(s, y, error of y): a tree sum of the squares of at most 64 a thread, root, reciprocal, two products."""
    s = x.double()
    if residual is not None:
        s = s + residual.double()
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * w.double()
    return s, y, 48 * U * y.abs()


def conv(x, w, bias, act, state_in, lens):
    """(y, error, state_out in x's type)."""
    B, L, D = x.shape
    W = w.shape[1]
    y, err = torch.zeros(B, L, D, dtype=torch.float64), torch.zeros(B, L, D, dtype=torch.float64)
    state = torch.zeros(B, W - 1, D, dtype=x.dtype)
    wd = w.double()
    for b in range(B):
        n = L if lens is None else min(max(int(lens[b]), 0), L)
        first = state_in[b] if state_in is not None else torch.zeros(W - 1, D, dtype=x.dtype)
        rows = torch.cat([first, x[b, :n]])
        state[b] = rows[n:]
        r = rows.double()
        v, mag = torch.zeros(n, D, dtype=torch.float64), torch.zeros(n, D, dtype=torch.float64)
        if bias is not None:
            v, mag = v + bias.double(), mag + bias.double().abs()
        for j in range(W):
            v = v + wd[:, j] * r[j:j + n]
            mag = mag + (wd[:, j] * r[j:j + n]).abs()
        e = (W + 1) * U * mag
        if act:
            s, es = silu(v)
            v, e = s, es + 1.1 * e          # |d silu| < 1.1
        y[b, :n], err[b, :n] = v, e
    return y, err, state


def softplus(v):
    return torch.logaddexp(v, torch.zeros_like(v))


def scan(u, dt, a, b, c, d_skip=None, z=None, dt_bias=None, sp=True, h_in=None, lens=None, masked=()):
    """(y, error of y, h, error of h) of the selective scan; b, c [B, L, G, N]."""
    B, L, D = u.shape
    G, N = b.shape[2:]
    a = a.double()
    h = h_in.double().clone() if h_in is not None else torch.zeros(B, D, N, dtype=torch.float64)
    eh = torch.zeros_like(h)
    y, ey = torch.zeros(B, L, D, dtype=torch.float64), torch.zeros(B, L, D, dtype=torch.float64)
    zero = torch.zeros(D, dtype=torch.float64)
    bias = dt_bias.double() if dt_bias is not None else zero
    skip = d_skip.double() if d_skip is not None else zero
    for t in range(L):
        on = torch.ones(B, dtype=torch.bool) if lens is None else lens > t
        raw = dt[:, t].double() + bias
        d = softplus(raw) if sp else raw
        # the sum's rounding moves softplus by at most |raw| U (its slope is at most 1, and at most itself)
        ed = U * (torch.minimum(torch.ones_like(d), d.abs()) * raw.abs() + 12 * d.abs()) if sp else U * raw.abs()
        ut = u[:, t].double()
        bt = b[:, t].double().repeat_interleave(D // G, 1)
        ct = c[:, t].double().repeat_interleave(D // G, 1)
        p = d[..., None] * a
        e = torch.exp(p)
        x = (d * ut)[..., None] * bt
        ep = ed[..., None] * a.abs() + 4 * U * p.abs()
        new = e * h + x
        enew = e * eh + (e * h).abs() * (ep + 4 * U) + x.abs() * 4 * U + (ed * ut.abs())[..., None] * bt.abs() + U * new.abs()
        out = (new * ct).sum(-1) + skip * ut
        eo = (ct.abs() * enew).sum(-1) + (N + 3) * U * ((new * ct).abs().sum(-1) + (skip * ut).abs())
        if z is not None:
            g, eg = silu(z[:, t].double())
            out, eo = out * g, eo * g.abs() + out.abs() * eg + 2 * U * (out * g).abs()
        h, eh = torch.where(on[:, None, None], new, h), torch.where(on[:, None, None], enew, eh)
        y[:, t], ey[:, t] = torch.where(on[:, None], out, 0.0), torch.where(on[:, None], eo, 0.0)
    return y, ey, h, eh


def w4(x, codes, scales, zeros, group, bias):
    """(y, error): a sum of k products in any order, each with its weight and its zero point offset by 16."""
    n, k = codes.shape
    s = scales.double().repeat_interleave(group, 1)[:, :k]
    z = zeros.double().repeat_interleave(group, 1)[:, :k] if zeros is not None else 8.0
    w = (codes.double() - z) * s
    y = x.double() @ w.t()
    err = (k + 8) * U * (x.double().abs() @ ((codes.double() + 48.0) * s.abs()).t())
    if bias is not None:
        y = y + bias.double()
        err = err + U * bias.double().abs()
    return y, err
