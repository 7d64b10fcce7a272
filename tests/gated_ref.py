"""The gated recurrence and its gradients from their formulas in 64 bits on the CPU, with a
bound of the error that 32-bit arithmetic may leave (tests/test_gpu_gated*.py).

U is the unit roundoff of float32.  Relative errors, counted from the roundings: an
exponential carries its argument's |p| U times two (the argument is rounded, and so is its
product with log2 e) and 3 U, a reciprocal or root 2 U more; k = rate softplus(decay) 8 U.  A
difference 1 - q has the absolute error of q and U.  A value that goes through t steps of the
recurrence meets the decays' errors of those steps, whatever blocks the steps are summed in,
so magnitudes are bounded by the recurrence of |b| (M below) and of |dh| (G)."""
import torch

from float_ref import U

TINY = 2.0 ** -118      # what hardware exponentials may flush


def sigmoid(v):
    """(sigmoid(v), its relative error)."""
    s = torch.sigmoid(v)
    return s, U * ((2 * v.abs() + 3) * (1 - s) + 4)


def gated(x, r, i, decay, z=None, rate=8.0, h_in=None, lens=None, dy=None):
    """{name: (value, error)} of y, h and, with dy, the gradients of the inputs."""
    B, L, D = x.shape
    x, r, i, decay = x.double(), r.double(), i.double(), decay.double()
    on = torch.ones(B, L, 1, dtype=torch.bool) if lens is None else (torch.arange(L) < lens.clamp(0, L).unsqueeze(1)).unsqueeze(-1)

    def keep(v):
        return torch.where(on, v, 0.0)

    soft = torch.logaddexp(decay, torch.zeros_like(decay))
    s, es = sigmoid(r)
    q, eq = sigmoid(i)
    n = rate * soft * s
    en = es + 9 * U
    a, ea = torch.exp(-n), n * (en + 2 * U) + 4 * U
    m = torch.sqrt(-torch.expm1(-2 * n))
    em = en / 2 + 8 * U
    b, eb = m * q * x, em + eq + 3 * U
    a, ea, b, eb = torch.where(on, a, 1.0), keep(ea), keep(b), keep(eb)
    h = torch.zeros(B, L + 1, D, dtype=torch.float64)
    M, eh = h.clone(), h.clone()
    if h_in is not None:
        h[:, 0], M[:, 0] = h_in.double(), h_in.double().abs()
    for t in range(L):
        h[:, t + 1] = a[:, t] * h[:, t] + b[:, t]
        M[:, t + 1] = a[:, t] * M[:, t] + b[:, t].abs()
        eh[:, t + 1] = (a[:, t] * eh[:, t] + (ea[:, t] + 4 * U) * a[:, t] * M[:, t] + eb[:, t] * b[:, t].abs() + 2 * U * M[:, t + 1]
                        + TINY * (1 + M[:, t]))
    act, eact, slope, eslope = torch.ones_like(x), torch.zeros_like(x), None, None
    if z is not None:
        z = z.double()
        g, eg = sigmoid(z)
        act, eact = z * g, (z * g).abs() * (eg + 2 * U) + TINY
        slope = g + act * (1 - g)
        eslope = g * eg + act.abs() * ((eg + 3 * U) * (1 - g) + g * eg + U) + U * slope.abs() + TINY
    out = {"y": (keep(h[:, 1:] * act), keep(eh[:, 1:] * act.abs() + M[:, 1:] * eact + 2 * U * M[:, 1:] * act.abs())),
           "h": (h[:, L], eh[:, L])}
    if dy is None:
        return out
    dy = keep(dy.double())
    dh, edh = dy * act, dy.abs() * (eact + U * act.abs())
    g = torch.zeros(B, L, D, dtype=torch.float64)
    G, eg = g.clone(), g.clone()
    c, C, ec = (torch.zeros(B, D, dtype=torch.float64) for _ in range(3))       # a g of the step after
    for t in range(L - 1, -1, -1):
        g[:, t], G[:, t] = dh[:, t] + c, dh[:, t].abs() + C
        eg[:, t] = edh[:, t] + ec + 2 * U * G[:, t]
        ec = a[:, t] * eg[:, t] + (ea[:, t] + 4 * U) * a[:, t] * G[:, t] + TINY * (1 + G[:, t])
        c, C = a[:, t] * g[:, t], a[:, t] * G[:, t]
    before, Mb, eb_ = h[:, :L], M[:, :L], eh[:, :L]
    ratio = torch.where(m > 0, n / torch.where(m > 0, m, 1.0), 0.0)
    t1 = q * x * a * a * ratio
    t2, T2 = n * a * before, n * a * Mb
    e1 = t1.abs() * (eq + 2 * ea + en + em + 8 * U)
    e2 = n * a * eb_ + T2 * (en + ea + 4 * U)
    p, P = g * (t1 - t2), G * (t1.abs() + T2)
    ep = eg * (t1.abs() + T2) + G * (e1 + e2) + 3 * U * P + TINY
    out["d_x"] = keep(g * m * q), keep(eg * m * q + G * m * q * (em + eq + 4 * U) + TINY)
    out["d_r"] = keep(p * (1 - s)), keep(ep * (1 - s) + P * (s * es + 2 * U))
    out["d_i"] = keep(g * b * (1 - q)), keep((eg * b.abs() + G * b.abs() * (eb + 3 * U)) * (1 - q) + G * b.abs() * (q * eq + U) + TINY)
    # sigmoid / softplus of decay: 16 U
    f = torch.where(decay < -30, torch.ones_like(decay), torch.sigmoid(decay) / torch.where(decay < -30, torch.ones_like(soft), soft))
    out["d_decay"] = keep(p).sum((0, 1)) * f, f * (keep(ep).sum((0, 1)) + (B * L + 20) * U * keep(P).sum((0, 1)))
    if z is not None:
        out["d_z"] = keep(dy * h[:, 1:] * slope), keep(dy.abs() * (eh[:, 1:] * slope.abs() + M[:, 1:] * (eslope + 3 * U * slope.abs())))
    if h_in is not None:
        out["d_h_in"] = c, ec
    return out
