"""Refusals of token sampling (no GPU: nothing is enqueued), and its oracle against brute force."""
import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

import sample_ref as R

A = ctypes.c_void_p(0x100000)     # never dereferenced: every call below fails validation
F, D = ctypes.c_float, ctypes.c_double


def sample(x=A, t=0, ld=8, scale=1.0, u=A, ta=1.0, pa=1.0, ma=0.0, ids=A, B=2, V=8, ws=None, wsb=0):
    return ("mi_sample_tokens", x, t, ld, D(scale), u, None, F(ta), None, 0, None, F(pa), None, F(ma), ids, None, B, V, ws, wsb, None)


@pytest.mark.parametrize("call,status,needle", [
    (sample(B=-1), 2, "negative"), (sample(B=1 << 22), 2, "rows"), (sample(V=0), 2, "vocab=0"), (sample(V=(1 << 24) + 1), 2, "vocab"),
    (sample(t=4), 4, "type"), (sample(t=-1), 4, "type"), (sample(ld=-8), 2, "stride"), (sample(scale=0.0), 4, "scale"),
    (sample(scale=math.nan), 4, "scale"), (sample(scale=math.inf), 4, "scale"), (sample(ta=math.nan), 4, "temperature"),
    (sample(pa=math.nan), 4, "top_p"), (sample(ma=math.nan), 4, "min_p"), (sample(x=None), 1, "required"),
    (sample(u=None), 1, "required"), (sample(ids=None), 1, "required"), (sample(V=40000), 4, "workspace"),
    (sample(V=40000, ws=A, wsb=99), 4, "workspace"), (sample(V=40000, ws=ctypes.c_void_p(0x100004), wsb=1 << 30), 3, "aligned")])
def test_argument_validation(call, status, needle):
    from mamba_int import _lib
    assert _lib.raw(*call) == status and needle in _lib.last_error()


def test_no_rows_is_a_noop():
    from mamba_int import _lib
    assert _lib.raw(*sample(B=0, x=None, u=None, ids=None)) == 0


def test_workspace_size():
    from mamba_int import _lib
    n = ctypes.c_size_t(9)
    assert _lib.raw("mi_sample_workspace_size", 512, 100000, ctypes.byref(n)) == 0 and n.value == 0
    assert _lib.raw("mi_sample_workspace_size", 3, 1000, ctypes.byref(n)) == 0 and n.value == 0
    assert _lib.raw("mi_sample_workspace_size", 3, 100000, ctypes.byref(n)) == 0 and n.value > 0
    assert _lib.raw("mi_sample_workspace_size", 3, 0, ctypes.byref(n)) == 2
    assert _lib.raw("mi_sample_workspace_size", -3, 8, ctypes.byref(n)) == 2
    assert _lib.raw("mi_sample_workspace_size", 3, 8, None) == 1


def test_integers_stay_out_of_the_other_operators():
    from mamba_int import ops
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.add_rms_norm(torch.zeros(2, 8, dtype=torch.int32), torch.zeros(8))


def test_host_tensors_and_wrong_shapes_are_refused():
    from mamba_int import ops
    x, u = torch.zeros(2, 8), torch.zeros(2)
    with pytest.raises(ValueError, match="device"):
        ops.sample_tokens(x, u)
    with pytest.raises(ValueError, match="rows, vocab"):
        ops.sample_tokens(x[0], u)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.sample_tokens(x.double(), u)
    with pytest.raises(RuntimeError, match="ambiguous"):
        ops.sample_tokens(x, u, logprob=torch.ones(2))


def test_oracle_against_fractions():
    """Masses that are whole numbers: exp(l) is one where l is a logarithm of it (rounded once)."""
    rng = np.random.default_rng(0)
    for _ in range(300):
        mass = [int(v) for v in rng.integers(0, 6, size=7)]
        if not any(mass):
            continue
        k, p, q = int(rng.integers(0, 9)), float(rng.choice([1.0, 0.26, 0.51, 0.83])), float(rng.choice([0.0, 0.3, 0.7]))
        u = (int(rng.integers(0, 997)) + 0.5) / 997
        order = sorted((i for i in range(7) if mass[i]), key=lambda i: (-mass[i], i))
        if 0 < k < 7:
            order = order[:k]
        total, kept, before = sum(mass[i] for i in order), [], 0
        for i in order:
            if kept and (p < 1 and Fraction(before) >= Fraction(p) * total or Fraction(mass[i], mass[order[0]]) < Fraction(q)):
                break
            kept.append(i)
            before += mass[i]
        kept.sort()
        total, run = sum(mass[i] for i in kept), 0
        for i in kept:
            run += mass[i]
            if run > Fraction(u) * total:
                break
        token, prob, border = R.draw([math.log(v) if v else -math.inf for v in mass], u, top_k=k, top_p=p, min_p=q)
        assert border > 1e-9 and token == i and abs(prob - mass[i] / total) < 1e-12
