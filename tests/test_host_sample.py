"""Token sampling's kernels on the CPU, their results and every address.

The source is compiled for the host against tests/host_sample (a block's threads run in
turns and exchange values as the waves do, AddressSanitizer watches buffers of exactly the
documented extents and every LDS array), so what is drawn is what the kernels draw; the
definition (tests/sample_ref.py) says what it has to be."""
import os
import re
import struct
import subprocess

import numpy as np
import pytest

import sample_ref as R
from test_host_addresses import _clang, _host_source

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(REPO, "mamba-integer_amd", "csrc")
HOST = os.path.join(HERE, "host_sample")
LOWEST = -2 ** 31


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    clang = _clang()
    if clang is None:
        pytest.skip("no clang++")
    tmp = tmp_path_factory.mktemp("host_sample")
    for f in ("mi_common.hpp", "float_ops.hpp", "common.hip", "sample.hip"):
        with open(os.path.join(CSRC, f)) as src, open(tmp / f.replace(".hip", ".cpp"), "w") as dst:
            dst.write(re.sub("#pragma unroll.*", "", _host_source(src.read())))
    exe = tmp / "draw_exe"
    out = subprocess.run([clang, "-std=c++17", "-O1", "-w", "-fno-strict-aliasing", "-fsanitize=address", f"-I{HOST}", f"-I{tmp}",
                          f"-I{os.path.join(REPO, 'include')}", str(tmp / "common.cpp"), str(tmp / "sample.cpp"),
                          os.path.join(HOST, "draw.cpp"), "-o", str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr[:3000]
    return str(exe)


def draw(program, tmp_path, cases):
    """[(ids, logprob)] of cases (logits float32 or int32 [B, V], u [B], parameters); a parameter
    is a number of every row or an array [B]."""
    with open(tmp_path / "cases", "wb") as f:
        for logits, u, par in cases:
            B, V = logits.shape
            values = [np.broadcast_to(np.asarray(par.get(n, d), np.int32 if n == "top_k" else np.float32), (B,))
                      for n, d in (("temperature", 1.0), ("top_p", 1.0), ("min_p", 0.0), ("top_k", 0))]
            every = all(np.ndim(par.get(n, 0)) == 0 for n in ("temperature", "top_p", "min_p", "top_k"))
            f.write(struct.pack("iiiid", 3 if logits.dtype == np.int32 else 0, B, V, every, par.get("scale", 1.0)))
            for v in (np.asarray(u, np.float32), *values, logits):
                f.write(np.ascontiguousarray(v).tobytes())
    out = subprocess.run([program, str(tmp_path / "cases"), str(tmp_path / "results")], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0, (out.stdout + out.stderr)[-4000:]
    got = []
    with open(tmp_path / "results", "rb") as f:
        for logits, _, _ in cases:
            B = logits.shape[0]
            got.append((np.frombuffer(f.read(8 * B), np.int64), np.frombuffer(f.read(4 * B), np.float32)))
    return got


def check(program, tmp_path, cases):
    """Tokens are equal where u and top_p's cut are no nearer to a border than 2^-29 of the mass
    (as in tests/test_gpu_sample.py, whose arithmetic this is), log probabilities 2^-28."""
    for (logits, u, par), (ids, lp) in zip(cases, draw(program, tmp_path, cases)):
        for b in range(logits.shape[0]):
            row = {n: (v[b] if np.ndim(v) else v) for n, v in par.items()}
            row = {n: int(v) if n == "top_k" else v if n == "scale" else np.float32(v).item() for n, v in row.items()}
            token, p, border = R.draw(logits[b], np.float32(u[b]).item(), **row)
            if border < 2.0 ** -29 and len(set(logits[b].tolist())) > 8:
                continue
            want = np.log(p) if token >= 0 else -np.inf
            assert ids[b] == token, (logits.shape, row, b, ids[b], token, border)
            assert lp[b] == want or abs(lp[b] - want) <= 2.0 ** -28 + 2.0 ** -24 * abs(want), (logits.shape, row, b, lp[b], want)


U = [0.0, 0.31, 0.77, 0.9999]


@pytest.mark.parametrize("V", [2048, 9001])
@pytest.mark.parametrize("par", [dict(top_k=1500), dict(top_k=2040), dict(top_p=0.9), dict(top_k=1900, top_p=0.95)])
def test_two_values_a_whole_range_apart(program, tmp_path, V, par):
    """int32 logits of 0 and of the lowest value, alike at an infinite temperature: cuts in the
    part of the places that begins at 0."""
    logits = np.zeros((4, V), np.int32)
    logits[:, np.random.default_rng(V).permutation(V)[:V // 2]] = LOWEST
    check(program, tmp_path, [(logits, U, dict(par, temperature=float("inf")))])


@pytest.mark.parametrize("V", [5000, 20000])
@pytest.mark.parametrize("below", [1, 2, 10, 260, 2500, 4900])
def test_lowest_integers_next_to_each_other(program, tmp_path, V, below):
    """int32 logits from the lowest one up, nearly alike, cut by count and by mass `below` tokens
    before the order's end."""
    logits = (LOWEST + np.random.default_rng(below).integers(0, 5_000_000, (4, V))).astype(np.int32)
    check(program, tmp_path, [(logits, U, dict(scale=1e-12, top_k=V - below)),
                              (logits, U, dict(scale=1e-12, top_p=1 - (below + 0.5) / V))])


def mixed(B, seed):
    """Parameters of B rows: every kind of filter, none, and the first of the order, in turn."""
    g = np.random.default_rng(seed)
    kinds = [dict(), dict(temperature=0.0), dict(top_k=20), dict(top_k=700), dict(top_p=0.8), dict(top_k=3000, top_p=0.7), dict(min_p=0.05),
             dict(top_p=0.9, min_p=0.01), dict(top_k=40, top_p=0.9, min_p=0.02), dict(temperature=2.5, top_p=0.95), dict(top_k=1),
             dict(temperature=float("nan"))]
    rows = [kinds[(b + seed) % len(kinds)] for b in range(B)]
    par = {n: np.array([r.get(n, d) for r in rows], np.int32 if n == "top_k" else np.float32)
           for n, d in (("temperature", 1.0), ("top_p", 1.0), ("min_p", 0.0), ("top_k", 0))}
    return par, g


@pytest.mark.parametrize("V", [777, 9001, 20000])
@pytest.mark.parametrize("dtype", [np.float32, np.int32])
def test_rows_of_every_kind(program, tmp_path, V, dtype):
    par, g = mixed(12, V)
    logits = 2.0 * g.standard_normal((12, V)) - np.log1p(np.arange(V))[g.permutation(V)]
    if dtype == np.int32:
        logits, par = np.round(logits * 1024), dict(par, scale=1.0 / 1024)
    check(program, tmp_path, [(logits.astype(dtype), g.random(12).astype(np.float32), par)])


@pytest.mark.parametrize("V", [777, 9001, 20000])
@pytest.mark.parametrize("par", [dict(), dict(top_k=20), dict(top_p=0.8), dict(top_k=600, top_p=0.7, min_p=0.01), dict(temperature=0.0),
                                 dict(temperature=float("inf"))])
def test_masked_rows(program, tmp_path, V, par):
    """Rows, and whole slices of them, of -inf, NaN and the lowest value; infinities; u out of range."""
    g = np.random.default_rng(V)
    low, inf, nan = np.finfo(np.float32).min, np.inf, np.nan
    logits = g.standard_normal((10, V)).astype(np.float32)
    for b, v in enumerate((-inf, low, nan)):
        logits[b, : V - 300] = v
        logits[3 + b] = v
    logits[6, 100], logits[6, V - 5] = inf, inf
    logits[7], logits[7, V // 2] = -inf, low
    logits[8, ::2], logits[8, 1::2] = 0.0, -0.0
    u = np.array([0.3, 0.6, 0.9, 0.5, 0.5, 0.5, 0.75, 0.5, 0.4, 1.0], np.float32)
    check(program, tmp_path, [(logits, u, par)])
