"""Every global and LDS address of the float operators' kernels, on the CPU.

The kernel sources are compiled for the host (tests/host_float on top of
tests/host_kernels: threads run one after another, AddressSanitizer watches buffers of
exactly the described extents and every LDS array) and called over random sizes,
strides, offsets and small devices' dispatch.  No kernel's addresses depend on data
beyond lengths, which are clamped, so a clean run covers the GPU's accesses at these
sizes."""
import concurrent.futures
import os
import re
import subprocess

import pytest

from test_host_addresses import _clang, _host_source

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(REPO, "mamba-integer_amd", "csrc")
HOST = os.path.join(HERE, "host_float")
UNITS = ["common", "norm", "conv", "selective_scan", "w4"]

_QUAD = "for (int i = 0; i < 4; ++i) { p[i] = a[i] * next; x[i] += e[i] * h[i]; y += c * x[i]; }"


def _source(text):
    return _host_source(re.sub(r'asm\("v_mul_f32 %0.*?\)\);', _QUAD, text, flags=re.S))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    clang = _clang()
    if clang is None:
        pytest.skip("no clang++")
    tmp = tmp_path_factory.mktemp("host_float")
    for f in ["mi_common.hpp", "float_ops.hpp"] + [u + ".hip" for u in UNITS]:
        with open(os.path.join(CSRC, f)) as src, open(tmp / f.replace(".hip", ".cpp"), "w") as dst:
            dst.write(_source(src.read()))
    flags = ["-std=c++17", "-O1", "-g", "-w", "-fno-strict-aliasing", "-fsanitize=address", f"-I{HOST}", f"-I{tmp}",
             f"-I{os.path.join(REPO, 'include')}"]

    def compile_one(src):
        out = subprocess.run([clang, *flags, "-c", str(src), "-o", str(tmp / (os.path.basename(src)[:-4] + ".o"))],
                             capture_output=True, text=True)
        assert out.returncode == 0, out.stderr[:3000]

    sources = [tmp / (u + ".cpp") for u in UNITS] + [os.path.join(HOST, "addresses.cpp")]
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(6, os.cpu_count() or 1)) as pool:
        list(pool.map(compile_one, sources))
    exe = tmp / "addresses_exe"
    out = subprocess.run([clang, "-fsanitize=address", *[str(tmp / (u + ".o")) for u in UNITS + ["addresses"]], "-o", str(exe)],
                         capture_output=True, text=True)
    assert out.returncode == 0, out.stderr[:3000]
    return str(exe)


@pytest.mark.parametrize("family,count", [("norm", 100), ("conv", 150), ("scan", 60), ("w4", 60), ("limits", 0)])
def test_addresses_in_bounds(program, family, count):
    out = subprocess.run([program, family, str(count), "1"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, (out.stdout + out.stderr)[-6000:]
