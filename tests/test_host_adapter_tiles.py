"""Every global and LDS address of the adapters' kernels on the CPU, where a block takes 64 tokens (as
many CUs as blocks of them, or fewer) and where products come out as NaN."""
import os
import re
import subprocess

import pytest

from test_host_addresses import _clang, _host_source

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(REPO, "mamba-integer_amd", "csrc")
HOST = os.path.join(HERE, "host_adapter")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    clang = _clang()
    if clang is None:
        pytest.skip("no clang++")
    tmp = tmp_path_factory.mktemp("host_adapter")
    for f in ("mi_common.hpp", "float_ops.hpp", "common.hip", "adapter.hip"):
        with open(os.path.join(CSRC, f)) as src, open(tmp / f.replace(".hip", ".cpp"), "w") as dst:
            dst.write(re.sub("#pragma unroll.*", "", _host_source(src.read())))
    exe = tmp / "tiles_exe"
    out = subprocess.run([clang, "-std=c++17", "-O1", "-w", "-fno-strict-aliasing", "-fsanitize=address", f"-I{HOST}", f"-I{tmp}",
                          f"-I{os.path.join(REPO, 'include')}", str(tmp / "common.cpp"), str(tmp / "adapter.cpp"),
                          os.path.join(HOST, "tiles.cpp"), "-o", str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr[:3000]
    return str(exe)


@pytest.mark.parametrize("cus", [1, 3, 256])
def test_addresses_in_bounds(program, cus):
    out = subprocess.run([program, str(cus), "12", "1"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, (out.stdout + out.stderr)[-6000:]
