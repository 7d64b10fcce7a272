"""The element types' codes of the Python binding are those of the header."""
import os
import re

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_codes():
    from mamba_int import _lib
    with open(os.path.join(REPO, "include", "mamba_int.h")) as f:
        body = re.search(r"typedef enum \{([^}]*)\} mi_dtype;", f.read()).group(1)
    codes = {n: int(v) for n, v in re.findall(r"MI_(\w+) = (\d+)", body)}
    assert set(codes) == {"F32", "BF16", "F16", "I32", "I8"}
    ours = {n: getattr(_lib, n if n[0] != "I" else "TYPE_" + n) for n in codes}
    assert ours == codes
