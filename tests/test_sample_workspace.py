"""The workspace of token sampling grows with the slices of a call, not with the most there can be."""
import ctypes

import pytest

LIST, BINS = 8 * 8192, 2048


@pytest.mark.parametrize("rows,vocab", [(1, 32000), (64, 32000), (256, 32000), (64, 131072), (3, 40000), (1, 1 << 24), (256, 1 << 24)])
def test_bytes(rows, vocab):
    """A row's candidates and bins (counts and masses), two words a slice, a counter, and a slice's
    masses, rounded up to 256 bytes: slices of 8192 tokens and more, 64 at most, 512 in all rows."""
    from mamba_int import _lib
    n = ctypes.c_size_t(0)
    assert _lib.raw("mi_sample_workspace_size", rows, vocab, ctypes.byref(n)) == 0
    slices = min((vocab + 8191) // 8192, 64, 512 // rows)
    assert slices > 1 and n.value <= rows * (LIST + 12 * BINS + 64 * 16 + 256 + slices * 8 * BINS)


def test_beside_the_logits():
    """A serving batch's workspace is no larger than twice its float32 logits."""
    from mamba_int import _lib
    n = ctypes.c_size_t(0)
    for rows, vocab in ((64, 32000), (256, 32000), (64, 131072), (8, 50257)):
        assert _lib.raw("mi_sample_workspace_size", rows, vocab, ctypes.byref(n)) == 0
        assert n.value <= 2 * 4 * rows * vocab
