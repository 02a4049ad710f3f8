"""Which kernels calls of the vocabulary loss and the embedding launch, on the CPU."""
import re

import pytest

from launches import launched
from test_gpu_head import LARGE, LARGE_GRADS, LARGE_LOGITS, SIZES

_GRAD = """
def grad(n, vocab, columns=1, flags=0):
    ok(L.ark_embed_grad(A(1) if n else None, columns, 2, A(2) if n else None, 8, n, vocab, columns,
                        1.0, A(3), columns, flags, A(4), 1 << 40, None))
    return shown()
"""


@pytest.mark.parametrize("vocab", [1, 7, 1 << 27, (1 << 27) + 1, 1 << 28])
def test_a_gradient_of_no_tokens_reads_none(vocab):
    """Neither tokens nor rows are there to read: only zeros are written, into a table
    of any size."""
    rows = launched(_GRAD + f"out = grad(0, {vocab})\nassert not grad(0, {vocab}, flags=1)")
    assert len(rows) == 1 and "zero_kernel" in rows[0][0], rows
    assert rows[0][1] * rows[0][2] * rows[0][3] < 1 << 32


def test_gradients_of_some_tokens():
    few, large, many = launched(_GRAD + "out = [grad(1, 7), grad(3, 1 << 28), grad(513, 7)]")
    assert [("few_kernel" in r[0]) for r in few] == [True]
    for rows in (large, many):
        assert ["sort_kernel" in r[0] for r in rows] == [True] + [False] * (len(rows) - 1)
        assert "sum_kernel" in rows[-1][0]


_HEAD = """
def head(t, d, v, top=0):
    need = ctypes.c_uint64()
    ok(L.ark_head_workspace(A(2), d, t, d, v, top or 1, 2, 7, ctypes.byref(need)))
    x = (A(1), d, A(2), d, 0, t, d, v)
    y = (A(3), 8, top, A(4), 2, top, top, 1.0) if top else (A(3), 8, -100, 1.0)
    call = L.ark_head_distill_grad if top else L.ark_head_cross_entropy_grad
    ok(call(*x, *y, 1.0, None, A(5), A(6), d, A(7), 2, d, 0, A(8), need.value, None))
    return [r[0] for r in shown()]
"""


def _tiles(names, kernel):
    """A kernel's waves' fragments, [8, 4] or [4, 2]."""
    found = [re.search(r"7ProductI.*?Lj(\d+)ELj(\d+)E", n) for n in names if kernel in n]
    assert len(found) == 1, names
    return [int(f) for f in found[0].groups()]


def test_the_large_tiles_are_tested():
    """The sizes that the GPU tests name as large are those of the large tiles, for the
    logits, for the gradients, or for both; the others' are not."""
    large, small = [8, 4], [4, 2]
    tiles = {}
    for sizes, want in ((LARGE, [large, large]), (LARGE_LOGITS, [large, small]),
                        (LARGE_GRADS, [small, large]), (SIZES[4:6], [small, small])):
        tiles.update({(*size, top): want for size in sizes for top in (0, 8, 130)})
    got = launched(_HEAD + f"out = [head(t, d, v, top) for t, d, v, top in {list(tiles)!r}]")
    for (size, want), names in zip(tiles.items(), got):
        assert [_tiles(names, "logits_kernel"), _tiles(names, "grad_kernel")] == want, size
