"""Which kernels calls of the vocabulary loss and the embedding launch, on the CPU."""
import pytest

from launches import launched

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
