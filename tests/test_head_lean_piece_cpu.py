"""Pieces of the vocabulary in a model that keeps no logits."""
import pytest

from llmc_b200.ops import kernels as KN


@pytest.mark.parametrize("V", [1, 300, 50257, 128256])
def test_a_third_of_the_logits(V):
    """No more than a third of the logits and a tile of columns, where they are large, and never more than the operators would hold by themselves."""
    for N in (1, 77, 1000, 2048, 4096, 8192, 16384, 65536, 10 ** 6):
        cols = KN.head_lean_piece(N, V)
        assert cols == V or (cols % 256 == 0 and cols < V)
        assert cols <= KN.head_piece(N, V)
        held = 2 * N * cols
        assert held <= max(KN.HEAD_LEAN_BYTES, 2 * N * V / 3 + 512 * N) or cols == 256
        if 2 * N * V <= KN.HEAD_LEAN_BYTES:
            assert cols == V
