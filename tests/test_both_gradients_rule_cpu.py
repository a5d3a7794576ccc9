"""Products whose two gradients go to one launch (csrc/gemm2.cu): what its kernels are there for."""
import pytest

from llmc_b200 import _lib


@pytest.mark.parametrize("sms", [148, 132, 100, 20])
def test_few_rows_always_have_pairs_for_panels(sms):
    """At most 128 rows: the weight gradient keeps panels wherever both gradients go to one launch, since a pair is left for every column of tiles."""
    slots = _lib.cuda().llmc_gemm2_both_slots
    seen = 0
    for M in (1, 16, 64, 65, 128):
        for C in list(range(8, 600, 8)) + list(range(600, 8200, 104)):
            for K in (100, 5000, 20001, 50257, 128256):
                S = slots(M, C, K, sms)
                if S > 0:
                    tiles = -(-C // 256)
                    assert sms // 2 - tiles * S >= tiles
                    seen += 1
    assert seen > 100 or sms < 100
