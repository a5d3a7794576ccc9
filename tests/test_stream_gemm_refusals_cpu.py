"""Sizes that csrc/stream_gemm.cu does not take are refused before anything is launched."""
import pytest

from llmc_b200 import _lib


@pytest.mark.parametrize("form", [0, 1, 2])
def test_depth_is_a_multiple_of_eight(form):
    assert _lib.cuda().llmc_stream_gemm(None, None, None, None, 8, 64, 60, 64, 64, 64, form, None) == -1
