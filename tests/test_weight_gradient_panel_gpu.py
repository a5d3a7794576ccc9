"""Weight gradients of at most 256 rows, whose panel of the rows stays in shared memory (csrc/gemm2.cu), against 64 bits.

Bound: fp32 sums of K exact products, 16 at a time (each addition may truncate, 2 eps): (K / 16 + 2) 4 eps of the sum of magnitudes; one rounding to bf16, 2^-8 of the result."""
import pytest
import torch

from llmc_b200 import ops

pytestmark = pytest.mark.gpu
EPS, B = 2.0 ** -24, 2.0 ** -8


@pytest.mark.parametrize("rows,OC,C", [(1, 5000, 1600), (16, 10248, 776), (64, 14336, 1024), (65, 2504, 1032), (200, 6144, 2048), (255, 4104, 1288), (256, 50304, 264), (256, 9000, 2056)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_weight_gradient(rows, OC, C, accumulate):
    g = torch.Generator(device="cuda").manual_seed(rows + OC)
    dout, inp = (torch.randn(rows, n, generator=g, device="cuda").to(torch.bfloat16) for n in (OC, C))
    old = torch.randn(OC, C, generator=g, device="cuda").to(torch.bfloat16)
    around = torch.full((OC + 2, C), 3.0, dtype=torch.bfloat16, device="cuda")
    dw = around[1:-1]
    dw.copy_(old)
    ops.matmul_wgrad(dw, dout, inp, accumulate=accumulate)
    a, b = dout.double(), inp.double()
    want = a.t() @ b
    bound = (rows / 16 + 2) * 4 * EPS * (a.abs().t() @ b.abs())
    if accumulate:
        want += old.double()
        bound += 2 * EPS * want.abs()
    assert ((dw.double() - want).abs() <= bound + 1.01 * B * want.abs() + 1e-30).all()
    assert (around[0] == 3).all() and (around[-1] == 3).all()
    again = old.clone()
    ops.matmul_wgrad(again, dout, inp, accumulate=accumulate)
    assert torch.equal(again, dw)
