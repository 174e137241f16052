"""bf16 results of the 8-bit product: one rounding of the f32 results, the same bits from call to call."""
import pytest
import torch

from pyptx_b200.examples.blackwell.fp8_gemm import build_fp8_gemm
from pyptx_b200.types import bf16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (12, 264, 2064), (30, 520, 1040), (24, 264, 8208), (100, 520, 1040), (2050, 2056, 528)])
def test_bf16_results_are_the_f32_ones_rounded_once_and_repeat(M, N, K):
    """In every form; between two calls the same kernel runs on other operands."""
    g = torch.Generator().manual_seed(M)

    def operands():
        kb, nb = -(-K // 128), -(-N // 128)
        a, b = ((torch.randn(r, K, generator=g) * 140).clamp(-448, 448).to(torch.float8_e4m3fn).cuda() for r in (M, N))
        return a, (torch.rand(M, kb, generator=g) + 0.5).cuda(), b, (torch.rand(nb, kb, generator=g) + 0.5).cuda()

    ins, other = operands(), operands()
    kernel = build_fp8_gemm(M, N, K, out_dtype=bf16)
    want = build_fp8_gemm(M, N, K)(*ins).bfloat16()
    for _ in range(20):
        kernel(*other)
        assert torch.equal(kernel(*ins), want)
