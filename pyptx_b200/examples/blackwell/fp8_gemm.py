"""8-bit matrix products for B200 with a scale for each block of 128.

Operands are e4m3 with f32 scales: activations one for each row and 128 columns, weights one for each
128 x 128 block.  The reference has no 8-bit GEMM; the dense product stands beside ``build_gemm`` and
the grouped one beside ``build_grouped_gemm_varlen``.
"""
from __future__ import annotations

from ..._ids import F_IN_BF16, K_FP8_QUANTIZE
from ...kernel import NativeKernel
from ...specs import Tile
from ...types import PtxType, bf16, e4m3, f32

SCALE_BLOCK = 128


def _blocks(n: int) -> int:
    return -(-n // SCALE_BLOCK)


def build_fp8_quantize(M: int, K: int, *, block_rows: int = 1, in_dtype: PtxType = bf16,
                       arch: str = "sm_100a") -> NativeKernel:
    """Kernel ``k(x[M,K]) -> (q[M,K] e4m3, scale[ceil(M/block_rows),ceil(K/128)] f32)`` with ``x ~ q * scale``.

    ``block_rows=1`` gives the activations' scales (one for each row and 128 columns), ``block_rows=128``
    the weights'.  ``scale = max(amax / 448, 2^-120)`` and ``q = e4m3(x * (1 / scale))``, in f32 with every
    step rounded to nearest.  A NaN stays in its own element; a block that holds an infinity comes back
    as NaN.  ``in_dtype`` is bf16 or f32.
    """
    assert M >= 1 and K >= 1, f"shape ({M}, {K}) must be positive"
    assert K % 16 == 0, f"K={K} must be divisible by 16"
    assert block_rows in (1, SCALE_BLOCK), f"block_rows must be 1 or {SCALE_BLOCK}, got {block_rows}"
    assert in_dtype in (f32, bf16), f"in_dtype must be f32 or bf16, got {in_dtype}"
    return NativeKernel(
        "fp8_quantize", K_FP8_QUANTIZE, (M, K, block_rows),
        in_specs=(Tile(M, K, in_dtype),),
        out_specs=(Tile(M, K, e4m3), Tile(-(-M // block_rows), _blocks(K), f32)),
        flags=F_IN_BF16 if in_dtype == bf16 else 0, arch=arch, meta={"block_rows": block_rows},
    )


__all__ = ["build_fp8_quantize"]
