"""8-bit matrix products for B200 with a scale for each block of 128.

Operands are e4m3 with f32 scales: activations one for each row and 128 columns, weights one for each
128 x 128 block.  The reference has no 8-bit GEMM; the dense product stands beside ``build_gemm`` and
the grouped one beside ``build_grouped_gemm_varlen``.

The product of a row's and a weight block's scale is formed in f32 before it meets the block's sum (which is 0
or between 2^-18 and 2^24.6).  Scales whose products lie in 2^-126 .. 2^127 are what these products are for.  A
smaller one is rounded to f32's subnormal step, which is an error of at most 2^-125 for each block of K; one of
2^128 and more is infinite, and the results of its row and column block infinite or NaN (a block of zeros
included).
"""
from __future__ import annotations

from ..._ids import F_IN_BF16, F_OUT_BF16, K_FP8_GEMM, K_FP8_GROUPED_GEMM, K_FP8_QUANTIZE
from ...kernel import NativeKernel
from ...specs import Layout, Tile
from ...types import PtxType, bf16, e4m3, f32, s32

SCALE_BLOCK = 128
MAX_EXPERTS = 1024


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


def _check(N: int, K: int, out_dtype: PtxType) -> None:
    assert N >= 1 and K >= 1, f"N={N} and K={K} must be positive"
    assert N % 8 == 0, f"N={N} must be divisible by 8"
    assert K % 16 == 0, f"K={K} must be divisible by 16"
    assert out_dtype in (f32, bf16), f"out_dtype must be f32 or bf16, got {out_dtype}"


def build_fp8_gemm(M: int, N: int, K: int, *, out_dtype: PtxType = f32, arch: str = "sm_100a") -> NativeKernel:
    """Kernel ``k(A[M,K] e4m3, a_scale[M,ceil(K/128)] f32, B_T[N,K] e4m3, b_scale[ceil(N/128),ceil(K/128)] f32)
    -> D[M,N]`` with ``D[m,n] = sum_b a_scale[m,b] * b_scale[n//128,b] * sum_{k in block b} A[m,k] * B_T[n,k]``.

    The operands are what ``build_fp8_quantize`` returns (``block_rows=1`` for ``A``, 128 for the weight
    ``B_T``, which is K-major as in ``build_gemm``).  ``M`` is free, from single tokens on; ``N`` divides by 8
    and ``K`` by 16.  Products within a block and the scaled sum over blocks are accumulated in f32 (the range of
    the scales' products: see the module).

    The gradient for the inputs is such a product too, of the gradient in 8 bits and the weight's bytes and grid of
    scales transposed (128 x 128 blocks stay 128 x 128 blocks)::

        dX = build_fp8_gemm(M, K, N)(*build_fp8_quantize(M, N)(dY), B_T.t().contiguous(), b_scale.t().contiguous())

    ``N`` divides by 16 there (else: eight columns of zeros for ``dY`` and eight rows of zeros for ``B_T``).  The 8-bit
    weight itself has no gradient.
    """
    assert M >= 1, f"M={M} must be positive"
    _check(N, K, out_dtype)
    return NativeKernel(
        "fp8_gemm", K_FP8_GEMM, (M, N, K),
        in_specs=(Tile(M, K, e4m3, Layout.TMA_128B, tma_box=(128, 128)), Tile(M, _blocks(K), f32),
                  Tile(N, K, e4m3, Layout.TMA_128B, tma_box=(128, 128)), Tile(_blocks(N), _blocks(K), f32)),
        out_specs=(Tile(M, N, out_dtype, Layout.ROW),),
        flags=F_OUT_BF16 if out_dtype == bf16 else 0, arch=arch,
    )


def build_fp8_grouped_gemm_varlen(G: int, M_total: int, N: int, K: int, *, out_dtype: PtxType = f32,
                                  arch: str = "sm_100a") -> NativeKernel:
    """Kernel ``k(A[M_total,K] e4m3, a_scale[M_total,ceil(K/128)], B_T[G*N,K] e4m3,
    b_scale[G*ceil(N/128),ceil(K/128)], offsets[G+1] s32) -> C[M_total,N]``: the 8-bit form of
    ``build_grouped_gemm_varlen``.

    Expert ``e`` owns rows ``[offsets[e], offsets[e+1])`` of ``A`` and ``C`` and its own ``N`` rows of ``B_T``.
    Offsets live on the device, are non-decreasing within ``[0, M_total]`` and, unlike the bf16 kernel's, need
    no alignment, so ``build_moe_route(..., block=1)`` wastes no rows.  Rows outside
    ``[offsets[0], offsets[G])`` are left unwritten.  ``M_total`` is the static capacity; tiles are chosen by
    ``M_total / G``, so a buffer sized close to the rows that come is quicker (64 experts of 2 rows, 2048 x 2048: 45 us
    in 128 rows, 63 in 8192).
    """
    assert 1 <= G <= MAX_EXPERTS, f"G={G} must be in [1, {MAX_EXPERTS}]"
    assert M_total >= 1, f"M_total={M_total} must be positive"
    _check(N, K, out_dtype)
    return NativeKernel(
        "fp8_grouped_gemm_varlen", K_FP8_GROUPED_GEMM, (G, M_total, N, K),
        in_specs=(Tile(M_total, K, e4m3, Layout.TMA_128B, tma_box=(128, 128)), Tile(M_total, _blocks(K), f32),
                  Tile(G * N, K, e4m3, Layout.TMA_128B, tma_box=(128, 128)), Tile(G * _blocks(N), _blocks(K), f32),
                  Tile(G + 1, s32)),
        out_specs=(Tile(M_total, N, out_dtype, Layout.ROW),),
        flags=F_OUT_BF16 if out_dtype == bf16 else 0, arch=arch,
    )


__all__ = ["build_fp8_quantize", "build_fp8_gemm", "build_fp8_grouped_gemm_varlen"]
