"""Mixture-of-experts token movement for B200: tokens sorted by expert for the grouped GEMMs, and back.

The reference's grouped GEMM takes rows that are stacked by expert already
(examples/blackwell/grouped_gemm.py:295-306); these kernels make them from a router's choices and bring
the experts' results back, in both directions of a training step::

    R = moe_rows(T, top_k, E)                                   # holds every routing outcome
    row_of, entry_of, offsets = build_moe_route(T, top_k, E)(ids)
    rows = build_moe_dispatch(T, top_k, R, H)(x, row_of, entry_of)
    y = build_grouped_gemm_varlen(E, R, N, H, out_dtype=bf16)(rows, weight, offsets)
    out = build_moe_combine(T, top_k, R, N)(y, router_weights, row_of)

``T`` tokens choose ``top_k`` experts each; entry ``i = t * top_k + j`` is choice ``j`` of token ``t``.
Sums are f32 in the order of ``j`` and no kernel uses atomics, so results do not change from run to run.
"""
from __future__ import annotations

from ..._ids import (F_IDS_S64, F_IN_BF16, F_OUT_BF16, K_MOE_COMBINE, K_MOE_COMBINE_BWD, K_MOE_DISPATCH,
                     K_MOE_DISPATCH_BWD, K_MOE_DISPATCH_FP8, K_MOE_ROUTE)
from ...kernel import NativeKernel
from ...specs import Tile
from ...types import PtxType, bf16, e4m3, f32, s32, s64

MAX_EXPERTS = 1024
MAX_TOP_K = 32
MAX_BLOCK = 1024
SCALE_BLOCK = 128


def moe_rows(T: int, top_k: int, E: int, block: int = 128) -> int:
    """Rows that hold every routing outcome of ``T * top_k`` entries when each expert's rows are padded
    to a multiple of ``block``: no more than ``min(E, T * top_k)`` experts have rows at all."""
    assert T >= 1 and top_k >= 1 and E >= 1 and block >= 1, "T, top_k, E and block must be positive"
    n = T * top_k
    return (n + min(E, n) * (block - 1)) // block * block


def _check(T: int, top_k: int, R: int, H: int, dtype: PtxType) -> None:
    assert T >= 1 and R >= 1 and H >= 1, f"T={T}, R={R} and H={H} must be positive"
    assert 1 <= top_k <= MAX_TOP_K, f"top_k={top_k} must be in [1, {MAX_TOP_K}]"
    assert dtype in (f32, bf16), f"dtype must be f32 or bf16, got {dtype}"
    unit = 8 if dtype == bf16 else 4
    assert H % unit == 0, f"H={H} must be divisible by {unit} (128-bit vector access)"


def _flags(dtype: PtxType) -> int:
    return F_OUT_BF16 if dtype == bf16 else 0


def build_moe_route(T: int, top_k: int, E: int, *, block: int = 128, rows: int | None = None,
                    ids_dtype: PtxType = s32, arch: str = "sm_100a") -> NativeKernel:
    """Kernel ``k(ids[T,top_k]) -> (row_of[T,top_k], entry_of[R], offsets[E+1])`` (all s32; ``ids`` s32 or s64).

    A stable sort of the entries by expert.  Expert ``e`` owns rows ``[offsets[e], offsets[e+1])``, a
    multiple of ``block`` of them (128 is what ``build_grouped_gemm_varlen`` takes; the 8-bit grouped
    GEMM takes 1).  ``row_of`` is each entry's row, ``entry_of`` its inverse with -1 in rows that no entry owns.
    Ids outside ``[0, E)`` (another rank's experts, padding tokens) are dropped: row -1.  ``rows`` (default
    ``moe_rows(...)``, which always suffices) is the static row count ``R``, a multiple of ``block``;
    entries that would land at or beyond it are dropped too and ``offsets`` is clipped to it.
    """
    assert T >= 1, f"T={T} must be positive"
    assert 1 <= top_k <= MAX_TOP_K, f"top_k={top_k} must be in [1, {MAX_TOP_K}]"
    assert 1 <= E <= MAX_EXPERTS, f"E={E} must be in [1, {MAX_EXPERTS}]"
    assert 1 <= block <= MAX_BLOCK, f"block={block} must be in [1, {MAX_BLOCK}]"
    R = moe_rows(T, top_k, E, block) if rows is None else rows
    assert R >= 1 and R % block == 0, f"rows={R} must be a positive multiple of block={block}"
    assert ids_dtype in (s32, s64), f"ids_dtype must be s32 or s64, got {ids_dtype}"
    return NativeKernel(
        "moe_route", K_MOE_ROUTE, (T, top_k, E, block, R),
        in_specs=(Tile(T, top_k, ids_dtype),),
        out_specs=(Tile(T, top_k, s32), Tile(R, s32), Tile(E + 1, s32)),
        flags=F_IDS_S64 if ids_dtype == s64 else 0, arch=arch, meta={"block": block, "rows": R},
    )


def build_moe_dispatch(T: int, top_k: int, R: int, H: int, *, dtype: PtxType = bf16,
                       arch: str = "sm_100a") -> NativeKernel:
    """Kernel ``k(x[T,H], row_of[T,top_k], entry_of[R]) -> rows[R,H]``: each token copied to its
    entries' rows; rows that no entry owns are zeros.  ``dtype`` (bf16 or f32) is that of both."""
    _check(T, top_k, R, H, dtype)
    return NativeKernel(
        "moe_dispatch", K_MOE_DISPATCH, (T, top_k, R, H),
        in_specs=(Tile(T, H, dtype), Tile(T, top_k, s32), Tile(R, s32)),
        out_specs=(Tile(R, H, dtype),), flags=_flags(dtype), arch=arch,
    )


def build_moe_dispatch_fp8(T: int, top_k: int, R: int, H: int, *, in_dtype: PtxType = bf16,
                           arch: str = "sm_100a") -> NativeKernel:
    """Kernel ``k(x[T,H], row_of, entry_of) -> (q[R,H] e4m3, scale[R,ceil(H/128)] f32)``: dispatch and
    ``build_fp8_quantize`` in one pass, each token quantised once.  Rows that no entry owns are zeros
    with scale 0."""
    _check(T, top_k, R, H, in_dtype)
    assert H % 16 == 0, f"H={H} must be divisible by 16"
    return NativeKernel(
        "moe_dispatch_fp8", K_MOE_DISPATCH_FP8, (T, top_k, R, H),
        in_specs=(Tile(T, H, in_dtype), Tile(T, top_k, s32), Tile(R, s32)),
        out_specs=(Tile(R, H, e4m3), Tile(R, -(-H // SCALE_BLOCK), f32)),
        flags=F_IN_BF16 if in_dtype == bf16 else 0, arch=arch,
    )


def build_moe_dispatch_bwd(T: int, top_k: int, R: int, H: int, *, dtype: PtxType = bf16,
                           arch: str = "sm_100a") -> NativeKernel:
    """Kernel ``k(row_of[T,top_k], d_rows[R,H]) -> dx[T,H]``: each token's gradient is the sum of its
    entries' rows (dropped entries add nothing), in f32, rounded once."""
    _check(T, top_k, R, H, dtype)
    return NativeKernel(
        "moe_dispatch_bwd", K_MOE_DISPATCH_BWD, (T, top_k, R, H),
        in_specs=(Tile(T, top_k, s32), Tile(R, H, dtype)),
        out_specs=(Tile(T, H, dtype),), flags=_flags(dtype), arch=arch,
    )


def build_moe_combine(T: int, top_k: int, R: int, H: int, *, dtype: PtxType = bf16,
                      arch: str = "sm_100a") -> NativeKernel:
    """Kernel ``k(rows[R,H], weights[T,top_k] f32, row_of[T,top_k]) -> out[T,H]``:
    ``out[t] = sum_j weights[t,j] * rows[row_of[t,j]]`` in f32, rounded once.  Dropped entries (row -1)
    add nothing, whatever their weight; a token without entries gives zeros."""
    _check(T, top_k, R, H, dtype)
    return NativeKernel(
        "moe_combine", K_MOE_COMBINE, (T, top_k, R, H),
        in_specs=(Tile(R, H, dtype), Tile(T, top_k, f32), Tile(T, top_k, s32)),
        out_specs=(Tile(T, H, dtype),), flags=_flags(dtype), arch=arch,
    )


def build_moe_combine_bwd(T: int, top_k: int, R: int, H: int, *, dtype: PtxType = bf16,
                          arch: str = "sm_100a") -> NativeKernel:
    """Kernel ``k(rows[R,H], weights, row_of, entry_of[R], dout[T,H]) -> (d_rows[R,H], d_weights[T,top_k] f32)``:
    ``d_rows[row_of[t,j]] = weights[t,j] * dout[t]`` (zeros in rows that no entry owns) and
    ``d_weights[t,j] = <rows[row_of[t,j]], dout[t]>`` (0 for dropped entries)."""
    _check(T, top_k, R, H, dtype)
    return NativeKernel(
        "moe_combine_bwd", K_MOE_COMBINE_BWD, (T, top_k, R, H),
        in_specs=(Tile(R, H, dtype), Tile(T, top_k, f32), Tile(T, top_k, s32), Tile(R, s32), Tile(T, H, dtype)),
        out_specs=(Tile(R, H, dtype), Tile(T, top_k, f32)), flags=_flags(dtype), arch=arch,
    )


def build_differentiable_moe_dispatch(T: int, top_k: int, R: int, H: int, *, dtype: PtxType = bf16):
    """``dispatch(x, row_of, entry_of) -> rows`` that takes part in autograd (gradient for ``x``), through
    the reference's hook (pyptx/torch_support.py:446-519)."""
    from ...torch_support import differentiable_kernel

    fwd = build_moe_dispatch(T, top_k, R, H, dtype=dtype)
    bwd = build_moe_dispatch_bwd(T, top_k, R, H, dtype=dtype)
    return differentiable_kernel(fwd, bwd, save_for_backward=(1,))


def build_differentiable_moe_combine(T: int, top_k: int, R: int, H: int, *, dtype: PtxType = bf16):
    """``combine(rows, weights, row_of, entry_of) -> out`` that takes part in autograd (gradients for
    ``rows`` and ``weights``); ``entry_of`` serves the backward pass, which clears unowned rows."""
    from ...torch_support import differentiable_kernel

    fwd = build_moe_combine(T, top_k, R, H, dtype=dtype)
    bwd = build_moe_combine_bwd(T, top_k, R, H, dtype=dtype)

    def forward(rows, weights, row_of, entry_of):
        return fwd(rows, weights, row_of)

    forward.__name__ = fwd.__name__
    return differentiable_kernel(forward, bwd)


def moe_dispatch_bytes(T: int, top_k: int, R: int, H: int, element: int = 2) -> int:
    """Algorithmic bytes of one dispatch: tokens read once, rows written once, both maps read."""
    return (T + R) * H * element + 4 * (T * top_k + R)


__all__ = ["moe_rows", "build_moe_route", "build_moe_dispatch", "build_moe_dispatch_fp8", "build_moe_dispatch_bwd",
           "build_moe_combine", "build_moe_combine_bwd", "build_differentiable_moe_dispatch",
           "build_differentiable_moe_combine", "moe_dispatch_bytes"]
