"""What handles of the movement, quantising and 8-bit kernels publish is what their launches take (no GPU: sizes are
planned for 148 SMs)."""
import pytest

from pyptx_b200.examples.blackwell import moe
from pyptx_b200.examples.blackwell.fp8_gemm import build_fp8_gemm, build_fp8_quantize
from pyptx_b200.types import bf16, f32

TYPES = {"bf16": (bf16, 2), "f32": (f32, 4)}


def _up(a, b):
    return -(-a // b)


def _steps(rows, width, step, most):
    """Steps of a warp: the most that leave 16 warps an SM and at most an eighth of the row beyond its end."""
    while most > 1 and (rows * _up(width, step * most) < 148 * 16 or _up(width, step * most) * step * most * 8 > width * 9):
        most //= 2
    return most


MOVES = [(1, 1, 1, 64), (64, 4, 256, 64), (16, 8, 128, 4096), (1001, 3, 3168, 1008), (8192, 4, 36832, 4096), (300, 2, 640, 16384)]


@pytest.mark.parametrize("T,k,R,H", MOVES)
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_movement_grids(T, k, R, H, kind):
    dtype, size = TYPES[kind]
    vecs = H * size // 16

    def grid(steps, step, width, clears):
        segs = _up(width, step * steps)
        return _up((_up(R, 32) if clears else 0) * segs + T * segs, 4)

    d = moe.build_moe_dispatch(T, k, R, H, dtype=dtype)
    assert d.grid == (grid(_steps(T, vecs, 32, 4), 32, vecs, True), 1, 1) and d.block == (128, 1, 1)
    q = moe.build_moe_dispatch_fp8(T, k, R, H, in_dtype=dtype)
    assert q.grid == (grid(_steps(T, H, 256, 4), 256, H, True), 1, 1)
    for c in (moe.build_moe_combine(T, k, R, H, dtype=dtype), moe.build_moe_dispatch_bwd(T, k, R, H, dtype=dtype)):
        assert c.grid == (grid(_steps(T, vecs, 32, 2), 32, vecs, False), 1, 1)
    b = moe.build_moe_combine_bwd(T, k, R, H, dtype=dtype)
    assert b.grid == (_up(_up(R, 32) * _up(vecs, 128), 4) + T, 1, 1)


@pytest.mark.parametrize("M,K,grid", [(8192, 8192, 16384), (1, 16, 1), (1000, 2064, 2250), (33, 4096, 132)])
def test_row_quantisation_grid(M, K, grid):
    """1000 x 2064: one step (two would end 496 columns past the row, more than an eighth), nine segments a row."""
    kernel = build_fp8_quantize(M, K)
    assert kernel.grid == (grid, 1, 1) and kernel.block == (128, 1, 1)
    steps = _steps(M, K, 256, 4)
    assert grid == _up(M * _up(K, 256 * steps), 4)
    blocks = build_fp8_quantize(M, K, block_rows=128)
    assert blocks.grid == (_up(M, 128) * _up(K, 128), 1, 1) and blocks.block == (512, 1, 1)


@pytest.mark.parametrize("M,N,K,tiles", [(1, 4096, 4096, 1), (8, 40, 144, 1), (9, 1016, 528, 2), (16, 1024, 4096, 2), (17, 2048, 2048, 4),
                                         (32, 1024, 1024, 4)])
def test_streaming_product_publishes_its_shared_memory(M, N, K, tiles):
    """One f32 for each warp, token of its tiles of eight and weight row of 16."""
    kernel = build_fp8_gemm(M, N, K)
    assert kernel.grid == (_up(N, 16), 1, 1) and kernel.smem == kernel.block[0] // 32 * 16 * 8 * tiles * 4 > 0
