"""Mixture-of-experts and 8-bit operators without a GPU: sizes, refusals, geometry, specs."""
import ctypes

import pytest
import torch

from oracle import formulas
from pyptx_b200 import _ids, _native
from pyptx_b200.examples.blackwell import moe
from pyptx_b200.examples.blackwell.fp8_gemm import build_fp8_gemm, build_fp8_grouped_gemm_varlen, build_fp8_quantize
from pyptx_b200.types import bf16, e4m3, f16, f32, s32, s64


def _create(kid, dims, flags=0):
    err = ctypes.create_string_buffer(_native.ERR_LEN)
    d = (ctypes.c_int64 * len(dims))(*dims)
    rc = _native.load().pb200_create(kid, d, len(dims), None, 0, flags, err)
    if rc > 0:
        _native.load().pb200_destroy(rc)
    return rc, err.value.decode()


@pytest.mark.parametrize("T,k,E,block", [(1, 1, 1, 1), (1, 8, 256, 128), (3, 2, 5, 128), (100, 4, 7, 16), (9, 3, 100, 1)])
def test_moe_rows_holds_every_outcome(T, k, E, block):
    R = moe.moe_rows(T, k, E, block)
    n = T * k
    assert R % block == 0
    # the worst case: as many experts as possible with one row too many for their last block
    used = min(E, n)
    counts = [1] * used
    left = n - used
    for i in range(used):
        add = min(left, (left // block) * block if i == 0 else 0)
        counts[i] += add
        left -= add
    counts[0] += left
    assert sum(counts) == n and sum(-(-c // block) * block for c in counts) <= R
    assert R <= n + used * (block - 1)


def test_specs_and_geometry():
    route = moe.build_moe_route(64, 4, 16, block=16, ids_dtype=s64)
    assert route.in_specs[0].dtype is s64 and [s.shape for s in route.out_specs] == [(64, 4), (route.meta["rows"],), (17,)]
    assert route.grid == (1, 1, 1) and route.block == (256, 1, 1)
    assert moe.build_moe_route(64, 4, 256).block == moe.build_moe_route(1024, 4, 16).block == (1024, 1, 1)
    assert moe.build_moe_route(8192, 4, 64).cluster == (8, 1, 1) and moe.build_moe_route(8192, 4, 64).scratch_bytes == 0
    wide = moe.build_moe_route(32769, 1, 64)                   # more than a cluster takes: the counts go through memory
    assert wide.cluster == (1, 1, 1) and wide.grid[0] > 8 and wide.scratch_bytes == 64 * wide.grid[0] * 4
    d = moe.build_moe_dispatch_fp8(64, 4, 256, 272)
    assert d.out_specs[0].dtype is e4m3 and d.out_specs[1].shape == (256, 3)
    q = build_fp8_quantize(300, 272, block_rows=128, in_dtype=f32)
    assert q.out_specs[1].shape == (3, 3) and q.scratch_bytes == 0
    for k in (moe.build_moe_dispatch(64, 4, 256, 64), moe.build_moe_combine_bwd(64, 4, 256, 64)):
        assert k.scratch_bytes == 0


@pytest.mark.parametrize("call,message", [
    (lambda: moe.build_moe_route(0, 1, 1), "T=0"),
    (lambda: moe.build_moe_route(4, 33, 64), "top_k=33"),
    (lambda: moe.build_moe_route(4, 2, 1025), "E=1025"),
    (lambda: moe.build_moe_route(4, 2, 0), "E=0"),
    (lambda: moe.build_moe_route(4, 2, 8, block=0), "block=0"),
    (lambda: moe.build_moe_route(4, 2, 8, block=16, rows=24), "multiple of block"),
    (lambda: moe.build_moe_route(4, 2, 8, ids_dtype=f32), "ids_dtype"),
    (lambda: moe.build_moe_dispatch(4, 2, 8, 12, dtype=bf16), "divisible by 8"),
    (lambda: moe.build_moe_dispatch(4, 2, 8, 6, dtype=f32), "divisible by 4"),
    (lambda: moe.build_moe_dispatch(4, 2, 0, 8), "R=0"),
    (lambda: moe.build_moe_dispatch_fp8(4, 2, 8, 24), "divisible by 16"),
    (lambda: moe.build_moe_combine(4, 2, 8, 64, dtype=f16), "f32 or bf16"),
    (lambda: moe.build_moe_combine_bwd(4, 0, 8, 64), "top_k=0"),
    (lambda: build_fp8_quantize(4, 24), "divisible by 16"),
    (lambda: build_fp8_quantize(4, 32, block_rows=64), "block_rows"),
    (lambda: build_fp8_quantize(0, 32), "positive"),
    (lambda: build_fp8_quantize(4, 32, in_dtype=s32), "f32 or bf16"),
    (lambda: moe.moe_rows(0, 1, 1), "positive"),
])
def test_builders_refuse(call, message):
    with pytest.raises(AssertionError, match=message):
        call()


@pytest.mark.parametrize("kid,dims,message", [
    (_ids.K_MOE_ROUTE, (4, 2, 8, 16), "needs 5 dims"),
    (_ids.K_MOE_ROUTE, (4, 2, 8, 16, 0), "positive"),
    (_ids.K_MOE_ROUTE, (4, 2, 8, 16, 24), "divisible by block"),
    (_ids.K_MOE_ROUTE, (4, 33, 8, 16, 32), "top_k=33"),
    (_ids.K_MOE_ROUTE, (4, 2, 1025, 16, 32), "E=1025"),
    (_ids.K_MOE_ROUTE, (4, 2, 8, 1025, 1025), "block=1025"),
    (_ids.K_MOE_ROUTE, (2 ** 30, 2, 8, 1, 32), "exceeds 2^30"),
    (_ids.K_MOE_ROUTE, (2 ** 33, 1, 8, 1, 32), "exceeds"),
    (_ids.K_MOE_DISPATCH, (4, 2, 8, 6), "divisible by 4"),
    (_ids.K_MOE_DISPATCH_FP8, (4, 2, 8, 24), "divisible by 16"),
    (_ids.K_MOE_COMBINE, (4, 2, 8), "needs 4 dims"),
    (_ids.K_MOE_COMBINE_BWD, (4, -1, 8, 64), "positive"),
    (_ids.K_MOE_DISPATCH, (2 ** 29, 1, 8, 2 ** 20), "too large"),
    (_ids.K_FP8_QUANTIZE, (4, 24, 1), "divisible by 16"),
    (_ids.K_FP8_QUANTIZE, (4, 32, 2), "block_rows"),
    (_ids.K_FP8_QUANTIZE, (2 ** 30, 2 ** 20, 1), "too large"),
    (_ids.K_FP8_QUANTIZE, (1, 2 ** 31 - 16, 1), "exceeds"),
    (_ids.K_MOE_ROUTE, (4, 2, 8, 1, 2 ** 31 - 4096), "exceeds"),
    (_ids.K_MOE_DISPATCH_FP8, (1, 1, 1, 2 ** 31 - 16), "exceeds"),
])
def test_library_refuses(kid, dims, message):
    rc, text = _create(kid, dims)
    assert rc == _ids.ERR_BAD_SHAPE and message in text, (rc, text)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="no CPU path"):
        moe.build_moe_route(4, 2, 8)(torch.zeros(4, 2, dtype=torch.int32))


def test_oracle_e4m3_rounding_matches_torch():
    x = torch.cat([torch.randn(4000) * 100, torch.randn(4000) * 0.01, torch.arange(-450, 450).float()]).clamp(-448, 448)
    assert torch.equal(formulas.e4m3_round(x.double()), x.to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("call,message", [
    (lambda: build_fp8_gemm(0, 8, 16), "M=0"),
    (lambda: build_fp8_gemm(1, 12, 16), "divisible by 8"),
    (lambda: build_fp8_gemm(1, 8, 24), "divisible by 16"),
    (lambda: build_fp8_gemm(1, 8, 16, out_dtype=f16), "f32 or bf16"),
    (lambda: build_fp8_grouped_gemm_varlen(1025, 8, 8, 16), "G=1025"),
    (lambda: build_fp8_grouped_gemm_varlen(2, 0, 8, 16), "M_total=0"),
])
def test_fp8_gemm_builders_refuse(call, message):
    with pytest.raises(AssertionError, match=message):
        call()


@pytest.mark.parametrize("kid,dims,message", [
    (_ids.K_FP8_GEMM, (1, 12, 16), "divisible by 8"),
    (_ids.K_FP8_GEMM, (1, 8, 24), "divisible by 16"),
    (_ids.K_FP8_GEMM, (1, 8), "needs 3 dims"),
    (_ids.K_FP8_GEMM, (0, 8, 16), "positive"),
    (_ids.K_FP8_GEMM, (2 ** 31 - 1, 8, 16), "2^31-1"),
    (_ids.K_FP8_GEMM, (2 ** 30, 2 ** 30, 16), "2^31-1"),
    (_ids.K_FP8_GROUPED_GEMM, (1025, 8, 8, 16), "G=1025"),
    (_ids.K_FP8_GROUPED_GEMM, (1024, 8, 2 ** 22, 16), "2^31-1"),
])
def test_library_refuses_fp8_gemm(kid, dims, message):
    rc, text = _create(kid, dims)
    assert rc == _ids.ERR_BAD_SHAPE and message in text, (rc, text)


def test_fp8_gemm_geometry():
    """Single tokens stream the weight; products with few tiles split K over a cluster; large ones fill the SMs
    with whole tiles."""
    one = build_fp8_gemm(1, 4096, 4096)
    assert one.cluster == (1, 1, 1) and one.grid == (256, 1, 1) and one.block[0] >= 128 and one.scratch_bytes == 0
    assert build_fp8_gemm(1, 40, 144).block == (64, 1, 1)
    for rows in (17, 64):
        few = build_fp8_gemm(rows, 4096, 4096)
        assert few.cluster[0] > 1 and few.grid[0] % few.cluster[0] == 0 and few.scratch_bytes == 0
    big = build_fp8_gemm(8192, 8192, 4096, out_dtype=bf16)
    assert big.cluster == (2, 1, 1) and 100 < big.grid[0] <= 148 and big.smem <= 227 * 1024
    grouped = build_fp8_grouped_gemm_varlen(64, 128, 2048, 2064)
    assert grouped.in_specs[3].shape == (64 * 16, 17) and grouped.in_specs[4].dtype is s32
