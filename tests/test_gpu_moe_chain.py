"""Chains of calls on the same buffers, call after call with other contents and nothing in between: kernels start while the
ones before them still run, and each must see what the last one wrote.  Whatever was read too early has other bits."""
import pytest
import torch

from pyptx_b200 import _native
from pyptx_b200.examples.blackwell import moe
from pyptx_b200.examples.blackwell.fp8_gemm import build_fp8_gemm, build_fp8_grouped_gemm_varlen, build_fp8_quantize

pytestmark = pytest.mark.gpu


def _launch(kernel, *buffers):
    if kernel.scratch_bytes:
        buffers += (torch.empty(kernel.scratch_bytes, dtype=torch.uint8, device="cuda"),)
    _native.launch_raw(kernel.handle, torch.cuda.current_stream().cuda_stream, [b.data_ptr() for b in buffers])


def _buffers(kernel):
    names = {"bf16": torch.bfloat16, "f32": torch.float32, "s32": torch.int32, "e4m3": torch.float8_e4m3fn}
    return [torch.empty(s.shape, dtype=names[s.dtype.name], device="cuda") for s in kernel.out_specs]


def _check(step, n, outs):
    """``step(i, wait)`` fills ``outs[i]``: in turn with a wait after every call, then back to back and replayed."""
    for i in range(n):
        step(i, torch.cuda.synchronize)
    want = [[t.clone() for t in o] for o in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(n):
            step(i, lambda: None)
    for replay in range(10):
        for o in outs:
            for t in o:
                t.zero_()
        if replay % 2:
            graph.replay()
        else:
            for i in range(n):
                step(i, lambda: None)
        torch.cuda.synchronize()
        for o, v in zip(outs, want):
            for a, b in zip(o, v):
                assert torch.equal(a, b)


@pytest.mark.parametrize("M,N,K", [(1, 2368, 1024), (4, 256, 512), (12, 1024, 1024), (30, 1024, 1024), (24, 1024, 1024),
                                   (40, 1024, 1024), (600, 4096, 512)])
@pytest.mark.parametrize("side", ["activations", "weight"])
def test_quantise_then_multiply(M, N, K, side):
    n = 20
    rows, block = (M, 1) if side == "activations" else (N, 128)
    quantize, gemm = build_fp8_quantize(rows, K, block_rows=block), build_fp8_gemm(M, N, K)
    other = build_fp8_quantize(N if block == 1 else M, K, block_rows=128 if block == 1 else 1)
    fixed = other(torch.randn(N if block == 1 else M, K, device="cuda").bfloat16())
    x = [torch.randn(rows, K, device="cuda").bfloat16() for _ in range(n)]
    q, scale = _buffers(quantize)
    outs = [_buffers(gemm) for _ in range(n)]

    def step(i, wait):
        _launch(quantize, x[i], q, scale)
        wait()
        _launch(gemm, *((q, scale, *fixed) if block == 1 else (*fixed, q, scale)), *outs[i])
        wait()

    _check(step, n, outs)


@pytest.mark.parametrize("T,k,E,H", [(4, 2, 8, 256), (16, 8, 64, 1024), (300, 4, 16, 512), (10000, 4, 40, 64)])
def test_route_move_multiply_and_back(T, k, E, H):
    n, N = 20, 64
    R = moe.moe_rows(T, k, E, 1)
    route, into8 = moe.build_moe_route(T, k, E, block=1), moe.build_moe_dispatch_fp8(T, k, R, H)
    grouped, dispatch = build_fp8_grouped_gemm_varlen(E, R, N, H), moe.build_moe_dispatch(T, k, R, H)
    combine, combine_bwd = moe.build_moe_combine(T, k, R, H), moe.build_moe_combine_bwd(T, k, R, H)
    dispatch_bwd = moe.build_moe_dispatch_bwd(T, k, R, H)
    ids = [torch.rand(T, E, device="cuda").topk(k, dim=-1).indices.int() for _ in range(n)]
    x, w = torch.randn(T, H, device="cuda").bfloat16(), torch.rand(T, k, device="cuda")
    w8 = torch.randn(E * N, H, device="cuda").to(torch.float8_e4m3fn)
    w_scale = torch.rand(E, -(-H // 128), device="cuda")
    row_of, entry_of, offsets = _buffers(route)
    (rows,), (q, scale), d_rows = _buffers(dispatch), _buffers(into8), _buffers(combine_bwd)[0]
    outs = [[*_buffers(grouped), *_buffers(combine), _buffers(combine_bwd)[1], *_buffers(dispatch_bwd)] for _ in range(n)]

    def step(i, wait):
        product, back, d_weights, dx = outs[i]
        for kernel, buffers in ((route, (ids[i], row_of, entry_of, offsets)), (into8, (x, row_of, entry_of, q, scale)),
                                (grouped, (q, scale, w8, w_scale, offsets, product)), (dispatch, (x, row_of, entry_of, rows)),
                                (combine, (rows, w, row_of, back)),
                                (combine_bwd, (rows, w, row_of, entry_of, x, d_rows, d_weights)),
                                (dispatch_bwd, (row_of, d_rows, dx))):
            _launch(kernel, *buffers)
            wait()

    _check(step, n, outs)
