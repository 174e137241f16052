"""The gradient of the 8-bit products for their inputs, as their builders describe it."""
import pytest
import torch

from oracle import formulas
from pyptx_b200.examples.blackwell.fp8_gemm import build_fp8_gemm, build_fp8_grouped_gemm_varlen, build_fp8_quantize
from pyptx_b200.types import f32

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def _weight(rows, cols, g):
    return build_fp8_quantize(rows, cols, block_rows=128, in_dtype=f32)((torch.randn(rows, cols, generator=g) / cols ** 0.5).cuda())


def _gemm_bound(blocks, want, mag):
    return (256 + blocks + 9) * U32 * mag


def _dequantized(q, scale, block_rows):
    rows, cols = q.shape
    s = scale.cpu().double().repeat_interleave(block_rows, dim=0)[:rows]
    return q.cpu().float().double() * s.repeat_interleave(128, dim=1)[:, :cols]


@pytest.mark.parametrize("M,N,K", [(1, 272, 400), (20, 4096, 512), (40, 272, 400), (200, 528, 1040), (2100, 1040, 2064)])
def test_input_gradient_of_the_product(M, N, K):
    """dX = k'(quantised dY, W^T): against the formula on the quantised operands, and dY W within dY's quantisation (half a
    step of e4m3, 2^-4 relative or 2^-10 of the block's scale, for each element) besides."""
    g = torch.Generator().manual_seed(M + N)
    w8, w_scale = _weight(N, K, g)
    dy = torch.randn(M, N, generator=g).bfloat16()
    dq, d_scale = build_fp8_quantize(M, N)(dy.cuda())
    wt, wt_scale = w8.t().contiguous(), w_scale.t().contiguous()
    dx = build_fp8_gemm(M, K, N)(dq, d_scale, wt, wt_scale).cpu().double()
    want, mag = formulas.fp8_gemm_ref(dq.cpu(), d_scale.cpu(), wt.cpu(), wt_scale.cpu())
    bound = _gemm_bound(d_scale.shape[1], want, mag)
    assert ((dx - want).abs() <= bound).all()
    w = _dequantized(w8, w_scale, 128)
    off = 2.0 ** -4 * dy.double().abs() + 2.0 ** -10 * d_scale.cpu().double().repeat_interleave(128, dim=1)[:, :N]
    # the scaled value is rounded to f32 before it is to e4m3: two more half steps of f32 of it
    assert ((dx - dy.double() @ w).abs() <= (off + 3 * U32 * dy.double().abs()) @ w.abs() + bound).all()


def test_input_gradient_of_the_product_against_differences():
    """<D(X + E) - D(X - E), dY> / 2 = <dX, E> where X, E and X +- E are 8-bit values (small whole numbers) of scale 1: D is
    linear, and both sides are sums of f32 results within their bounds.  dY is a multiple of its quantisation."""
    M, N, K = 70, 272, 400
    g = torch.Generator().manual_seed(2)
    w8, w_scale = _weight(N, K, g)
    dq = torch.randint(-8, 9, (M, N), generator=g).float()
    x, e = (torch.randint(-4, 5, (M, K), generator=g).float() for _ in range(2))
    one = torch.ones(M, -(-K // 128)).cuda()
    forward, backward = build_fp8_gemm(M, N, K), build_fp8_gemm(M, K, N)
    eight = lambda t: t.to(torch.float8_e4m3fn).cuda()
    up, down = (forward(eight(x + s * e), one, w8, w_scale).cpu().double() for s in (1, -1))
    dx = backward(eight(dq), torch.ones(M, -(-N // 128)).cuda(), w8.t().contiguous(), w_scale.t().contiguous()).cpu().double()
    left, right = ((up - down) * 0.5 * dq.double()).sum(), (dx * e.double()).sum()
    w = _dequantized(w8, w_scale, 128).abs()
    slack = _gemm_bound(4, None, 0.5 * ((x + e).abs().double() + (x - e).abs().double()) @ w.T * dq.abs().double()).sum()
    slack += _gemm_bound(3, None, dq.abs().double() @ w * e.abs().double()).sum()
    assert abs(left - right) <= slack


def test_input_gradient_of_the_grouped_product():
    """The experts' weights transposed one by one."""
    counts, N, K = [3, 0, 40, 130], 272, 400
    E, M = len(counts), sum(counts)
    g = torch.Generator().manual_seed(8)
    pairs = [_weight(N, K, g) for _ in counts]
    wt, wt_scale = torch.cat([q.t() for q, _ in pairs]).contiguous(), torch.cat([s.t() for _, s in pairs]).contiguous()
    dq, d_scale = build_fp8_quantize(M, N)(torch.randn(M, N, generator=g).bfloat16().cuda())
    offsets = torch.tensor([sum(counts[:e]) for e in range(E + 1)], dtype=torch.int32)
    dx = build_fp8_grouped_gemm_varlen(E, M, K, N)(dq, d_scale, wt, wt_scale, offsets.cuda()).cpu().double()
    for e in range(E):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        want, mag = formulas.fp8_gemm_ref(dq[lo:hi].cpu(), d_scale[lo:hi].cpu(), pairs[e][0].t().cpu(), pairs[e][1].t().cpu())
        assert ((dx[lo:hi] - want).abs() <= _gemm_bound(3, want, mag)).all()


def test_input_gradient_with_a_width_that_does_not_divide_by_sixteen():
    """N % 16 = 8: eight columns of zeros for dY, eight rows of zeros for the weight; its grid of scales stays."""
    M, N, K = 33, 264, 400
    g = torch.Generator().manual_seed(5)
    w8, w_scale = _weight(N, K, g)
    dy = torch.randn(M, N, generator=g).bfloat16().cuda()
    dq, d_scale = build_fp8_quantize(M, N + 8)(torch.nn.functional.pad(dy, (0, 8)))
    wt = torch.cat([w8, torch.zeros(8, K, device="cuda").to(w8.dtype)]).t().contiguous()
    dx = build_fp8_gemm(M, K, N + 8)(dq, d_scale, wt, w_scale.t().contiguous()).cpu().double()
    want, mag = formulas.fp8_gemm_ref(dq[:, :N].cpu(), d_scale.cpu(), w8.t().cpu(), w_scale.t().cpu())
    assert ((dx - want).abs() <= _gemm_bound(d_scale.shape[1], want, mag)).all()
