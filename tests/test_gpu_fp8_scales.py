"""The 8-bit products at both ends of f32: what the builders say of the two scales' product, in every form of the
kernel, against float64.

The product of a row's and a weight block's scale is formed in f32.  While it lies in 2^-126 .. 2^127, a result's error is
that of the other tests of these products (256 + blocks + 9 half steps of the terms' magnitudes); as results may be
subnormal here, each of these roundings adds half of f32's smallest step, 2^-150, and a bf16 result its own half step, 2^-134
at least.  A smaller product is off by half of the smallest step too, 2^-150, times the block's sum of at most
128 * 448^2 < 2^24.62: 2^-125.38 for a block.  One of 2^128 and more is infinite, in its own row and column block alone."""
import pytest
import torch

from oracle import formulas
from pyptx_b200.examples.blackwell.fp8_gemm import build_fp8_gemm, build_fp8_grouped_gemm_varlen
from pyptx_b200.types import bf16, f32

pytestmark = pytest.mark.gpu

PTX = {"bf16": bf16, "f32": f32}
# streaming with one, two and four tiles of tokens; 32-row tiles, whole and shared K; 128-row tiles, whole and shared; pairs
DENSE = [(1, 4096, 1040), (7, 136, 400), (13, 264, 2064), (30, 520, 1040), (20, 1032, 4112), (24, 264, 8208), (100, 520, 1040),
         (40, 264, 4112), (2050, 2056, 528)]
# 32-row tiles, 128-row tiles, pairs
GROUPED = [([3, 0, 24, 40, 1], 264, 656), ([50, 90, 0, 130, 17], 264, 656), ([300, 129, 0, 513, 1], 520, 656)]


def _bits(shape, g):
    return (torch.randn(shape, generator=g) * 140).clamp(-448, 448).to(torch.float8_e4m3fn)


def _pow2(exponent, g):
    """2^exponent times a factor in [1, 2), exact in f32 down to its smallest step."""
    return (torch.exp2(exponent.double()) * (1 + torch.rand(exponent.shape, generator=g, dtype=torch.float64))).float()


def _check(got, a, sa, b, sb, kind, small_blocks=0):
    """``small_blocks``: blocks of K whose scales may multiply to less than 2^-126."""
    want, mag = formulas.fp8_gemm_ref(a, sa, b, sb)
    roundings = 256 + sa.shape[1] + 9
    bound = roundings * 2.0 ** -24 * mag + roundings * 2.0 ** -150 + small_blocks * 2.0 ** -125.38
    if kind == "bf16":
        bound = bound + (2.0 ** -8 * (want.abs() + bound)).clamp_min(2.0 ** -134)
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() - bound).max()
    assert worst <= 0, f"beyond the bound by {worst:.3e}"


def _scales(M, N, K, low, high, g, experts=1):
    """Scales whose products' exponents are spread over [low, high], from one small factor to two."""
    kb, nb = -(-K // 128), -(-N // 128)
    eb = torch.randint(max(-60, high - 126), 21, (1, kb), generator=g)
    ea = torch.randint(low, high + 1, (M, kb), generator=g) - eb
    return _pow2(ea, g), _pow2(eb, g).repeat(experts * nb, 1)


@pytest.mark.parametrize("M,N,K", DENSE)
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("low,high", [(-126, -110), (85, 94)])
def test_products_of_scales_at_the_ends_of_the_range(M, N, K, kind, low, high):
    """Results around 2^-100, and around 2^120 (each block's terms below 2^(94 + 2 + 24.6), at most 65 blocks)."""
    g = torch.Generator().manual_seed(M + N + K)
    a, b = _bits((M, K), g), _bits((N, K), g)
    sa, sb = _scales(M, N, K, low, high, g)
    out = build_fp8_gemm(M, N, K, out_dtype=PTX[kind])(a.cuda(), sa.cuda(), b.cuda(), sb.cuda())
    _check(out, a, sa, b, sb, kind)


@pytest.mark.parametrize("M,N,K", DENSE)
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_smaller_products_of_scales(M, N, K, kind):
    """Down to 2^-200; a fifth of the rows are ordinary and keep their precision."""
    g = torch.Generator().manual_seed(M + N + K)
    a, b = _bits((M, K), g), _bits((N, K), g)
    sa, sb = _scales(M, N, K, -139, -111, g)
    sb[:, ::2] *= 2.0 ** -61
    sa[4::5] = _pow2(torch.randint(0, 11, sa[4::5].shape, generator=g), g)
    out = build_fp8_gemm(M, N, K, out_dtype=PTX[kind])(a.cuda(), sa.cuda(), b.cuda(), sb.cuda())
    small = torch.arange(M) % 5 != 4
    _check(out[small.cuda()], a[small], sa[small], b, sb, kind, sa.shape[1])
    if not small.all():
        _check(out[~small.cuda()], a[~small], sa[~small], b, sb, kind)


@pytest.mark.parametrize("M,N,K", [(12, 264, 528), (24, 1032, 4112), (24, 1032, 528), (100, 520, 528), (2050, 2056, 528)])
def test_products_beyond_the_range_stay_in_their_rows(M, N, K):
    """2^100 x 2^30: infinite (NaN over a block of zeros) in the row and the column block; 2^-122 and 0 beside them."""
    g = torch.Generator().manual_seed(M)
    a, b = _bits((M, K), g), _bits((N, K), g).float().abs().clamp_min(1.0).to(torch.float8_e4m3fn)
    kb, nb = -(-K // 128), -(-N // 128)
    sa, sb = _pow2(torch.randint(-9, -6, (M, kb), generator=g), g), _pow2(torch.randint(-9, -6, (nb, kb), generator=g), g)
    sb[1, 2] = 2.0 ** 30                            # columns 128 .. 255
    sa[:, 2] *= 2.0 ** -40
    kernel = build_fp8_gemm(M, N, K)
    clean = kernel(a.cuda(), sa.cuda(), b.cuda(), sb.cuda())
    a2, sa2 = a.float(), sa.clone()
    a2[5, 256:384], a2[11, 256:384] = -2.0, 0.0
    sa2[5, 2] = sa2[11, 2] = 2.0 ** 100
    sa2[2::7, :2] *= 2.0 ** -118
    sa2[3::7, 1] = 0.0
    out = kernel(a2.to(torch.float8_e4m3fn).cuda(), sa2.cuda(), b.cuda(), sb.cuda())
    assert (out[5, 128:256] == float("-inf")).all() and torch.isnan(out[11, 128:256]).all()
    beside = torch.cat([out[:, :128], out[:, 256:]], dim=1)
    assert torch.isfinite(beside).all()
    same = torch.ones(M, dtype=torch.bool)
    same[5] = same[11] = same[2::7] = same[3::7] = False
    assert torch.equal(out[same.cuda()], clean[same.cuda()])
    rest = ~same
    rest[5] = rest[11] = False
    _check(out[rest.cuda()], a[rest], sa2[rest], b, sb, "f32", 2)


@pytest.mark.parametrize("counts,N,K", GROUPED)
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_grouped_with_smaller_products_of_scales(counts, N, K, kind):
    G, M, nb = len(counts), sum(counts), -(-N // 128)
    g = torch.Generator().manual_seed(M + N)
    a, b = _bits((M, K), g), _bits((G * N, K), g)
    sa, sb = _scales(M, N, K, -150, -111, g, experts=G)
    offsets = torch.tensor([sum(counts[:e]) for e in range(G + 1)], dtype=torch.int32)
    out = build_fp8_grouped_gemm_varlen(G, M, N, K, out_dtype=PTX[kind])(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), offsets.cuda())
    for e in range(G):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        if hi > lo:
            _check(out[lo:hi], a[lo:hi], sa[lo:hi], b[e * N:(e + 1) * N], sb[e * nb:(e + 1) * nb], kind, sa.shape[1])
