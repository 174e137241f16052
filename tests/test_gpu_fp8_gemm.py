"""GPU parity of the block-scaled e4m3 GEMMs against float64 products of the same 8-bit operands, and a
mixture-of-experts layer run through them.

Error bound of an f32 result: the tensor core adds 128 exact products (each of them has 8 significant
bits) in f32, the epilogue rounds the two scales' product, and one fma per block of K adds it to the sum.
With a rounding of at most one f32 step (2^-23; the tensor core may cut off instead of rounding) for each of
the products of a block and half a step for everything else, the result differs from the exact one by at
most (128 * 2^-23 + (blocks + 1) * 2^-24) times the sum of the terms' magnitudes; splitting K adds at
most 8 more half steps."""
import pytest
import torch

from oracle import formulas
from pyptx_b200.examples.blackwell import moe
from pyptx_b200.examples.blackwell.fp8_gemm import build_fp8_gemm, build_fp8_grouped_gemm_varlen, build_fp8_quantize
from pyptx_b200.examples.blackwell.swiglu import build_fused_silu_mul
from pyptx_b200.types import bf16, f32

pytestmark = pytest.mark.gpu

PTX = {"bf16": bf16, "f32": f32}
U32 = 2.0 ** -24
HALF_STEP = {"bf16": 2.0 ** -8, "f32": 0.0}


def _bound(blocks, kind, want, mag):
    return HALF_STEP[kind] * want.abs() + (256 + blocks + 9) * U32 * mag


def _operands(M, N, K, seed, experts=1):
    g = torch.Generator().manual_seed(seed)
    kb, nb = -(-K // 128), -(-N // 128)
    a = (torch.randn(M, K, generator=g) * 140).clamp(-448, 448).to(torch.float8_e4m3fn)
    b = (torch.randn(experts * N, K, generator=g) * 140).clamp(-448, 448).to(torch.float8_e4m3fn)
    sa = torch.exp2(2 * torch.randn(M, kb, generator=g)) / 140
    sb = torch.exp2(2 * torch.randn(experts * nb, kb, generator=g)) / 140
    return a, sa, b, sb


def _check(out, a, sa, b, sb, kind):
    want, mag = formulas.fp8_gemm_ref(a, sa, b, sb)
    got = out.cpu().double()
    assert got.shape == want.shape and torch.isfinite(got).all()
    excess = ((got - want).abs() - _bound(sa.shape[1], kind, want, mag)).max()
    assert excess <= 0, f"beyond the bound by {excess:.3e}"


# ---- known answers ------------------------------------------------------------------------------

@pytest.mark.parametrize("M,N,K", [(128, 256, 128), (1, 128, 64), (300, 520, 272), (128, 128, 1024)])
def test_ones_give_k_times_the_scales(M, N, K):
    kb, nb = -(-K // 128), -(-N // 128)
    one = torch.ones(M, K).to(torch.float8_e4m3fn).cuda()
    w = torch.ones(N, K).to(torch.float8_e4m3fn).cuda()
    sa = torch.exp2((torch.arange(M) % 5).float())[:, None].repeat(1, kb).cuda()
    sb = torch.exp2((torch.arange(nb) % 3).float())[:, None].repeat(1, kb).cuda()
    d = build_fp8_gemm(M, N, K)(one, sa, w, sb).cpu()
    want = K * sa[:, :1].cpu() * sb[:, 0].cpu().repeat_interleave(128)[:N]
    assert torch.equal(d, want)


def test_rows_columns_and_k_are_where_they_belong():
    """One nonzero per operand row pins every index: A[i, i % K], B[j, j % K], values coded by index."""
    M, N, K = 256, 384, 256
    a, b = torch.zeros(M, K), torch.zeros(N, K)
    i, j = torch.arange(M), torch.arange(N)
    a[i, i % K] = (1 + i % 15).float()
    b[j, (j * 7) % K] = (1 + j % 13).float()
    d = build_fp8_gemm(M, N, K)(a.to(torch.float8_e4m3fn).cuda(), torch.ones(M, 2).cuda(),
                               b.to(torch.float8_e4m3fn).cuda(), torch.ones(3, 2).cuda()).cpu()
    assert torch.equal(d, a @ b.T)


def test_every_scale_block_counts_once():
    """All-ones operands and scales that are distinct powers of two: the result is the sum over blocks."""
    M, N, K = 130, 264, 1040
    kb, nb = 9, 3
    sa = torch.exp2(-(torch.arange(M)[:, None] + torch.arange(kb)[None]).remainder(7).float())
    sb = torch.exp2(-(3 * torch.arange(nb)[:, None] + torch.arange(kb)[None]).remainder(5).float())
    width = torch.tensor([128.0] * 8 + [16.0])
    want = (sa * width) @ sb.T                      # exact: sums of few powers of two
    d = build_fp8_gemm(M, N, K)(torch.ones(M, K).to(torch.float8_e4m3fn).cuda(), sa.cuda(),
                               torch.ones(N, K).to(torch.float8_e4m3fn).cuda(), sb.cuda()).cpu()
    assert torch.equal(d, want.repeat_interleave(128, dim=1)[:, :N])


# ---- dense --------------------------------------------------------------------------------------

@pytest.mark.parametrize("M,N,K", [
    (1, 8, 16), (1, 4096, 4096), (2, 136, 128), (3, 520, 2064), (8, 2056, 8208), (9, 1016, 528), (16, 1024, 4096), (17, 72, 5120), (24, 4104, 2048), (12, 8200, 2064), (31, 264, 144), (32, 256, 256),
    (17, 1024, 1024), (32, 2048, 2048), (25, 1000, 528), (32, 8, 16), (28, 4096, 1024), (31, 520, 2176),
    (300, 1000, 2576), (40, 1024, 4096), (33, 264, 8992), (20, 200, 8208), (130, 2056, 2640),      # K shared by 2 to 8 CTAs
    (33, 256, 384), (64, 2056, 1040), (127, 128, 512), (128, 384, 640), (129, 248, 272), (333, 2056, 1040),
    (512, 512, 16), (1000, 1000, 1008), (2048, 2048, 256), (1030, 4104, 528), (4000, 1544, 400), (8192, 264, 128),
])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_dense(M, N, K, kind):
    a, sa, b, sb = _operands(M, N, K, M + 3 * N + 7 * K)
    d = build_fp8_gemm(M, N, K, out_dtype=PTX[kind])(a.cuda(), sa.cuda(), b.cuda(), sb.cuda())
    _check(d, a, sa, b, sb, kind)


@pytest.mark.parametrize("M,N,K", [(10, 256, 512), (16, 256, 512), (20, 256, 512), (28, 520, 4224), (40, 256, 512)])
def test_special_scales_and_values_stay_in_their_rows(M, N, K):
    """Streaming, 32-row and 128-row forms."""
    a, sa, b, sb = _operands(M, N, K, 5)
    clean = build_fp8_gemm(M, N, K)(a.cuda(), sa.cuda(), b.cuda(), sb.cuda())
    a2, sa2 = a.float(), sa.clone()
    a2[3, 200] = float("nan")
    sa2[7, 1] = float("inf")
    sa2[9] = 0.0
    out = build_fp8_gemm(M, N, K)(a2.to(torch.float8_e4m3fn).cuda(), sa2.cuda(), b.cuda(), sb.cuda())
    assert torch.isnan(out[3]).all() and not torch.isfinite(out[7]).any() and (out[9] == 0).all()
    keep = torch.ones(M, dtype=torch.bool)
    keep[[3, 7, 9]] = False
    assert torch.equal(out[keep.cuda()], clean[keep.cuda()])


@pytest.mark.parametrize("M,N,K", [(8192, 264, 128), (4096, 520, 64), (16384, 136, 128), (4096, 4096, 128),
                                   (40000, 120, 128)])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_tiles_in_quick_succession(M, N, K, kind):
    """One scale block a tile and several tiles a CTA: a tile's results leave through buffers that the next
    tile fills at once."""
    a, sa, b, sb = _operands(M, N, K, 11)
    kernel = build_fp8_gemm(M, N, K, out_dtype=PTX[kind])
    ins = [t.cuda() for t in (a, sa, b, sb)]
    first = kernel(*ins)
    _check(first, a, sa, b, sb, kind)
    for _ in range(10):
        assert torch.equal(kernel(*ins), first)


def test_special_weights_stay_in_their_columns():
    for M, N, K in ((3, 384, 256), (20, 384, 256), (20, 384, 2304), (200, 384, 256)):
        a, sa, b, sb = _operands(M, N, K, 6)
        clean = build_fp8_gemm(M, N, K)(a.cuda(), sa.cuda(), b.cuda(), sb.cuda())
        b2, sb2 = b.float(), sb.clone()
        b2[77, 130] = float("nan")
        sb2[2, 0] = float("inf")                             # columns 256 .. 383
        out = build_fp8_gemm(M, N, K)(a.cuda(), sa.cuda(), b2.to(torch.float8_e4m3fn).cuda(), sb2.cuda())
        assert torch.isnan(out[:, 77]).all() and not torch.isfinite(out[:, 256:]).any()
        keep = torch.arange(256) != 77
        assert torch.equal(out[:, :256][:, keep.cuda()], clean[:, :256][:, keep.cuda()])


def test_results_beyond_two_to_the_31_elements():
    M, N, K = 270000, 8192, 128                              # 2.2e9 results
    g = torch.Generator(device="cuda").manual_seed(3)
    a = (torch.randn(M, K, generator=g, device="cuda") * 140).clamp(-448, 448).to(torch.float8_e4m3fn)
    b = (torch.randn(N, K, generator=g, device="cuda") * 140).clamp(-448, 448).to(torch.float8_e4m3fn)
    sa, sb = torch.rand(M, 1, generator=g, device="cuda"), torch.rand(N // 128, 1, generator=g, device="cuda")
    d = build_fp8_gemm(M, N, K, out_dtype=bf16)(a, sa, b, sb)
    for rows in (slice(0, 64), slice(262100, 262200), slice(M - 70, M)):
        _check(d[rows], a[rows].cpu(), sa[rows].cpu(), b.cpu(), sb.cpu(), "bf16")


def test_repeated_calls_give_the_same_bits():
    for M, N, K in ((1, 1024, 4096), (700, 1024, 512)):
        a, sa, b, sb = (t.cuda() for t in _operands(M, N, K, 1))
        kernel = build_fp8_gemm(M, N, K)
        first = kernel(a, sa, b, sb)
        for _ in range(3):
            assert torch.equal(kernel(a, sa, b, sb), first)


@pytest.mark.parametrize("M", [1, 12, 40])
def test_a_weight_made_by_the_kernel_before(M):
    """The weight is quantised right before each product, replay after replay: no stale bytes."""
    N, K = 1024, 4096
    quantize, gemm = build_fp8_quantize(N, K, block_rows=128), build_fp8_gemm(M, N, K)
    w = torch.empty(N, K, dtype=torch.bfloat16, device="cuda")
    a, sa = torch.randn(M, K, device="cuda").to(torch.float8_e4m3fn), torch.rand(M, K // 128, device="cuda")
    gemm(a, sa, *quantize(w.zero_()))
    graph, outs = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        for _ in range(8):                       # the same buffers again and again, another weight each time
            q, s = quantize(w)
            outs.append(gemm(a, sa, q, s))
            del q, s
            w.neg_().mul_(1.5)
    for seed in range(5):
        g = torch.Generator(device="cuda").manual_seed(seed)
        w.normal_(generator=g)
        graph.replay()
        got = [o.clone() for o in outs]
        w.normal_(generator=g.manual_seed(seed))
        for o in got:
            torch.cuda.synchronize()
            q, s = quantize(w)
            torch.cuda.synchronize()
            assert torch.equal(o, gemm(a, sa, q, s))
            w.neg_().mul_(1.5)


# ---- grouped ------------------------------------------------------------------------------------

def _grouped(counts, N, K, kind, capacity=None, first=0):
    G, total = len(counts), first + sum(counts)
    M = total if capacity is None else capacity
    a, sa, b, sb = _operands(M, N, K, G + N + K + total, experts=G)
    offsets = torch.tensor([first + sum(counts[:e]) for e in range(G + 1)], dtype=torch.int32)
    kernel = build_fp8_grouped_gemm_varlen(G, M, N, K, out_dtype=PTX[kind])
    out = kernel(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), offsets.cuda())
    nb = -(-N // 128)
    for e in range(G):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        if hi > lo:
            _check(out[lo:hi], a[lo:hi], sa[lo:hi], b[e * N:(e + 1) * N], sb[e * nb:(e + 1) * nb], kind)


@pytest.mark.parametrize("counts,N,K", [
    ([1], 8, 16), ([0, 1, 0], 128, 128), ([5, 0, 0, 7, 1], 264, 272), ([128, 128], 256, 256), ([130, 1, 33, 32, 300], 520, 640),
    ([0] * 63 + [3], 136, 144), ([2] * 300, 72, 128), ([1000, 0, 17], 1032, 528), ([40, 700, 3, 260], 384, 1024),
    ([1] * 1024, 64, 64), ([24, 40, 8, 24], 264, 1168), ([100, 27, 0, 90], 384, 1552), ([513, 255, 256, 1, 0, 700], 264, 272), ([300, 2500], 520, 1296),
])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_grouped(counts, N, K, kind):
    _grouped(counts, N, K, kind)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("counts,N,K", [([128] * 40, 1024, 128), ([120] * 40, 1024, 128), ([24] * 100, 640, 1040), ([96, 32, 128] * 20, 640, 64), ([700, 300] * 4, 2048, 128)])
def test_grouped_tiles_in_quick_succession(counts, N, K, kind):
    """As above for the grouped forms: 128-column tiles (fewer than 128 rows an expert) and CTA pairs."""
    for _ in range(3):
        _grouped(counts, N, K, kind)


def test_grouped_leaves_rows_outside_the_offsets_alone():
    G, M, N, K = 3, 400, 264, 256
    a, sa, b, sb = _operands(M, N, K, 2, experts=G)
    kernel = build_fp8_grouped_gemm_varlen(G, M, N, K)
    from pyptx_b200 import _native
    out = torch.full((M, N), -7.0, device="cuda")
    for offs in ([10, 50, 50, 177], [0, 0, 0, 0], [400, 400, 400, 400]):
        out.fill_(-7.0)
        ins = [t.cuda() for t in (a, sa, b, sb)] + [torch.tensor(offs, dtype=torch.int32).cuda()]
        _native.launch_raw(kernel.handle, torch.cuda.current_stream().cuda_stream, [t.data_ptr() for t in ins] + [out.data_ptr()])
        torch.cuda.synchronize()
        assert (out[:offs[0]] == -7.0).all() and (out[offs[-1]:] == -7.0).all()
        for e in range(G):
            lo, hi = offs[e], offs[e + 1]
            if hi > lo:
                _check(out[lo:hi], a[lo:hi], sa[lo:hi], b[e * N:(e + 1) * N], sb[e * 3:(e + 1) * 3], "f32")


def test_grouped_offsets_are_made_safe():
    """Offsets that decrease or leave [0, M_total] are taken as their running maximum, clipped."""
    G, M, N, K = 4, 200, 128, 128
    a, sa, b, sb = _operands(M, N, K, 3, experts=G)
    kernel = build_fp8_grouped_gemm_varlen(G, M, N, K)
    out = kernel(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), torch.tensor([-5, 60, 20, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32).cuda())
    for e, (lo, hi) in enumerate(((0, 60), (60, 60), (60, 200), (200, 200))):
        if hi > lo:
            _check(out[lo:hi], a[lo:hi], sa[lo:hi], b[e * N:(e + 1) * N], sb[e:e + 1], "f32")


# ---- used together ------------------------------------------------------------------------------

@pytest.mark.parametrize("T,k,E,H,F,block", [(1, 2, 4, 256, 128, 1), (50, 4, 16, 512, 384, 1), (700, 2, 6, 1024, 512, 16)])
def test_a_layer_of_experts(T, k, E, H, F, block):
    """Route, dispatch into 8 bits, gate and up products, SwiGLU, quantise, down product, combine -- against
    the same layer in float64 on the dequantised operands of each product."""
    g = torch.Generator().manual_seed(T)
    R = moe.moe_rows(T, k, E, block)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16)
    ids = torch.rand(T, E, generator=g).topk(k, dim=-1).indices
    probs = torch.softmax(torch.randn(T, k, generator=g), dim=-1)
    weights = {name: torch.randn(E * rows, cols, generator=g) / cols ** 0.5 for name, rows, cols in
               (("gate", F, H), ("up", F, H), ("down", H, F))}
    quant = {name: build_fp8_quantize(w.shape[0], w.shape[1], block_rows=128, in_dtype=f32)(w.cuda()) for name, w in weights.items()}

    row_of, entry_of, offsets = moe.build_moe_route(T, k, E, block=block)(ids.to(torch.int32).cuda())
    q, scale = moe.build_moe_dispatch_fp8(T, k, R, H)(x.cuda(), row_of, entry_of)
    up_kernel = build_fp8_grouped_gemm_varlen(E, R, F, H)
    gate, up = up_kernel(q, scale, *quant["gate"], offsets), up_kernel(q, scale, *quant["up"], offsets)
    act = build_fused_silu_mul(R, F)(gate, up)
    aq, a_scale = build_fp8_quantize(R, F, in_dtype=f32)(act)
    y = build_fp8_grouped_gemm_varlen(E, R, H, F, out_dtype=bf16)(aq, a_scale, *quant["down"], offsets)
    out = moe.build_moe_combine(T, k, R, H)(y, probs.cuda(), row_of).cpu().double()

    ends = offsets.tolist()
    y_want, y_tol = torch.zeros(R, H, dtype=torch.float64), torch.zeros(R, H, dtype=torch.float64)
    for e in range(E):
        lo, hi = ends[e], ends[e + 1]
        if lo == hi:
            continue
        def part(name, rows):
            w, s = (t.cpu() for t in quant[name])
            nb = -(-rows // 128)
            return w[e * rows:(e + 1) * rows], s[e * nb:(e + 1) * nb]
        for got, name in ((gate, "gate"), (up, "up")):
            _check(got[lo:hi], q.cpu()[lo:hi], scale.cpu()[lo:hi], *part(name, F), "f32")
        want, mag = formulas.fp8_gemm_ref(aq.cpu()[lo:hi], a_scale.cpu()[lo:hi], *part("down", H))
        y_want[lo:hi], y_tol[lo:hi] = want, _bound(a_scale.shape[1], "bf16", want, mag)
    want, mag = formulas.moe_combine_ref(y_want, probs, row_of.cpu())
    tol, _ = formulas.moe_combine_ref(y_tol, probs, row_of.cpu())
    assert ((out - want).abs() <= tol * (1 + 2.0 ** -7) + 2.0 ** -8 * want.abs() + 2 * k * U32 * mag).all()


def test_graph_and_side_stream():
    M, N, K = 20, 512, 1024
    a, sa, b, sb = (t.cuda() for t in _operands(M, N, K, 8))
    kernel = build_fp8_gemm(M, N, K, out_dtype=bf16)
    quantize = build_fp8_quantize(M, K)
    x = torch.randn(M, K, device="cuda").to(torch.bfloat16)

    def step():
        return kernel(*quantize(x), b, sb)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2):
        x.copy_(torch.randn(M, K, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())
