"""Training through the mixture-of-experts movement in bf16; it and the 8-bit products under torch.compile."""
import pytest
import torch

from oracle import formulas
from pyptx_b200.examples.blackwell import moe
from pyptx_b200.examples.blackwell.fp8_gemm import build_fp8_gemm, build_fp8_grouped_gemm_varlen, build_fp8_quantize
from pyptx_b200.types import bf16, f32

pytestmark = pytest.mark.gpu

U32, HALF16 = 2.0 ** -24, 2.0 ** -8


def _routing(T, k, E, block, seed, dropped=0.2):
    g = torch.Generator().manual_seed(seed)
    ids = torch.rand(T, E, generator=g).topk(k, dim=-1).indices.to(torch.int32)
    ids = torch.where(torch.rand(T, k, generator=g) < dropped, torch.full_like(ids, -1), ids)
    return (*moe.build_moe_route(T, k, E, block=block)(ids.cuda()), moe.moe_rows(T, k, E, block))


# ---- bf16 through autograd ------------------------------------------------------------------------

@pytest.mark.parametrize("T,k,E,H,block", [(1, 1, 1, 8, 1), (37, 3, 6, 1000, 4), (300, 4, 16, 520, 128)])
def test_bf16_gradients_of_dispatch_and_combine(T, k, E, H, block):
    row_of, entry_of, _, R = _routing(T, k, E, block, T)
    dispatch, combine = moe.build_differentiable_moe_dispatch(T, k, R, H), moe.build_differentiable_moe_combine(T, k, R, H)
    g = torch.Generator().manual_seed(H)
    x, d_rows, y, dout = (torch.randn(n, H, generator=g).bfloat16() for n in (T, R, R, T))
    w = torch.rand(T, k, generator=g) - 0.3

    xc = x.cuda().requires_grad_()
    rows = dispatch(xc, row_of, entry_of)
    assert rows.dtype == torch.bfloat16 and rows.requires_grad
    rows.backward(d_rows.cuda())
    want, mag = formulas.moe_combine_ref(d_rows, None, row_of.cpu())
    assert xc.grad.dtype == torch.bfloat16
    assert ((xc.grad.cpu().double() - want).abs() <= HALF16 * want.abs() + 2 * k * U32 * mag).all()

    yc, wc = y.cuda().requires_grad_(), w.cuda().requires_grad_()
    out = combine(yc, wc, row_of, entry_of)
    out.backward(dout.cuda())
    want_rows, want_w, mag_w = formulas.moe_combine_bwd_ref(y, w, row_of.cpu(), dout)
    assert yc.grad.dtype == torch.bfloat16 and wc.grad.dtype == torch.float32
    assert ((yc.grad.cpu().double() - want_rows).abs() <= (HALF16 + 2 * U32) * want_rows.abs()).all()
    assert ((wc.grad.cpu().double() - want_w).abs() <= H * U32 * mag_w).all()


def test_bf16_gradients_against_differences():
    """combine is linear in its weights and dispatch in its tokens, so central differences of step d are derivatives up to
    roundings: half a step of bf16 for each result on both sides, H half steps of f32 for the gradient's own sums, and half
    a step of bf16 for each gradient value that is bf16."""
    T, k, E, H, block = 50, 2, 5, 264, 8
    row_of, entry_of, _, R = _routing(T, k, E, block, 3)
    combine, dispatch = moe.build_differentiable_moe_combine(T, k, R, H), moe.build_differentiable_moe_dispatch(T, k, R, H)
    g = torch.Generator(device="cuda").manual_seed(4)
    y, dout = (torch.randn(n, H, generator=g, device="cuda").bfloat16() for n in (R, T))
    w = torch.rand(T, k, generator=g, device="cuda", requires_grad=True)
    d = torch.randn(T, k, generator=g, device="cuda")
    (gw,) = torch.autograd.grad(combine(y, w, row_of, entry_of), w, dout)
    with torch.no_grad():
        up, down = (combine(y, w + s * d, row_of, entry_of).double() for s in (1, -1))
        slope, weight = (gw.double() * d).sum(), dout.double()
        _, _, mag = formulas.moe_combine_bwd_ref(y.cpu(), w.detach().cpu(), row_of.cpu(), dout.cpu())
        slack = HALF16 * 0.5 * ((up.abs() + down.abs()) * weight.abs()).sum() + H * U32 * (mag.cuda() * d.abs()).sum()
        assert abs(((up - down) * 0.5 * weight).sum() - slope) <= slack * (1 + 2.0 ** -6)

    # dispatch: whole numbers up to 128, which bf16 holds, so the values on both sides are exact
    x = torch.randint(-64, 65, (T, H), generator=g, device="cuda").bfloat16().requires_grad_()
    step = torch.randint(-64, 65, (T, H), generator=g, device="cuda").bfloat16()
    d_rows = torch.randn(R, H, generator=g, device="cuda").bfloat16()
    (gx,) = torch.autograd.grad(dispatch(x, row_of, entry_of), x, d_rows)
    with torch.no_grad():
        up, down = (dispatch(x + s * step, row_of, entry_of).double() for s in (1, -1))
        slope = (gx.double() * step.double()).sum()
        _, mag = formulas.moe_combine_ref(d_rows.cpu(), None, row_of.cpu())
        slack = ((HALF16 * gx.double().abs() + 2 * k * U32 * mag.cuda()) * step.double().abs()).sum()
        assert abs(((up - down) * 0.5 * d_rows.double()).sum() - slope) <= slack * (1 + 2.0 ** -6)


def test_bf16_expanded_gradient_and_a_shared_leaf():
    T, k, E, H = 20, 2, 4, 64
    row_of, entry_of, _, R = _routing(T, k, E, 1, 6, dropped=0.0)
    dispatch = moe.build_differentiable_moe_dispatch(T, k, R, H)
    x = torch.randn(T, H, device="cuda").bfloat16().requires_grad_()
    (dispatch(x, row_of, entry_of).sum() + 2 * dispatch(x, row_of, entry_of).sum()).backward()
    assert torch.equal(x.grad, torch.full_like(x, 3.0 * k))


# ---- torch.compile ------------------------------------------------------------------------------------

def _weight(rows, cols, g):
    return build_fp8_quantize(rows, cols, block_rows=128, in_dtype=f32)((torch.randn(rows, cols, generator=g) / cols ** 0.5).cuda())


def test_compiled_training_step():
    T, k, E, H, block = 48, 2, 6, 128, 8
    row_of, entry_of, _, R = _routing(T, k, E, block, 9)
    dispatch, combine = moe.build_differentiable_moe_dispatch(T, k, R, H), moe.build_differentiable_moe_combine(T, k, R, H)
    x = torch.randn(T, H, device="cuda").bfloat16()
    w = torch.rand(T, k, device="cuda")

    def step(x_, w_):
        return combine(dispatch(x_, row_of, entry_of), w_, row_of, entry_of)

    grads = []
    for f in (step, torch.compile(step)):
        leaves = x.clone().requires_grad_(), w.clone().requires_grad_()
        out = f(*leaves)
        out.backward(torch.ones_like(out))
        grads.append((out.detach(), *(t.grad for t in leaves)))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


def test_compiled_eight_bit_products():
    M, N, K = 40, 264, 272
    g = torch.Generator().manual_seed(11)
    w8, w_scale = _weight(N, K, g)
    x = torch.randn(M, K, generator=g).bfloat16().cuda()
    offsets = torch.tensor([0, 13, 13, M], dtype=torch.int32).cuda()
    quantize, gemm = build_fp8_quantize(M, K), build_fp8_gemm(M, N, K, out_dtype=bf16)
    grouped = build_fp8_grouped_gemm_varlen(3, M, N, K)
    w3, w3_scale = w8.repeat(3, 1), w_scale.repeat(3, 1)

    def step(x_):
        q, scale = quantize(x_)
        return gemm(q, scale, w8, w_scale), grouped(q, scale, w3, w3_scale, offsets)

    for a, b in zip(torch.compile(step)(x), step(x)):
        assert torch.equal(a, b)
